"""Edited logits (qmh_logits_edit) of so many sequences, most of them without rows, that their workgroups are more than one launch takes."""
import ctypes

import numpy as np
import pytest

import _ops as o

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_more_workgroups_than_a_launch_holds(gpu, dtype):
    q, dt, rs = gpu, o.TYPES[dtype], np.random.default_rng(4)
    n_seq, per, rows, V = 65535, 1024, 1024, 16385  # 5 segments x 32 pieces of rows x 65535 workgroups of 512 threads: 1.25 times 2^32
    counts = np.zeros(n_seq, np.int64)
    counts[[0, 7, 41234, 52428, 52430, 65534]] = [3, 500, 40, 1, 200, 280]
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    owner = np.repeat(np.arange(n_seq), counts)
    x = rs.integers(-24, 25, (rows, V)) / 4
    token, bias = rs.integers(0, V, n_seq).astype(np.int32), (rs.integers(0, 17, n_seq) / 4).astype(np.float32)
    dev = q.DeviceBuffer.from_array
    dx, out, best = o.Guarded(q, o.encode(x, dt)), o.Guarded(q, np.zeros((rows, V), o.raw(dt))), o.Guarded(q, np.full(rows, -7, np.int32))
    keep = [dev(first), dev(token), dev(bias), dev(np.ones(n_seq, np.int32))]
    a = q.LogitsArgs(dtype=dt, n_rows=rows, vocab=V, logits=dx.ptr, stride=V, out=out.ptr, out_stride=V, best=best.ptr, n_seq=n_seq, rows_per_seq=per,
                     first=keep[0].ptr, bias_token=keep[1].ptr, bias=keep[2].ptr, bias_len=keep[3].ptr, bias_stride=1)
    L = q.load_library()
    need = L.qmh_logits_edit_ws(ctypes.byref(a))
    assert need > 0
    ws = o.Guarded(q, np.full(need, 0xFF, np.uint8))
    q._check(L.qmh_logits_edit(ctypes.byref(a), ws.ptr, need, None), "logits_edit")
    q.sync()
    ws.get()
    want = x.copy()
    want[np.arange(rows), token[owner]] += bias[owner]
    assert len(owner) == rows
    assert np.array_equal(o.decode(out.get(), dt), want)  # quarters: exact
    assert np.array_equal(best.get(), want.argmax(1))
