"""qmh_paged_append of heads that hold infinities and NaN: what a rotation does not turn stays as it is, bit for bit."""
import ctypes

import numpy as np
import pytest

import _ops as o
from test_gpu_paged import pages_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("hd,rot", [(64, 0), (64, 32), (64, 64), (80, 20), (248, 6), (24, 12), (8, 2)])
def test_append_elements_that_are_not_turned(gpu, dtype, layout, hd, rot):
    q, dt, H, KV, n = gpu, o.TYPES[dtype], 2, 1, 24
    rs = np.random.default_rng(hd + rot)
    x = rs.standard_normal((n, H + 2 * KV, hd))
    odd = rs.choice([np.inf, -np.inf, 0.0, -0.0, 1.0, -1.0, 6e4, 1e-7], x.shape)
    x = np.where(rs.random(x.shape) < 0.3, odd, x)
    x[n // 2 :] = np.where(rs.random(x[n // 2 :].shape) < 0.05, np.nan, x[n // 2 :])
    x[:, :, :rot] = rs.standard_normal((n, H + 2 * KV, rot))  # the turned part is ordinary
    enc = o.encode(x, dt)
    pool = [o.Guarded(q, np.zeros((2, KV, 16, hd), o.raw(dt))) for _ in range(2)]
    p = pages_of(q, dt, KV, hd, 16, 2, pool[0].ptr, pool[1].ptr)
    dx, out = o.Guarded(q, enc.reshape(n, -1)), o.Guarded(q, np.zeros((n, H * hd), o.raw(dt)))
    seq, slot, pos, table = (o.Guarded(q, np.array(a, np.int32)) for a in (np.zeros(n), np.arange(n), np.arange(n) * 3, [[1, 0]]))
    width, es = (H + 2 * KV) * hd, o.BYTES[dt]
    rotary = q.Rotary(rot, layout, max_pos=100) if rot else None
    a = q.AppendArgs(pages=ctypes.pointer(p), rotary=rotary.handle if rotary else None, n_tokens=n, n_heads=H, q=dx.ptr, q_stride=width,
                     q_out=out.ptr, q_out_stride=H * hd, k=dx.ptr + H * hd * es, k_stride=width, v=dx.ptr + (H + KV) * hd * es, v_stride=width, n_seq=1,
                     table=table.ptr, table_stride=2, seq=seq.ptr, slot=slot.ptr, pos=pos.ptr)
    q._check(q.load_library().qmh_paged_append(ctypes.byref(a), None), "append")
    q.sync()
    rows = lambda b: b.get()[[1, 0]].transpose(0, 2, 1, 3).reshape(32, KV, hd)[:n]  # noqa: E731
    got = np.concatenate([out.get().reshape(n, H, hd), rows(pool[0]), rows(pool[1])], 1)
    if rotary:
        rotary.close()
    nan = np.isnan(o.decode(enc, dt))
    assert np.array_equal(np.isnan(o.decode(got, dt))[:, :, rot:], nan[:, :, rot:]), "NaN elsewhere"
    same = (got.view(np.uint32 if dt == o.F32 else np.uint16) == enc.view(np.uint32 if dt == o.F32 else np.uint16)) | nan
    assert same[:, :, rot:].all(), "an element that is not turned has changed"
    want = o.rotate(o.decode(enc, dt), np.arange(n) * 3, o.freqs(rot, "none") if rot else np.zeros(0), layout)
    r = np.abs(o.decode(enc, dt)[:, :3, :rot]).max(initial=0)
    o.close(o.decode(got, dt)[:, :3, :rot], want[:, :3, :rot], 8 * o.U32 * r + o.HALF[dt] * np.abs(want[:, :3, :rot]) + o.TINY[dt], "turned")
