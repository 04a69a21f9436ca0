"""qmh_paged_reorder with lengths that are none, or above the bound."""
import ctypes

import numpy as np
import pytest

import _ops as o
from test_gpu_paged import pages_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams", [2, 12, 20])
def test_paged_reorder_lengths_that_are_none(gpu, beams):
    """A parent whose length is below 0 gives nothing, however far below; one above the bound gives up to the bound."""
    q, KV, hd, ps = gpu, 1, 16, 16
    rs = np.random.default_rng(beams)
    most = 3 * ps + 5
    length = np.array([[-1, -2 ** 31, 2 ** 31 - 1, -2 ** 31 + 1, 7, -2 ** 31 + 40, 0][i % 7] for i in range(beams)], np.int32)
    table, n_pages = o.make_tables(rs, [4] * beams, 4)
    k, v = (rs.integers(0, 2 ** 16, (n_pages, KV, ps, hd)).astype(np.uint16) for _ in range(2))
    parent = ((np.arange(beams) + 1) % beams).astype(np.int32)
    dk, dv = o.Guarded(q, k), o.Guarded(q, v)
    dtab, dlen, dpar = (o.Guarded(q, x) for x in (table, length, parent))
    p = pages_of(q, o.F16, KV, hd, ps, n_pages, dk.ptr, dv.ptr)
    q._check(q.load_library().qmh_paged_reorder(ctypes.byref(p), dtab.ptr, 4, dlen.ptr, most, dpar.ptr, 1, beams, None), "reorder")
    q.sync()
    wk, wv = k.copy(), v.copy()
    for i, f in enumerate(parent):
        for t in range(min(max(int(length[f]), 0), most)):
            a, b = table[f, t // ps], table[i, t // ps]
            wk[b, :, t % ps], wv[b, :, t % ps] = k[a, :, t % ps], v[a, :, t % ps]
    assert np.array_equal(dk.get(), wk) and np.array_equal(dv.get(), wv)
