"""qmh_beam_reorder of many beams whose rows end inside a word, in workgroups that several waves share."""
import ctypes

import numpy as np
import pytest

import _ops as o

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("beams", [16, 17, 20, 33, 64])
@pytest.mark.parametrize("outer,rows,row_stride,live", [(1, 300, 136, 134), (2, 300, 512, 262), (1, 777, 8, 5), (1, 500, 4, 3), (1, 500, 4, 1), (2, 64, 1028, 1025),
                                                        (1, 300, 136, 135), (1, 301, 60, 57)])
def test_beam_reorder_tails(gpu, inplace, beams, outer, rows, row_stride, live):
    """Strides of whole words, and 1 to 3 bytes at the end of each row."""
    q = gpu
    rs = np.random.default_rng(beams * 7 + live)
    groups = 2
    B = groups * beams
    src = rs.integers(0, 256, (outer, B, rows, row_stride)).astype(np.uint8)
    dst = src if inplace else rs.integers(0, 256, src.shape).astype(np.uint8)
    ring = ((np.arange(B) % beams + 1) % beams).astype(np.int32)
    for parent in (ring, rs.integers(0, beams, B).astype(np.int32), rs.integers(-1, beams + 1, B).astype(np.int32)):
        ds = o.Guarded(q, src)
        dd = ds if inplace else o.Guarded(q, dst)
        dp = o.Guarded(q, parent)
        st = q.BeamState(n_outer=outer, outer_stride=B * rows * row_stride, seq_stride=rows * row_stride, n_rows=rows, row_stride=row_stride, live=live)
        q._check(q.load_library().qmh_beam_reorder(ctypes.byref(st), dd.ptr, ds.ptr, dp.ptr, groups, beams, None), "reorder")
        q.sync()
        own = np.arange(B)
        frm = np.where((parent >= 0) & (parent < beams), own - own % beams + parent, own)
        want = dst.copy()
        want[..., :live] = src[:, frm][..., :live]
        assert np.array_equal(dd.get(), want)
        if not inplace:
            assert np.array_equal(ds.get(), src)
