"""qmh_beam_select_ws of no groups: nothing is needed, whatever the other sizes."""
import ctypes

import pytest

import _ops as o

P = 1 << 20  # an address: sizes are asked for, nothing is read


@pytest.mark.parametrize("beams,vocab,n_out", [(1, 1, 1), (4, 32000, 8), (64, 128256, 64)])
def test_no_groups_need_no_workspace(qmh, beams, vocab, n_out):
    a = qmh.BeamArgs(dtype=o.F32, n_groups=0, n_beams=beams, vocab=vocab, n_out=n_out, logits=P, stride=vocab, score=P, out_score=2 * P,
                     out_parent=P, out_token=P)
    ws = qmh.load_library().qmh_beam_select_ws
    assert ws(ctypes.byref(a)) == 0
    a.n_groups = 1
    assert ws(ctypes.byref(a)) > 0
