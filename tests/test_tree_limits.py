"""Sizes of the ops for drafted trees that are too large together, though each is within its range: refused before anything reaches a
device, and the largest that are not."""
import ctypes

import pytest

from test_paged_refusals import P, refused
from test_tree_refusals import logits_args


@pytest.mark.parametrize("kw", [
    dict(n_seq=65535, rows_per_seq=1 << 20, n_rows=1 << 20, vocab=8193), dict(n_seq=1 << 15, rows_per_seq=1 << 19, n_rows=1 << 20, vocab=1 << 15),
    dict(n_seq=1024, rows_per_seq=1 << 20, n_rows=1 << 20, vocab=(1 << 19) + 1)])
def test_logits_of_too_many_workgroups(qmh, kw):
    n = kw["vocab"]
    L = qmh.load_library()
    a = logits_args(qmh, first=P, stride=n, out_stride=n, allow=None, node_token=None, **kw)
    assert L.qmh_logits_edit_ws(ctypes.byref(a)) == 0
    refused(qmh, L.qmh_logits_edit(ctypes.byref(a), P, 1 << 40, None), "logits_edit")
    assert "too many" in qmh.last_error()


@pytest.mark.parametrize("kw", [
    dict(n_seq=65535, rows_per_seq=1 << 20, n_rows=1 << 20, vocab=8192), dict(n_seq=65535, rows_per_seq=1 << 20, n_rows=1024, vocab=8193),
    dict(n_seq=1024, rows_per_seq=1 << 20, n_rows=1 << 20, vocab=127 << 12)])
def test_logits_that_are_not(qmh, kw):
    """These get as far as the workspace's check (best tokens of more than 4096 need one), or (without a device) as the device's."""
    n = kw["vocab"]
    assert n > 4096
    a = logits_args(qmh, first=P, stride=n, out_stride=n, allow=None, node_token=None, **kw)
    assert qmh.load_library().qmh_logits_edit(ctypes.byref(a), None, 0, None) == -1
    assert "too many" not in qmh.last_error()
