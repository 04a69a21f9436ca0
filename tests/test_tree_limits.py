"""Sizes of the ops for drafted trees that are too large together, though each is within its range, and arrays that overlap: refused
before anything reaches a device, and the largest sizes that are not."""
import ctypes

import pytest

from test_paged_refusals import P, refused
from test_tree_refusals import accept_args, logits_args, plan_args, tree_args


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


@pytest.mark.parametrize("n_seq,q_len", [(1026, 1024), (1 << 20, 1 << 20), (2, 1 << 20)])
def test_attention_counts_rows_not_sequences_times_nodes(qmh, n_seq, q_len):
    """The rows that there are (here -1: refused for that), not n_seq * q_len, are bounded where first says whose they are."""
    L = qmh.load_library()
    base = dict(n_seq=n_seq, q_len=q_len)
    for first, what in ((P, "n_rows"), (None, "queries")):
        a = tree_args(qmh, base=base, n_rows=-1, first=first, mask=None)
        assert L.qmh_tree_attention_ws(ctypes.byref(a)) == 0
        refused(qmh, L.qmh_tree_attention(ctypes.byref(a), P, 1 << 40, None), "tree_attention")
        assert what in qmh.last_error()
    for bad in (dict(n_seq=(1 << 20) + 2), dict(q_len=(1 << 20) + 1)):
        a = tree_args(qmh, base={**base, **bad}, mask=None)
        refused(qmh, L.qmh_tree_attention(ctypes.byref(a), P, 1 << 40, None), "tree_attention")
        assert "queries" in qmh.last_error()


INPUTS, OUTPUTS = "parent token choice len first table".split(), "count path next keep history history_len".split()


@pytest.mark.parametrize("out,other", [(x, y) for x in OUTPUTS for y in INPUTS + OUTPUTS if x != y])
def test_accept_of_arrays_that_are_two_things(qmh, out, other):
    d = {k: (10 + i) * P for i, k in enumerate(INPUTS + OUTPUTS)}
    d[out] = d[other]
    refused(qmh, qmh.load_library().qmh_tree_accept(ctypes.byref(accept_args(qmh, **d)), None), "tree_accept")
    assert "overlap" in qmh.last_error()


def test_plan_of_positions_that_count_from_the_length(qmh):
    """Lengths are written before positions are: base has to be a copy."""
    L, a = qmh.load_library(), plan_args(qmh, base=P)
    assert L.qmh_paged_plan_ws(ctypes.byref(a)) == 0
    refused(qmh, L.qmh_paged_plan(ctypes.byref(a), P, 1 << 40, None), "paged_plan")
    assert "base" in qmh.last_error()
