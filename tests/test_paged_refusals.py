"""What the ops for several continuations of one prompt refuse: every bad argument is an error code with a message that
names the op, before anything reaches a device."""
import ctypes

import pytest

import _ops as o

P = 1 << 20  # an address that no refused call looks at


def pages(lib, **kw):
    d = dict(dtype=o.BF16, n_kv_heads=2, head_dim=64, page_size=16, n_pages=8, k=P, v=P)
    d.update(kw)
    return lib.Pages(**d)


def append(lib, pg=None, **kw):
    d = dict(n_tokens=4, n_heads=4, q=P, q_stride=512, q_out=P, q_out_stride=512, k=P, k_stride=512, v=P, v_stride=512, eps=1e-5, n_seq=2,
             table=P, table_stride=4, seq=P, slot=P, pos=P)
    d.update(kw)
    a = lib.AppendArgs(**d)
    a.pages = ctypes.pointer(pages(lib, **(pg or {})))
    return lib.load_library().qmh_paged_append(ctypes.byref(a), None)


def attention_args(lib, pg=None, **kw):
    d = dict(n_heads=4, n_seq=4, q_len=1, n_groups=2, q=P, q_stride=256, out=2 * P, out_stride=256, table=P, len=P, table_stride=8,
             max_len=100, prefix_table=P, prefix_len=P, prefix_stride=8, max_prefix=128, scale=0.125)
    d.update(kw)
    a = lib.AttentionArgs(**d)
    a.pages = ctypes.pointer(pages(lib, **(pg or {})))
    return a


def beam_args(q, **kw):
    d = dict(dtype=o.F32, n_groups=2, n_beams=4, vocab=100, n_out=8, eos=2, logits=P, stride=100, score=P, out_score=2 * P, out_parent=P,
             out_token=P)
    d.update(kw)
    return q.BeamArgs(**d)


def refused(q, rc, what):
    assert rc == -1, "taken"
    assert what in q.last_error(), q.last_error()


BAD_PAGES = [dict(dtype=2), dict(dtype=7), dict(head_dim=0), dict(head_dim=12), dict(head_dim=264), dict(page_size=8), dict(page_size=48),
             dict(page_size=2048), dict(n_pages=0), dict(n_pages=1 << 31), dict(n_kv_heads=0), dict(k=None), dict(v=P + 8)]


@pytest.mark.parametrize("pg", BAD_PAGES)
def test_pages(qmh, pg):
    refused(qmh, append(qmh, pg), "paged_append")
    assert qmh.load_library().qmh_paged_attention_ws(ctypes.byref(attention_args(qmh, pg))) == 0
    refused(qmh, qmh.load_library().qmh_paged_attention(ctypes.byref(attention_args(qmh, pg)), P, 1 << 30, None), "paged_attention")
    p = pages(qmh, **pg)
    refused(qmh, qmh.load_library().qmh_paged_reorder(ctypes.byref(p), P, 4, P, 60, P, 2, 2, None), "paged_reorder")


@pytest.mark.parametrize("kw", [dict(n_tokens=-1), dict(q=None), dict(q_out=None), dict(q_stride=255), dict(q_out_stride=255), dict(q=P + 1),
                                dict(q_out=P, q_out_stride=640), dict(n_heads=0), dict(k=None), dict(v=None), dict(k_stride=127),
                                dict(v_stride=-512), dict(table=None), dict(seq=None), dict(slot=None), dict(n_seq=0), dict(table_stride=0),
                                dict(table_stride=1 << 28), dict(q=None, q_out=None, k=None, v=None), dict(q_gain=P, eps=-1.0),
                                dict(k_gain=P, eps=float("nan"))])
def test_append(qmh, kw):
    refused(qmh, append(qmh, **kw), "paged_append")


@pytest.mark.parametrize("kw", [dict(n_heads=0), dict(n_heads=3), dict(n_seq=-1), dict(q_len=0), dict(q_len=1 << 20), dict(n_groups=0), dict(n_groups=3),
                                dict(q=None), dict(out=None), dict(q_stride=255), dict(q_stride=260), dict(out_stride=252), dict(q=P + 2), dict(out=P + 8),
                                dict(max_len=-1), dict(max_prefix=-1), dict(max_len=129), dict(max_prefix=129), dict(table=None),
                                dict(len=None), dict(prefix_table=None), dict(prefix_len=None), dict(scale=float("inf")),
                                dict(scale=float("nan"))])
def test_attention(qmh, kw):
    L = qmh.load_library()
    a = attention_args(qmh, **kw)
    assert L.qmh_paged_attention_ws(ctypes.byref(a)) == 0
    refused(qmh, L.qmh_paged_attention(ctypes.byref(a), P, 1 << 40, None), "paged_attention")


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(n_groups=-1), dict(n_groups=65536), dict(n_beams=0), dict(n_beams=65), dict(n_out=0), dict(n_out=65),
                                dict(vocab=0), dict(vocab=(1 << 24) + 1, stride=1 << 25), dict(logits=None), dict(logits=P + 2),
                                dict(stride=99), dict(score=None), dict(out_score=None), dict(out_parent=None), dict(out_token=None),
                                dict(out_score=P), dict(done=P, eos=-1), dict(done=P, eos=100)])
def test_select(qmh, kw):
    L = qmh.load_library()
    a = beam_args(qmh, **kw)
    assert L.qmh_beam_select_ws(ctypes.byref(a)) == 0
    refused(qmh, L.qmh_beam_select(ctypes.byref(a), P, 1 << 40, None), "beam_select")


@pytest.mark.parametrize("kw", [dict(n_outer=-1), dict(n_rows=-1), dict(live=-1), dict(row_stride=-1), dict(seq_stride=-1), dict(outer_stride=-1),
                                dict(row_stride=63), dict(seq_stride=1 << 50)])
def test_reorder(qmh, kw):
    d = dict(n_outer=2, outer_stride=1 << 16, seq_stride=1 << 12, n_rows=4, row_stride=128, live=64)
    d.update(kw)
    s = qmh.BeamState(**d)
    refused(qmh, qmh.load_library().qmh_beam_reorder(ctypes.byref(s), P, P, P, 2, 4, None), "beam_reorder")


@pytest.mark.parametrize("kw", [dict(seq_stride=63), dict(outer_stride=63)])
def test_reorder_overlapping_states(qmh, kw):
    d = dict(n_outer=2, outer_stride=1 << 16, seq_stride=1 << 12, n_rows=1, row_stride=128, live=64)
    d.update(kw)
    refused(qmh, qmh.load_library().qmh_beam_reorder(ctypes.byref(qmh.BeamState(**d)), P, P, P, 1, 4, None), "beam_reorder")


def test_most_tokens_and_positions(qmh):
    refused(qmh, append(qmh, n_tokens=(1 << 24) + 1), "paged_append")
    p = pages(qmh)
    refused(qmh, qmh.load_library().qmh_paged_reorder(ctypes.byref(p), P, 1 << 27, P, (1 << 30) + 1, P, 2, 2, None), "paged_reorder")


def test_reorder_arguments(qmh):
    L = qmh.load_library()
    s = qmh.BeamState(n_outer=1, outer_stride=0, seq_stride=64, n_rows=1, row_stride=64, live=64)
    for args in ((None, P, P, P, 2, 4), (ctypes.byref(s), None, P, P, 2, 4), (ctypes.byref(s), P, None, P, 2, 4), (ctypes.byref(s), P, P, None, 2, 4),
                 (ctypes.byref(s), P, P, P, -1, 4), (ctypes.byref(s), P, P, P, 65536, 4), (ctypes.byref(s), P, P, P, 2, 0), (ctypes.byref(s), P, P, P, 2, 65)):
        refused(qmh, L.qmh_beam_reorder(*args, None), "beam_reorder")
    p = pages(qmh)
    for args in ((None, 4, P, 60, P, 2, 2), (P, 4, None, 60, P, 2, 2), (P, 4, P, 65, P, 2, 2), (P, 4, P, -1, P, 2, 2), (P, 4, P, 60, None, 2, 2),
                 (P, 4, P, 60, P, 2, 65)):
        refused(qmh, L.qmh_paged_reorder(ctypes.byref(p), *args, None), "paged_reorder")


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=258), dict(max_pos=0), dict(max_pos=(1 << 24) + 1), dict(theta=1.0),
                                dict(theta=float("nan")), dict(magnitude=float("inf")), dict(scaling="linear", factor=0.0),
                                dict(scaling="ntk", rot_dim=2, factor=2.0), dict(scaling="bands", factor=2.0, low=4.0, high=4.0),
                                dict(scaling="yarn", factor=2.0, low=0.0), dict(scaling="yarn", factor=2.0, first_len=0)])
def test_rotary(qmh, kw):
    d = dict(rot_dim=64)
    d.update(kw)
    with pytest.raises(qmh.QmhError, match="rotary"):
        qmh.Rotary(**d)


def test_null_arguments(qmh):
    L = qmh.load_library()
    refused(qmh, L.qmh_paged_append(None, None), "paged_append")
    refused(qmh, L.qmh_paged_attention(None, None, 0, None), "paged_attention")
    refused(qmh, L.qmh_beam_select(None, None, 0, None), "beam_select")
    assert L.qmh_paged_attention_ws(None) == 0 and L.qmh_beam_select_ws(None) == 0
    assert not L.qmh_rotary_create(None)
    L.qmh_rotary_free(None)
