"""What the ops for drafted trees refuse: every bad argument is an error code with a message that names the op, before anything
reaches a device."""
import ctypes

import pytest

import _ops as o
from test_paged_refusals import BAD_PAGES, P, attention_args, pages, refused


def plan_args(q, **kw):
    d = dict(n_seq=4, page_size=16, table=P, table_stride=8, len=P, keep=P, add=P, free_pages=P, free_size=100, free_state=P, n_tokens=64, first=P,
             seq=P, slot=P, pos=P)
    d.update(kw)
    return q.PlanArgs(**d)


def tree_args(q, base=None, pg=None, **kw):
    d = dict(n_rows=64, first=P, mask=P, mask_stride=0, mask_words=1)
    d.update(kw)
    return q.TreeArgs(base=attention_args(q, pg, **{"q_len": 16, **(base or {})}), **d)


def logits_args(q, **kw):
    d = dict(dtype=o.F32, n_rows=8, vocab=100, logits=P, stride=100, out=2 * P, out_stride=100, best=P, n_seq=2, rows_per_seq=4, history=P,
             history_stride=10, history_len=P, bias_token=P, bias=P, bias_len=P, bias_stride=5, allow=P, allow_stride=4, n_allow=8, node_token=P,
             node_stride=4, mask=P, mask_stride=4, mask_words=1)
    d.update(kw)
    return q.LogitsArgs(**d)


def accept_args(q, pg=None, **kw):
    d = dict(n_seq=4, tree_size=16, parent=P, parent_stride=16, token=P, token_stride=16, n_rows=64, choice=P, len=P, count=2 * P, path=P, next=3 * P,
             keep=4 * P, history=P, history_stride=10, history_len=P, n_layers=2, layer_stride=8 * 2 * 16 * 64, table=P, table_stride=4)
    d.update(kw)
    a = q.AcceptArgs(**d)
    if pg is not False:
        a.pages = ctypes.pointer(pages(q, **(pg or {})))
    return a


@pytest.mark.parametrize("kw", [
    dict(n_seq=-1), dict(n_seq=65536), dict(page_size=8), dict(page_size=48), dict(page_size=2048), dict(page_size=0), dict(table=None), dict(len=None),
    dict(free_pages=None), dict(free_state=None), dict(table_stride=0), dict(table_stride=1 << 29), dict(table_stride=1 << 27), dict(free_size=0),
    dict(free_size=(1 << 30) + 1), dict(n_tokens=-1), dict(n_tokens=(1 << 24) + 1), dict(first=None), dict(seq=None), dict(slot=None), dict(pos=None),
    dict(parent=P, tree_size=0), dict(parent=P, tree_size=1025), dict(parent=P, tree_size=8, parent_stride=7), dict(mask=P),
    dict(parent=P, tree_size=8, n_tokens=0)])
def test_plan(qmh, kw):
    L, a = qmh.load_library(), plan_args(qmh, **kw)
    assert L.qmh_paged_plan_ws(ctypes.byref(a)) == 0
    refused(qmh, L.qmh_paged_plan(ctypes.byref(a), P, 1 << 40, None), "paged_plan")


@pytest.mark.parametrize("pg", BAD_PAGES)
def test_pages(qmh, pg):
    L = qmh.load_library()
    a = tree_args(qmh, pg=pg)
    assert L.qmh_tree_attention_ws(ctypes.byref(a)) == 0
    refused(qmh, L.qmh_tree_attention(ctypes.byref(a), P, 1 << 40, None), "tree_attention")
    refused(qmh, L.qmh_tree_accept(ctypes.byref(accept_args(qmh, pg)), None), "tree_accept")


@pytest.mark.parametrize("kw", [
    dict(base=dict(n_heads=3)), dict(base=dict(q=None)), dict(base=dict(scale=float("nan"))), dict(base=dict(max_len=129)), dict(base=dict(n_groups=3)),
    dict(n_rows=-1), dict(n_rows=(1 << 20) + 1), dict(first=None, n_rows=63), dict(mask_words=0), dict(base=dict(q_len=33)), dict(mask=P + 2),
    dict(mask_stride=15), dict(mask_stride=-16), dict(mask_stride=1 << 50), dict(mask_words=1 << 28)])
def test_attention(qmh, kw):
    L, a = qmh.load_library(), tree_args(qmh, **kw)
    assert L.qmh_tree_attention_ws(ctypes.byref(a)) == 0
    refused(qmh, L.qmh_tree_attention(ctypes.byref(a), P, 1 << 40, None), "tree_attention")


@pytest.mark.parametrize("kw", [
    dict(dtype=2), dict(dtype=9), dict(n_rows=-1), dict(n_rows=(1 << 20) + 1), dict(vocab=0), dict(vocab=(1 << 24) + 1, stride=1 << 25, out_stride=1 << 25),
    dict(n_seq=-1), dict(n_seq=65536, first=P), dict(rows_per_seq=0), dict(rows_per_seq=5), dict(logits=None), dict(logits=P + 2), dict(stride=99),
    dict(out=None, best=None), dict(out_stride=99), dict(out=P + 1), dict(out=P, out_stride=101), dict(history_len=None), dict(history_stride=0),
    dict(history_stride=(1 << 24) + 1), dict(bias_token=None), dict(bias_len=None), dict(bias_stride=0), dict(allow=P + 2), dict(allow_stride=3),
    dict(n_allow=7), dict(allow_row=P, n_allow=-1), dict(node_stride=3), dict(mask_words=0), dict(mask_stride=3), dict(mask=P + 1),
    dict(rows_per_seq=1025, first=P, node_stride=2000, mask_words=40)])
def test_logits(qmh, kw):
    L, a = qmh.load_library(), logits_args(qmh, **kw)
    assert L.qmh_logits_edit_ws(ctypes.byref(a)) == 0
    refused(qmh, L.qmh_logits_edit(ctypes.byref(a), P, 1 << 40, None), "logits_edit")


@pytest.mark.parametrize("kw", [
    dict(n_seq=-1), dict(n_seq=65536), dict(tree_size=0), dict(tree_size=1025), dict(parent=None), dict(token=None), dict(choice=None), dict(len=None),
    dict(parent_stride=15), dict(token_stride=15), dict(parent_stride=-1), dict(n_rows=-1), dict(n_rows=63), dict(n_rows=(1 << 20) + 1),
    dict(count=None), dict(next=None), dict(keep=None), dict(keep=P), dict(next=P), dict(count=P), dict(count=3 * P), dict(count=4 * P), dict(next=4 * P),
    dict(history_len=None), dict(history_stride=0), dict(n_layers=0), dict(n_layers=1025), dict(layer_stride=16383), dict(layer_stride=16388),
    dict(layer_stride=1 << 50), dict(table=None), dict(table_stride=0), dict(table_stride=1 << 28)])
def test_accept(qmh, kw):
    refused(qmh, qmh.load_library().qmh_tree_accept(ctypes.byref(accept_args(qmh, **kw)), None), "tree_accept")


def test_null_arguments(qmh):
    L = qmh.load_library()
    refused(qmh, L.qmh_paged_plan(None, None, 0, None), "paged_plan")
    refused(qmh, L.qmh_tree_attention(None, None, 0, None), "tree_attention")
    refused(qmh, L.qmh_logits_edit(None, None, 0, None), "logits_edit")
    refused(qmh, L.qmh_tree_accept(None, None), "tree_accept")
    assert L.qmh_paged_plan_ws(None) == L.qmh_tree_attention_ws(None) == L.qmh_logits_edit_ws(None) == 0


def test_structures_are_the_headers(qmh, tmp_path):
    """The binding's structures have the header's sizes and offsets."""
    import subprocess
    names = {"qmh_plan_args": qmh.PlanArgs, "qmh_tree_args": qmh.TreeArgs, "qmh_logits_args": qmh.LogitsArgs, "qmh_accept_args": qmh.AcceptArgs}
    lines = ['#include <stdio.h>', f'#include "{qmh.INCLUDE}"', "int main(void) {"]
    for n, c in names.items():
        lines.append(f'printf("%zu", sizeof({n}));')
        lines += [f'printf(" %zu", offsetof({n}, {f[0]}));' for f in c._fields_] + ['printf("\\n");']
    src = tmp_path / "s.c"
    src.write_text("\n".join(lines) + "return 0; }")
    subprocess.run(["gcc", "-o", str(tmp_path / "s"), str(src)], check=True)
    got = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split("\n")
    for line, c in zip(got, names.values()):
        assert [int(x) for x in line.split()] == [ctypes.sizeof(c)] + [getattr(c, f[0]).offset for f in c._fields_]
