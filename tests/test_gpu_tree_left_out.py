"""Sequences of a shared prefix beside one that is left out (qmh_tree_attention): those with good rows of their own have their results,
whatever the workspace held, also where prefix and own pages are joined from parts."""
import ctypes

import numpy as np
import pytest

import _ops as o
import _trees as tr

pytestmark = pytest.mark.gpu

Q, ROWS = 5, 16  # the most nodes of a sequence, rows of q and out


def run(q, dt, H, KV, hd, first, own, prefix, groups=1, Q=Q, ROWS=ROWS, static=False):
    """Outputs and tolerance-checked rows of the good sequences; bytes of the others' rows are anything."""
    rs, ps, B = np.random.default_rng(hd + len(first)), 16, len(own)
    tables, n_pages = o.make_tables(rs, [-(-n // ps) for n in prefix + own], -(-max(prefix + own) // ps) + 1)
    k, v = (o.encode(rs.standard_normal((n_pages, KV, ps, hd)), dt) for _ in range(2))
    x = o.encode(rs.standard_normal((ROWS, H * hd)) * 1.5, dt)
    see = [tr.ancestors(tr.tree(rs, Q)) for _ in range(1 if static else B)]
    words = -(-Q // 32)
    dk, dv, dx, out = o.Guarded(q, k), o.Guarded(q, v), o.Guarded(q, x), o.Guarded(q, np.full((ROWS, H * hd), 0x55, o.raw(dt)))
    dev = q.DeviceBuffer.from_array
    tab, ptab, n, pn, at, mask = (dev(np.ascontiguousarray(y)) for y in (
        tables[groups:], tables[:groups], np.array(own, np.int32), np.array(prefix, np.int32), np.array(first, np.int32), tr.pack(np.array(see), words)))
    pages = q.Pages(dtype=dt, n_kv_heads=KV, head_dim=hd, page_size=ps, n_pages=n_pages, k=dk.ptr, v=dv.ptr)
    scale = float(np.float32(hd ** -0.5))
    base = q.AttentionArgs(pages=ctypes.pointer(pages), n_heads=H, n_seq=B, q_len=Q, n_groups=groups, q=dx.ptr, q_stride=H * hd, out=out.ptr,
                           out_stride=H * hd, table=tab.ptr, len=n.ptr, table_stride=tables.shape[1], max_len=max(own), prefix_table=ptab.ptr,
                           prefix_len=pn.ptr, prefix_stride=tables.shape[1], max_prefix=max(prefix + [0]), scale=scale)
    a = q.TreeArgs(base=base, n_rows=ROWS, first=at.ptr, mask=mask.ptr, mask_stride=0 if static else Q * words, mask_words=words)
    L = q.load_library()
    need = L.qmh_tree_attention_ws(ctypes.byref(a))
    ws = o.Guarded(q, np.full(max(need, 16), 0xFF, np.uint8))
    q._check(L.qmh_tree_attention(ctypes.byref(a), ws.ptr, need, None), "tree_attention")
    q.sync()
    ws.get()
    full = out.get()
    got, xv = o.decode(full, dt).reshape(ROWS, H, hd), o.decode(x, dt).reshape(ROWS, H, hd)
    kv = [o.decode(y, dt) for y in (k, v)]
    good = 0
    for i in range(B):
        a0, a1 = first[i], first[i + 1]
        if a0 < 0 or a1 > ROWS or a1 < a0 or a1 - a0 > Q:
            continue
        pk, pv = (o.rows_of(y, tables[i // (B // groups)], prefix[i // (B // groups)], ps) for y in kv)
        ok, ov = (o.rows_of(y, tables[groups + i], own[i], ps) for y in kv)
        for j in range(a1 - a0):
            t = np.concatenate([np.ones(own[i] - (a1 - a0), bool), see[0 if static else i][j, :a1 - a0]])
            kk, ww = np.concatenate([pk, ok[t]]), np.concatenate([pv, ov[t]])
            want, mag, reach = o.attention(xv[a0 + j], kk, ww, scale)
            # scores of hd products, exponentials to 2 steps, sums of n terms, 16-bit probabilities rounded to the type, then the result
            tol = mag * (2 * ((hd + 4) * o.U32 * reach + 4 * o.U32) + (len(kk) + 64) * o.U32 + (o.HALF[dt] if dt != o.F32 else 0)) * 1.01
            tol = tol + o.HALF[dt] * np.abs(want) + o.TINY[dt] * (1 + len(kk) * np.abs(ww).max())
            o.close(got[a0 + j], want, tol, f"sequence {i} node {j}, workspace {need}")
            good += 1
    nobody = [r for r in range(ROWS) if r < first[0] or r >= first[-1]]
    assert (full[nobody] == 0x55).all(), "rows that are nobody's"
    return need, good


# the last one ends past the arrays, the first one starts before them, one has more nodes than a sequence may, one's end is beyond any
# array; good ones beside them in each group
FIRSTS = [[0, 4, 9, 30], [-3, 4, 9, 12], [0, 10, 12, 16], [0, 4, 14, 16], [0, 3, 5, 2 ** 31 - 1], [-2 ** 31, 1, 6, 8]]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("first", FIRSTS)
def test_good_sequences_beside_one_that_is_left_out(gpu, dtype, first):
    dt = o.TYPES[dtype]
    # in parts, joined from the workspace; and short enough for one pass without
    need, good = run(gpu, dt, 4, 2, 64, first, [700, 300, 90], [900])
    assert need > 0 and good >= 2
    need, good = run(gpu, dt, 4, 2, 64, first, [40, 30, 20], [50])
    assert need == 0 and good >= 2


@pytest.mark.parametrize("H,KV,hd", [(24, 2, 64), (16, 1, 128), (8, 1, 256)])
def test_more_rows_than_the_prefix_has_tiles_for(gpu, H, KV, hd):
    """A group whose left-out sequence has more rows than all of the group may have: its good one's rows lie behind them."""
    need, good = run(gpu, o.F32, H, KV, hd, [0, 14, 16], [300, 600], [900])
    assert need > 0 and good == 2
    need, good = run(gpu, o.BF16, H, KV, hd, [0, 2, 4, 13, 16], [600, 300, 300, 600], [900, 1100], groups=2)
    assert need > 0 and good == 7


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 70, 600])
def test_few_rows_of_many_sequences(gpu, dtype, prefix):
    """1100 sequences of up to 1000 nodes, of which a few have some: the rows there are count, not the product."""
    counts = np.zeros(1100, int)
    counts[[0, 3, 500, 501, 777, 1099]] = [1, 40, 7, 3, 180, 69]
    first = [0, *np.cumsum(counts).tolist()]
    need, good = run(gpu, o.TYPES[dtype], 8, 2, 32, first, [int(n) + 9 for n in counts], [prefix] * 11, groups=11, Q=1000, ROWS=300, static=True)
    assert good == 300
