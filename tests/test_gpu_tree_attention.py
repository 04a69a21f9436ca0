"""Attention of drafted trees over pages (qmh_tree_attention) against a statement in 64 bits: heads, node counts, contexts that end
anywhere in a step, masks of any kind, values that are not finite where they are not seen, bad lengths and rows."""
import ctypes

import numpy as np
import pytest

import _ops as o
import _trees as tr

pytestmark = pytest.mark.gpu


def run(q, dt, H, KV, hd, ps, groups, nodes, own, prefix=None, q_len=None, ragged=True, masks="tree", static=False, seed=0, scale=None, pad=0,
        extra_words=0, spoil=None, touch=None, gap=0, more=0, check=True):
    """nodes, own: of each sequence, own with its nodes. Returns the outputs [rows, H, hd] and where each sequence's start."""
    rs = np.random.default_rng(seed)
    B, per = len(nodes), len(nodes) // groups
    prefix = prefix or [0] * groups
    q_len = q_len or max(max(nodes), 1)
    scale = float(np.float32(hd ** -0.5 if scale is None else scale))
    counts = [-(-max(n, 0) // ps) for n in prefix] + [-(-max(n, 0) // ps) for n in own]
    tables, n_pages = o.make_tables(rs, counts, max(counts) + 1)
    pool = [rs.standard_normal((n_pages, KV, ps, hd)) for _ in range(2)]
    first = tr.starts(nodes) + gap
    rows = (int(first[-1]) + 3) if ragged else B * q_len + more
    if not ragged:
        assert all(n == q_len for n in nodes)
    x = o.encode(rs.standard_normal((rows, H * hd + pad)) * 1.5, dt)
    words = -(-q_len // 32) + extra_words
    see = np.zeros((B, q_len, q_len), bool)
    for i in range(1 if static else B):
        if masks == "tree":
            see[i] = tr.ancestors(tr.tree(rs, q_len))
        elif masks == "chain":
            see[i] = np.tril(np.ones((q_len, q_len), bool))
        elif masks == "random":
            see[i] = rs.random((q_len, q_len)) < 0.4
        elif masks == "none":
            see[i] = False
    if static:
        see[:] = see[0]
    packed = tr.pack(see[:1] if static else see, words, rs)
    if touch:
        touch(pool, tables[groups:], own, nodes, see)
    k, v = (o.encode(y, dt) for y in pool)
    prefix, own, bad = list(prefix), list(own), np.zeros(B, bool)
    if spoil:
        spoil(tables[groups:], own, first, bad)
    dk, dv, dx, dout = o.Guarded(q, k), o.Guarded(q, v), o.Guarded(q, x), o.Guarded(q, np.full((rows, H * hd + pad), 0x55, o.raw(dt)))
    dev = q.DeviceBuffer.from_array
    keep = [dev(a) for a in (tables[groups:], np.array(own, np.int32), tables[:groups], np.array(prefix, np.int32), first, packed)]
    pages = q.Pages(dtype=dt, n_kv_heads=KV, head_dim=hd, page_size=ps, n_pages=n_pages, k=dk.ptr, v=dv.ptr)
    cap = tables.shape[1] * ps
    base = q.AttentionArgs(pages=ctypes.pointer(pages), n_heads=H, n_seq=B, q_len=q_len, n_groups=groups, q=dx.ptr, q_stride=H * hd + pad,
                           out=dout.ptr, out_stride=H * hd + pad, table=keep[0].ptr, len=keep[1].ptr, table_stride=tables.shape[1],
                           max_len=min(max(max(own), 0), cap), prefix_table=keep[2].ptr, prefix_len=keep[3].ptr, prefix_stride=tables.shape[1],
                           max_prefix=max(prefix), scale=scale)
    a = q.TreeArgs(base=base, n_rows=rows, first=keep[4].ptr if ragged else None, mask=None if masks == "chain" else keep[5].ptr,
                   mask_stride=0 if static else q_len * words, mask_words=words)
    L = q.load_library()
    need = L.qmh_tree_attention_ws(ctypes.byref(a))
    ws = o.Guarded(q, np.zeros(max(need, 16), np.uint8), pad=4096)
    q._check(L.qmh_tree_attention(ctypes.byref(a), ws.ptr, need, None), "tree_attention")
    q.sync()
    ws.get()
    full = dout.get()
    for d in (dk, dv, dx):
        assert d.get().tobytes() == d.like.tobytes()
    if pad:
        assert (full[:, H * hd:] == 0x55).all()
    got = o.decode(full[:, :H * hd], dt).reshape(rows, H, hd)
    if not check:
        return got, first
    xv = o.decode(x, dt)[:, :H * hd].reshape(rows, H, hd)
    kv_, vv = o.decode(k, dt), o.decode(v, dt)
    at = first if ragged else np.arange(B + 1) * q_len
    untouched = full[:, :H * hd] == 0x55
    assert untouched[:at[0]].all() and untouched[at[-1]:].all(), "rows that are nobody's"
    for i, n in enumerate(nodes):
        g = i // per
        if bad[i]:
            assert np.isnan(got[at[i]:at[i] + n]).all(), f"sequence {i}: NaN"
            continue
        pk, pv = (o.rows_of(y, tables[g], prefix[g], ps) for y in (kv_, vv))
        ok, ov = (o.rows_of(y, tables[groups + i], own[i], ps) for y in (kv_, vv))
        for j in range(n):
            t = np.concatenate([np.ones(own[i] - n, bool), see[i, j, :n]])
            kk, ww = np.concatenate([pk, ok[t]]), np.concatenate([pv, ov[t]])
            want, mag, reach = o.attention(xv[at[i] + j], kk, ww, scale)
            # as for consecutive queries: scores of hd products, exponentials to 2 steps, sums of n terms, 16-bit
            # probabilities rounded to the type, then the result
            ds = (hd + 4) * o.U32 * reach + 4 * o.U32
            with np.errstate(invalid="ignore"):
                tol = mag * (2 * ds + (len(kk) + 64) * o.U32 + (o.HALF[dt] if dt != o.F32 else 0)) * 1.01
                tol = tol + o.HALF[dt] * np.abs(want) + o.TINY[dt]
                if dt == o.F16:
                    tol = tol + len(kk) * o.TINY[dt] * np.abs(np.nan_to_num(ww, posinf=0, neginf=0)).max(initial=0)
            row = got[at[i] + j]
            if dt != o.F16 and len(ww) and np.nan_to_num(np.abs(ww), nan=0, posinf=0).max() > 2.0 ** 112:
                # weights are up to 2^15 before they are divided by their sum: 2^15 times such a value passes 32 bits (2^128)
                assert (np.isfinite(row) | (np.sign(row) == np.sign(want))).all()
                row = np.where(np.isfinite(row), row, want)
            o.close(row, want, tol, f"sequence {i} node {j} of {n} ({own[i]} own, {prefix[g]} shared)")
    return got, at


SHAPES = [(6, 2, 48), (12, 12, 64), (32, 4, 64), (3, 3, 128), (5, 1, 80), (14, 2, 96), (2, 1, 8), (4, 2, 256), (1, 1, 136), (40, 1, 32)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", SHAPES)
def test_heads(gpu, dtype, H, KV, hd):
    run(gpu, o.TYPES[dtype], H, KV, hd, 16, 2, [5, 1, 9, 7, 0, 12], [70, 33, 9, 40, 5, 13], prefix=[40, 7], seed=hd)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 17, 31, 32, 33, 63, 64, 65, 100, 129])
def test_node_counts(gpu, dtype, n):
    run(gpu, o.TYPES[dtype], 4, 2, 64, 32, 3, [n, n, n], [n, n + 1, n + 200], ragged=False, seed=n)
    run(gpu, o.TYPES[dtype], 2, 2, 128, 16, 1, [n, max(n // 2, 1), n - 1], [n + 45, n + 30, n + 7], seed=n)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("masks", ["tree", "random"])
def test_contexts_that_end_anywhere(gpu, dtype, masks):
    nodes = [1 + (7 * c) % 40 for c in range(48)]
    run(gpu, o.TYPES[dtype], 2, 1, 32, 16, 48, nodes, [c + n for c, n in zip(range(48), nodes)], q_len=45, masks=masks, extra_words=1, seed=5)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups,nodes,own,prefix", [
    (1, [3], [3], [0]), (1, [3], [1000], [1500]), (2, [33, 20, 40, 1], [50, 2000, 900, 1], [700, 0]), (1, [70], [3100], [0]),
    (1, [8] * 20, list(range(8, 28)), [513])])
def test_lengths(gpu, dtype, groups, nodes, own, prefix):
    run(gpu, o.TYPES[dtype], 8, 2, 64, 64, groups, nodes, own, prefix=prefix, pad=64, seed=len(nodes))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_long_tree(gpu, dtype):
    run(gpu, o.TYPES[dtype], 2, 1, 64, 16, 1, [1000], [1100], seed=3)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("static", [False, True])
def test_masks_of_any_kind(gpu, dtype, static):
    for masks in ("random", "tree", "chain"):
        run(gpu, o.TYPES[dtype], 4, 2, 64, 16, 2, [37, 40, 1, 12], [37, 90, 64, 12], prefix=[0, 33], q_len=40, masks=masks, static=static, seed=9)
    # nothing of the tree is seen: the context alone, or zeros
    got, at = run(gpu, o.TYPES[dtype], 4, 2, 64, 16, 2, [37, 3], [37, 50], masks="none", static=static, seed=10)
    assert (got[:37] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_what_is_not_seen_has_no_effect(gpu, dtype, hd):
    """Keys and values of some nodes are infinite or NaN: other branches of the tree do not notice."""
    for value in (np.inf, -np.inf, np.nan):
        for where in (0, 1):
            def touch(pool, table, own, nodes, see):
                for i, n in enumerate(nodes):
                    for k in range(3, n, 5):
                        t = own[i] - n + k
                        pool[where][table[i][t // 16], :, t % 16, (3 * k) % hd] = value
            run(gpu, o.TYPES[dtype], 2, 1, hd, 16, 1, [36, 9], [70, 9], touch=touch, seed=hd)
    # the same in pieces of a long context, trees over a piece's end; and where the context has such values, too, which all see
    for ctx in (False, True):
        def long(pool, table, own, nodes, see):
            for i, n in enumerate(nodes):
                for k in [*range(3, n, 5)] + ([-7 - n] if ctx else []):
                    t = own[i] - n + k
                    pool[1][table[i][t // 16], :, t % 16, (3 * abs(k)) % hd] = [np.inf, np.nan][(k + ctx) % 2]
        run(gpu, o.TYPES[dtype], 2, 1, hd, 16, 2, [36, 100], [1304, 1100], prefix=[0, 0], touch=long, seed=hd + 1)
        run(gpu, o.TYPES[dtype], 2, 1, hd, 16, 1, [36, 20], [700, 1100], prefix=[600], touch=long, masks="chain", seed=hd + 2)
    # the type's largest numbers are finite
    big = {"f32": 3e38, "f16": 65504.0, "bf16": 3e38}[dtype]

    def large(pool, table, own, nodes, see):
        t = own[0] - nodes[0] + 2
        pool[1][table[0][t // 16], :, t % 16] = -big
    run(gpu, o.TYPES[dtype], 2, 1, hd, 16, 1, [20], [60], touch=large, seed=1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bad_lengths_and_pages_give_nan(gpu, dtype):
    def spoil(table, own, first, bad):
        own[0], own[1] = 4, -7  # fewer than the nodes
        table[2, 0] = -5
        bad[:3] = True
    run(gpu, o.TYPES[dtype], 4, 2, 64, 16, 5, [5, 5, 5, 5, 5], [20, 20, 20, 20, 20], spoil=spoil, seed=4)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_a_bad_page_of_nodes_beside_values_that_are_not_finite(gpu, dtype):
    """Chains over two pages: rows that see the second one, which is none, are NaN, whatever the first one holds."""
    def touch(pool, table, own, nodes, see):
        pool[1][table[0][2], :, 4, 3] = np.inf  # node 4, at position 36

    def spoil(table, own, first, bad):
        table[0, 3] = -1  # positions 48 on: nodes 16 on
    got, at = run(gpu, o.TYPES[dtype], 2, 1, 64, 16, 2, [20, 20], [52, 52], masks="chain", touch=touch, spoil=spoil, check=False, seed=2)
    assert np.isnan(got[16:20]).all()
    assert np.isfinite(got[20:40]).all()


def test_pages_past_4_gib(gpu):
    """Nodes and context in pages that lie more than 4 GiB into the pools, and a path moved between them."""
    q, L, KV, hd, ps = gpu, gpu.load_library(), 16, 256, 1024
    page = KV * ps * hd * 2  # 8 MiB
    n_pages = 1100
    pool = [q.DeviceBuffer(n_pages * page) for _ in range(2)]
    rs = np.random.default_rng(0)
    table = np.array([[1099, 1050]], np.int32)
    own, n = 1024 + 6, 9  # nodes 0 to 2 in the first page, the others in the second
    kv = [o.encode(rs.standard_normal((own, KV, hd)), o.F16) for _ in range(2)]
    for b, x in zip(pool, kv):
        for p in range(2):
            rows = x[p * ps:(p + 1) * ps]
            for h in range(KV):
                part = np.ascontiguousarray(rows[:, h])
                q._check(L.qmh_memcpy_h2d(b.ptr + int(table[0, p]) * page + h * ps * hd * 2, part.ctypes.data, part.nbytes), "rows")
    x = o.encode(rs.standard_normal((n, KV * hd)), o.F16)
    parent = tr.tree(rs, n)
    parent[5] = 2
    see = tr.ancestors(parent)
    dev = q.DeviceBuffer.from_array
    dx, out, tab, length, mask = dev(x), q.DeviceBuffer(x.nbytes), dev(table), dev(np.array([own], np.int32)), dev(tr.pack(see, 1))
    pages = q.Pages(dtype=o.F16, n_kv_heads=KV, head_dim=hd, page_size=ps, n_pages=n_pages, k=pool[0].ptr, v=pool[1].ptr)
    base = q.AttentionArgs(pages=ctypes.pointer(pages), n_heads=KV, n_seq=1, q_len=n, n_groups=1, q=dx.ptr, q_stride=KV * hd, out=out.ptr,
                           out_stride=KV * hd, table=tab.ptr, len=length.ptr, table_stride=2, max_len=own, scale=0.0625)
    a = q.TreeArgs(base=base, n_rows=n, mask=mask.ptr, mask_words=1)
    need = L.qmh_tree_attention_ws(ctypes.byref(a))
    ws = q.DeviceBuffer(max(need, 16))
    q._check(L.qmh_tree_attention(ctypes.byref(a), ws.ptr, need, None), "attention")
    q.sync()
    got = o.decode(out.to_array(np.uint16), o.F16).reshape(n, KV, hd)
    k, v = (o.decode(y, o.F16) for y in kv)
    for j in range(n):
        t = np.concatenate([np.ones(own - n, bool), see[j]])
        want, mag, reach = o.attention(o.decode(x[j], o.F16).reshape(KV, hd), k[t], v[t], 0.0625)
        tol = mag * (2 * ((hd + 4) * o.U32 * reach + 4 * o.U32) + (own + 64) * o.U32 + o.HALF[o.F16]) * 1.01 + o.HALF[o.F16] * np.abs(want)
        o.close(got[j], want, tol + own * o.TINY[o.F16] * np.abs(v).max(), f"node {j}")
    # the path 0, 2, 5 ...: node 5 (second page) moves to position 2 of the tree (first page)
    token, choice = np.arange(n, dtype=np.int32), np.full(n, -1, np.int32)
    parent[2] = 0
    choice[0], choice[2] = 2, 5
    d = {m: dev(y) for m, y in dict(parent=parent, token=token, choice=choice, count=np.zeros(1, np.int32), next=np.zeros(1, np.int32),
                                    keep=np.zeros(1, np.int32)).items()}
    a = q.AcceptArgs(n_seq=1, tree_size=n, parent=d["parent"].ptr, parent_stride=n, token=d["token"].ptr, token_stride=n, n_rows=n,
                     choice=d["choice"].ptr, len=length.ptr, count=d["count"].ptr, next=d["next"].ptr, keep=d["keep"].ptr,
                     pages=ctypes.pointer(pages), n_layers=1, table=tab.ptr, table_stride=2)
    q._check(L.qmh_tree_accept(ctypes.byref(a), None), "accept")
    q.sync()
    assert d["count"].to_array(np.int32)[0] == 3
    begin = own - n
    for b, y in zip(pool, kv):
        for h in (0, KV - 1):
            row = np.zeros(hd, np.uint16)
            for to, src in ((begin + 1, begin + 2), (begin + 2, begin + 5), (begin, begin)):
                q._check(L.qmh_memcpy_d2h(row.ctypes.data, b.ptr + int(table[0, to // ps]) * page + (h * ps + to % ps) * hd * 2, row.nbytes), "row")
                assert np.array_equal(row, y[src, h]), (to, src)


@pytest.mark.parametrize("first", [[0, 4, 3, 8], [0, 4, 40, 8], [-1, 4, 6, 8], [0, 7, 9, 2 ** 31 - 1], [2, 4, 6, 12]])
def test_bad_rows_are_left_out(gpu, first):
    """Rows that run backwards, behind the arrays or past the most nodes: nothing outside the arrays is touched (the guards of
    run), and sequences with good rows of their own have them."""
    def spoil(table, own, at, bad):
        at[:] = first
    got, _ = run(gpu, o.F32, 2, 2, 64, 16, 3, [4, 2, 2], [20, 20, 20], q_len=5, spoil=spoil, check=False, seed=6)
    assert got.shape[0] == 11


def test_rows_behind_the_last_sequence_without_first(gpu):
    run(gpu, o.F16, 4, 2, 64, 16, 2, [4, 4], [900, 20], ragged=False, more=6, seed=12)
    run(gpu, o.F32, 4, 2, 64, 16, 2, [4, 4], [9, 20], ragged=False, more=6, seed=12)


def test_rows_that_start_behind_others(gpu):
    run(gpu, o.F16, 4, 2, 64, 16, 1, [3, 0, 5], [300, 20, 5], prefix=[700], gap=4, seed=11)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd,q_len,own", [(4, 2, 64, 3, 300), (2, 2, 128, 1, 2000), (8, 1, 32, 20, 57)])
def test_a_chain_is_what_consecutive_queries_are(gpu, dtype, H, KV, hd, q_len, own):
    """With a chain for a mask, or with none, the result is that of qmh_paged_attention: the same sums, divided into parts in
    another way."""
    q, L, dt, rs = gpu, gpu.load_library(), o.TYPES[dtype], np.random.default_rng(3)
    tables, n_pages = o.make_tables(rs, [-(-own // 16)] * 2, -(-own // 16))
    hk, hv = (rs.standard_normal((n_pages, KV, 16, hd)) for _ in range(2))
    hx = rs.standard_normal((2 * q_len, H * hd))
    k, v, x = (q.DeviceBuffer.from_array(o.encode(y, dt)) for y in (hk, hv, hx))
    out = [q.DeviceBuffer(2 * q_len * H * hd * o.BYTES[dt]) for _ in range(2)]
    tab, n = q.DeviceBuffer.from_array(tables), q.DeviceBuffer.from_array(np.array([own, own - 1], np.int32))
    words = -(-q_len // 32)
    mask = q.DeviceBuffer.from_array(tr.pack(np.tril(np.ones((q_len, q_len), bool)), words))
    pages = q.Pages(dtype=dt, n_kv_heads=KV, head_dim=hd, page_size=16, n_pages=n_pages, k=k.ptr, v=v.ptr)
    base = q.AttentionArgs(pages=ctypes.pointer(pages), n_heads=H, n_seq=2, q_len=q_len, n_groups=2, q=x.ptr, q_stride=H * hd, out=out[0].ptr,
                           out_stride=H * hd, table=tab.ptr, len=n.ptr, table_stride=tables.shape[1], max_len=own, scale=0.2)
    need = L.qmh_paged_attention_ws(ctypes.byref(base))
    ws = q.DeviceBuffer(max(need, 16))
    q._check(L.qmh_paged_attention(ctypes.byref(base), ws.ptr, need, None), "paged")
    q.sync()
    want = o.decode(out[0].to_array(o.raw(dt)), dt)
    # either side's error, as in run: 16-bit weights and results are off by half a step each, 32-bit scores by hd + 4 roundings of
    # the largest sum of products, sums by a rounding a term; values are at most `top`
    top, reach = np.abs(hv).max() * 1.01, np.abs(hk).max() * np.abs(hx).max() * hd * 0.2
    tol = 2 * top * (2 * o.HALF[dt] + 2 * ((hd + 4) * o.U32 * reach + 4 * o.U32) + (own + 64) * o.U32)
    for m in (None, mask.ptr):
        base.out = out[1].ptr
        a = q.TreeArgs(base=base, n_rows=2 * q_len, mask=m, mask_words=words)
        need = L.qmh_tree_attention_ws(ctypes.byref(a))
        ws = q.DeviceBuffer(max(need, 16))
        q._check(L.qmh_tree_attention(ctypes.byref(a), ws.ptr, need, None), "tree")
        q.sync()
        o.close(o.decode(out[1].to_array(o.raw(dt)), dt), want, tol, f"mask {bool(m)}")
