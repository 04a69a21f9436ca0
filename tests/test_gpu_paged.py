"""qmh_paged_append, qmh_paged_attention and qmh_paged_reorder against 64-bit statements of the operators.

Tolerances come from the roundings the operators make: one to the result's type (half a step), 32-bit sums and
products before it, and for 16-bit attention the probabilities' rounding to that type. Every array has guard
bytes around it; what may not be read (rows behind a length, pages of nobody) holds NaN, and table entries
behind a sequence's last page lead outside the pool."""
import ctypes

import numpy as np
import pytest

import _ops as o

pytestmark = pytest.mark.gpu


def pages_of(q, dt, kv, hd, ps, n_pages, k, v):
    return q.Pages(dtype=dt, n_kv_heads=kv, head_dim=hd, page_size=ps, n_pages=n_pages, k=k, v=v)


# ------------------------------------------------------------------------------------- append

def run_append(q, dt, H, KV, hd, ps, n, layout="pairs", scaling="none", rot=None, gains=False, far=0, seqs=1, seed=0, shift=0,
               pad_stride=0, inplace=False, use_q=True, use_kv=True, use_pos=True, magnitude=1.0, max_pos=131072, drop=()):
    rs = np.random.default_rng(seed)
    rot = hd if rot is None else rot
    runs = [n // seqs + (i < n % seqs) for i in range(seqs)]
    start = rs.integers(0, 2 * ps, seqs)
    counts = [int(-(-(s + r) // ps)) for s, r in zip(start, runs)]
    table, n_pages = o.make_tables(rs, counts, max(counts) + 1)
    seq = np.repeat(np.arange(seqs), runs).astype(np.int32)
    slot = np.concatenate([np.arange(s, s + r) for s, r in zip(start, runs)]).astype(np.int32)
    pos = (slot + far).astype(np.int32)
    order = rs.permutation(n)  # tokens in any order
    seq, slot, pos = seq[order], slot[order], pos[order]
    width = (H + 2 * KV) * hd + pad_stride
    x = o.encode(rs.standard_normal((n, width)) * np.exp2(rs.integers(-3, 4, (n, 1))), dt)
    gq, gk = (1 + 0.2 * rs.standard_normal((2, hd))).astype(np.float32)
    pool_k, pool_v = (o.encode(rs.standard_normal((n_pages, KV, ps, hd)), dt) for _ in range(2))
    out0 = o.encode(rs.standard_normal((n, H * hd)), dt)
    seq_in, slot_in, pos_in = seq.copy(), slot.copy(), pos.copy()
    gone = np.zeros(n, bool)
    for i, (name, value) in enumerate(drop):  # tokens that name something outside its range
        t = (7 * i + 1) % n
        {"seq": seq_in, "slot": slot_in, "pos": pos_in}[name][t] = value
        gone[t] = True
    L = q.load_library()
    es = o.BYTES[dt]
    dx = o.Guarded(q, x, shift)
    dk, dv = o.Guarded(q, pool_k), o.Guarded(q, pool_v)
    dout = o.Guarded(q, out0, shift)
    dt_, ds, dl, dp = (o.Guarded(q, a) for a in (table, seq_in, slot_in, pos_in))
    dgq, dgk = o.Guarded(q, gq), o.Guarded(q, gk)
    p = pages_of(q, dt, KV, hd, ps, n_pages, dk.ptr if use_kv else None, dv.ptr if use_kv else None)
    a = q.AppendArgs(pages=ctypes.pointer(p), n_tokens=n, n_heads=H, eps=1e-5, n_seq=seqs)
    rotary = q.Rotary(rot, layout, scaling, max_pos, factor=8.0, low=1.0, high=32.0 if scaling == "yarn" else 4.0,
                      magnitude=magnitude) if rot else None
    a.rotary = rotary.handle if rotary else None
    if use_q:
        a.q, a.q_stride = dx.ptr, width
        a.q_out, a.q_out_stride = (dx.ptr, width) if inplace else (dout.ptr, H * hd)
    if use_kv:
        a.k, a.k_stride = dx.ptr + H * hd * es, width
        a.v, a.v_stride = dx.ptr + (H + KV) * hd * es, width
        a.table, a.table_stride, a.seq = dt_.ptr, table.shape[1], ds.ptr
    a.slot = dl.ptr
    a.pos = dp.ptr if use_pos else None
    if gains:
        a.q_gain, a.k_gain = dgq.ptr, dgk.ptr
    q._check(L.qmh_paged_append(ctypes.byref(a), None), "append")
    q.sync()
    got_x, got_out, got_k, got_v = dx.get(), dout.get(), dk.get(), dv.get()
    if rotary:
        rotary.close()

    # the operator in 64 bits
    xv = o.decode(x, dt)[:, :(H + 2 * KV) * hd].reshape(n, H + 2 * KV, hd)
    f = o.freqs(rot, scaling, high=32.0 if scaling == "yarn" else 4.0) if rot else np.zeros(0)
    eps = float(np.float32(1e-5))
    at = pos if use_pos else slot

    def one(y, g):
        z = o.norm(y, g.astype(np.float64), eps) if gains else y
        r = o.rotate(z, at, f, layout, float(np.float32(magnitude)))
        # relative to a pair's elements (the head's largest bounds both): the norm's sum of hd squares, its root,
        # quotient and two products; then for each of a turn's two terms the sine's or cosine's rounding (its angle's
        # 64-bit error below a tenth of one), the product's and the sum's
        rel = (hd + 8 if gains else 0) * o.U32 + 4 * o.U32
        tol = rel * 2 * abs(magnitude) * np.abs(z).max(-1, keepdims=True)
        return r, tol + o.HALF[dt] * np.abs(r) + o.TINY[dt]

    wq, tq = one(xv[:, :H], gq)
    wk, tk = one(xv[:, H:H + KV], gk)
    if use_q:
        got = got_x[:, :H * hd] if inplace else got_out
        before = x[:, :H * hd] if inplace else out0
        keep = ~gone
        o.close(o.decode(got[keep], dt), wq.reshape(n, -1)[keep], tq.reshape(n, -1)[keep], "queries")
        assert np.array_equal(got[gone], before[gone]), "queries of left-out tokens"
    if not inplace:
        assert np.array_equal(got_x, x)
    else:
        assert np.array_equal(got_x[:, H * hd:], x[:, H * hd:])
    if not use_q:
        assert np.array_equal(got_out, out0)
    if use_kv:
        want_v = pool_v.copy()
        seen = np.zeros((n_pages, ps), bool)
        for t in np.flatnonzero(~gone):
            page, off = table[seq[t], slot[t] // ps], slot[t] % ps
            seen[page, off] = True
            o.close(o.decode(got_k[page, :, off], dt), wk[t], tk[t], f"key {t}")
            want_v[page, :, off] = x[t, (H + KV) * hd:(H + 2 * KV) * hd].reshape(KV, hd)
        assert np.array_equal(got_v, want_v), "values"
        rest = ~seen[:, None, :, None] & np.ones_like(pool_k, bool)
        assert np.array_equal(got_k[rest], pool_k[rest]), "rows of nobody"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("H,KV,hd,rot,gains", [(6, 2, 48, 48, False), (32, 4, 64, 32, True), (5, 1, 80, 80, True), (3, 3, 128, 128, True),
                                               (2, 1, 256, 64, True), (1, 1, 8, 8, True), (7, 7, 24, 12, False), (4, 2, 40, 0, True),
                                               (2, 2, 248, 6, True), (3, 1, 136, 136, False)])
def test_append_shapes(gpu, dtype, layout, H, KV, hd, rot, gains):
    run_append(gpu, o.TYPES[dtype], H, KV, hd, 16, 13, layout, rot=rot, gains=gains, far=1000, seqs=3, seed=hd)


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "bands", "yarn"])
@pytest.mark.parametrize("far", [0, 1023, 131072 - 64, (1 << 24) - 64])
def test_append_positions(gpu, scaling, far):
    run_append(gpu, o.F32, 2, 1, 64, 16, 20, "halves", scaling, far=far, seed=far % 97, max_pos=1 << 24,
               magnitude=1.2 if scaling == "yarn" else 1.0)


@pytest.mark.parametrize("n,seqs,ps", [(1, 1, 16), (2, 2, 1024), (63, 5, 64), (700, 3, 32), (2500, 2500, 16)])
def test_append_counts(gpu, n, seqs, ps):
    run_append(gpu, o.BF16, 4, 2, 32, ps, n, "halves", gains=True, seqs=seqs, seed=n)


@pytest.mark.parametrize("dtype,shift,pad", [("f32", 4, 1), ("f16", 2, 3), ("bf16", 4, 2), ("f16", 8, 4), ("f32", 0, 5)])
def test_append_alignment(gpu, dtype, shift, pad):
    for layout in ("pairs", "halves"):
        run_append(gpu, o.TYPES[dtype], 3, 2, 64, 16, 9, layout, gains=True, seqs=2, seed=5, shift=shift, pad_stride=pad)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kw", [dict(inplace=True), dict(use_kv=False), dict(use_q=False), dict(use_pos=False), dict(rot=0)])
def test_append_parts(gpu, dtype, kw):
    run_append(gpu, o.TYPES[dtype], 4, 2, 64, 16, 11, "halves", gains=True, seqs=2, seed=3, **kw)


def test_append_leaves_out_what_is_out_of_range(gpu):
    bad = [("seq", -1), ("seq", 4), ("slot", -1), ("slot", 1 << 20), ("pos", -1), ("pos", 2048), ("seq", 2 ** 31 - 1),
           ("slot", -2 ** 31), ("pos", 2 ** 31 - 1)]
    run_append(gpu, o.F16, 4, 2, 64, 16, 80, "halves", gains=True, seqs=4, seed=9, max_pos=2048, drop=bad)


@pytest.mark.parametrize("use_kv", [True, False])
def test_append_pads_without_a_rotation(gpu, use_kv):
    """A negative position marks padding whether or not it is used to rotate."""
    run_append(gpu, o.F16, 4, 2, 64, 16, 40, rot=0, gains=True, seqs=2, seed=12, use_kv=use_kv, drop=[("pos", -1), ("pos", -2 ** 31)])


# ------------------------------------------------------------------------------------- attention

def run_attention(q, dt, H, KV, hd, ps, groups, per, q_len, prefix, own, seed=0, scale=None, pad=0, values=None, keys=None,
                  spoil=None, stream=None, max_len=None, max_prefix=None):
    """prefix: positions of each group; own: positions of each sequence (its queries' among them)."""
    rs = np.random.default_rng(seed)
    B = groups * per
    up = lambda n: -(-n // ps)  # noqa: E731
    L = max(own) if max_len is None else max_len
    P = max(prefix) if max_prefix is None else max_prefix
    stride = max(1, up(L), up(P)) + 1
    tables, n_pages = o.make_tables(rs, [up(n) for n in prefix] + [up(max(n, 0)) for n in own], stride)
    kf = rs.standard_normal((n_pages, KV, ps, hd))
    vf = rs.standard_normal((n_pages, KV, ps, hd))
    live = np.zeros((n_pages, ps), bool)
    for i, n in enumerate(list(prefix) + list(own)):
        t = np.arange(max(n, 0))
        live[tables[i][t // ps], t % ps] = True
    if keys is not None:
        kf = keys(kf)
    if values is not None:
        vf = values(vf, tables, prefix, own)
    kf[~live[:, None, :].repeat(KV, 1)] = np.nan
    vf[~live[:, None, :].repeat(KV, 1)] = np.nan
    k, v = o.encode(kf, dt), o.encode(vf, dt)
    width = H * hd + pad
    x = o.encode(rs.standard_normal((B * q_len, width)) * 1.5, dt)
    out0 = o.encode(np.full((B * q_len, width), 7.0), dt)
    scale = float(np.float32(hd ** -0.5 if scale is None else scale))
    plen, olen = np.array(prefix, np.int32), np.array(own, np.int32)
    tab, ptab = tables[groups:].copy(), tables[:groups].copy()
    bad = np.zeros(B, bool)
    if spoil:
        spoil(tab, ptab, olen, plen, bad, n_pages)
    dk, dv, dx, dout = o.Guarded(q, k), o.Guarded(q, v), o.Guarded(q, x), o.Guarded(q, out0)
    dtab, dptab, dlen, dplen = (o.Guarded(q, a) for a in (tab, ptab, olen, plen))
    p = pages_of(q, dt, KV, hd, ps, n_pages, dk.ptr, dv.ptr)
    a = q.AttentionArgs(pages=ctypes.pointer(p), n_heads=H, n_seq=B, q_len=q_len, n_groups=groups, q=dx.ptr, q_stride=width,
                        out=dout.ptr, out_stride=width, table=dtab.ptr, len=dlen.ptr, table_stride=stride, max_len=L,
                        prefix_table=dptab.ptr, prefix_len=dplen.ptr, prefix_stride=stride, max_prefix=P, scale=scale)
    lib = q.load_library()
    need = lib.qmh_paged_attention_ws(ctypes.byref(a))
    ws = o.Guarded(q, np.full(max(need, 16), 0xFF, np.uint8))  # NaN everywhere
    outs = []
    for _ in range(2):  # the same bits again, over the workspace as the first call left it
        q._check(lib.qmh_paged_attention(ctypes.byref(a), ws.ptr, need, stream), "attention")
        q.sync()
        outs.append(dout.get())
    ws.get()
    assert outs[0].tobytes() == outs[1].tobytes() and np.array_equal(dx.get(), x)
    assert np.array_equal(outs[0][:, H * hd:], out0[:, H * hd:]), "written between the rows"
    got = o.decode(outs[0][:, :H * hd], dt).reshape(B, q_len, H, hd)
    xv = o.decode(x, dt)[:, :H * hd].reshape(B, q_len, H, hd)
    kv_, vv = o.decode(k, dt), o.decode(v, dt)
    for i in range(B):
        g = i // per
        if bad[i]:
            assert np.isnan(got[i]).all(), f"sequence {i} has no whole length or page: NaN"
            continue
        pk, pv = (o.rows_of(y, tables[g], prefix[g], ps) for y in (kv_, vv))
        for j in range(q_len):
            n = max(own[i] - q_len + 1 + j, 0)
            kk = np.concatenate([pk, o.rows_of(kv_, tables[groups + i], n, ps)])
            ww = np.concatenate([pv, o.rows_of(vv, tables[groups + i], n, ps)])
            want, mag, reach = o.attention(xv[i, j], kk, ww, scale)
            # scores: hd products and sums, the scale; their error moves each probability by twice that, exponentials to
            # 2 steps; sums of n terms; 16-bit probabilities are rounded to the type; then the result
            ds = (hd + 4) * o.U32 * reach + 4 * o.U32
            tol = mag * (2 * ds + (len(kk) + 64) * o.U32 + (o.HALF[dt] if dt != o.F32 else 0)) * 1.01
            tol = tol + o.HALF[dt] * np.abs(want) + o.TINY[dt]
            if dt == o.F16:  # probabilities far below the largest fall under the type's normal range
                tol = tol + len(kk) * o.TINY[dt] * np.abs(np.nan_to_num(ww)).max(initial=0)
            o.close(got[i, j], want, tol, f"sequence {i} query {j} ({n} own, {prefix[g]} shared)")
    return got


SHAPES = [(6, 2, 48), (12, 12, 64), (32, 4, 64), (3, 3, 128), (5, 1, 80), (14, 2, 96), (2, 1, 8), (4, 2, 256), (1, 1, 136), (40, 1, 32)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,hd", SHAPES)
def test_attention_heads(gpu, dtype, H, KV, hd):
    run_attention(gpu, o.TYPES[dtype], H, KV, hd, 16, 2, 3, 1, [70, 33], [1, 17, 31, 32, 48, 5], seed=hd)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_len", [1, 2, 3, 8, 33])
def test_attention_queries(gpu, dtype, q_len):
    run_attention(gpu, o.TYPES[dtype], 6, 2, 64, 32, 2, 2, q_len, [129, 64], [q_len, q_len + 1, q_len + 64, 200], seed=q_len)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("groups,per,prefix,own", [
    (1, 1, [0], [1]), (1, 1, [1], [0]), (1, 1, [0], [0]), (1, 4, [15], [1, 2, 15, 16]), (3, 1, [16, 17, 0], [0, 1, 33]),
    (1, 2, [1000], [1, 700]), (2, 2, [511, 513], [300, 0, 129, 127]), (1, 1, [3000], [2]), (1, 1, [0], [2500]), (1, 70, [40], list(range(70)))])
def test_attention_lengths(gpu, dtype, groups, per, prefix, own):
    run_attention(gpu, o.TYPES[dtype], 4, 2, 64, 16, groups, per, 1, prefix, own, seed=len(own))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ps", [16, 64, 1024])
def test_attention_pages_and_strides(gpu, dtype, ps):
    run_attention(gpu, o.TYPES[dtype], 4, 4, 128, ps, 2, 2, 2, [ps, ps + 1], [2, ps - 1, ps + 3, 2 * ps], seed=ps, pad=64)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_rows_that_see_nothing(gpu, dtype):
    # more queries than own positions: the first ones see the prefix only, or nothing
    run_attention(gpu, o.TYPES[dtype], 2, 2, 64, 16, 2, 2, 5, [0, 20], [0, 3, 2, 5], seed=1)
    got = run_attention(gpu, o.TYPES[dtype], 2, 2, 64, 16, 1, 2, 3, [0], [0, 1], seed=2)
    assert (got[0] == 0).all() and (got[1, :2] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 16, 47, 130, 1000])
def test_attention_every_position_counts(gpu, dtype, n):
    """Equal scores, and values that are zero but for one position of the prefix and one of the own pages: a
    position that is missed, doubled or taken from another row shows in full."""
    for at in sorted({0, 1, n // 2, n - 2, n - 1} & set(range(n))):
        def spike(v, tables, prefix, own):
            v = np.zeros_like(v)
            for i, m in enumerate(list(prefix) + list(own)):
                t = min(at, m - 1)
                v[tables[i][t // 32], :, t % 32] = 64.0 * (i + 1)
            return v
        run_attention(gpu, o.TYPES[dtype], 8, 2, 64, 32, 1, 2, 1, [n], [n, max(1, n // 2)], keys=lambda k: k * 0, values=spike, seed=n)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_large_and_lowest_scores(gpu, dtype):
    # scores in the thousands: one position takes all
    run_attention(gpu, o.TYPES[dtype], 2, 1, 64, 16, 1, 2, 1, [100], [40, 3], scale=20.0, seed=4)
    big = 6e4 if dtype == "f16" else 3e38
    # keys of the type's lowest value, at scale 0: equal scores, or NaN where the products pass 32 bits
    run_attention(gpu, o.TYPES[dtype], 2, 1, 64, 16, 1, 1, 1, [0], [40], keys=lambda k: np.where(np.arange(64) == 0, -big, 0 * k), scale=0.0,
                  seed=5)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_negative_scale(gpu, dtype):
    run_attention(gpu, o.TYPES[dtype], 4, 2, 64, 16, 2, 2, 3, [70, 0], [3, 17, 40, 600], scale=-0.125, seed=14)
    run_attention(gpu, o.TYPES[dtype], 2, 2, 128, 32, 1, 3, 1, [1500], [1, 0, 33], scale=-0.5, seed=15)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_bad_lengths_and_pages_give_nan(gpu, dtype):
    def spoil(tab, ptab, olen, plen, bad, n_pages):
        olen[0], olen[1] = -1, 81  # the sequences of group 0
        tab[2, 1], tab[3, 0] = -1, n_pages  # those of group 1, and group 1's prefix:
        ptab[1, 2] = 2 ** 31 - 1
        plen[2] = -5  # group 2's
        bad[:6] = True

    run_attention(gpu, o.TYPES[dtype], 4, 2, 64, 16, 5, 2, 2, [40, 40, 40, 40, 40], [20, 20, 40, 40, 2, 80, 30, 30, 9, 9], spoil=spoil, seed=6)


def test_attention_on_another_stream_and_in_a_graph(gpu):
    """On a stream of the caller's, and captured into a graph that is replayed with new contents."""
    hip = _hip()
    q, dt, H, KV, hd, ps = gpu, o.BF16, 4, 2, 64, 16
    rs = np.random.default_rng(8)
    stream, graph, exe = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
    tables, n_pages = o.make_tables(rs, [20, 10, 10], 20)
    bufs = {name: q.DeviceBuffer(n) for name, n in dict(k=n_pages * KV * ps * hd * 2, v=n_pages * KV * ps * hd * 2, x=2 * H * hd * 2,
                                                       out=2 * H * hd * 2, eager=2 * H * hd * 2).items()}
    dtab, dptab = q.DeviceBuffer.from_array(tables[1:]), q.DeviceBuffer.from_array(tables[:1])
    dlen, dplen = q.DeviceBuffer(8), q.DeviceBuffer(4)
    p = pages_of(q, dt, KV, hd, ps, n_pages, bufs["k"].ptr, bufs["v"].ptr)
    a = q.AttentionArgs(pages=ctypes.pointer(p), n_heads=H, n_seq=2, q_len=1, n_groups=1, q=bufs["x"].ptr, q_stride=H * hd,
                        out=bufs["out"].ptr, out_stride=H * hd, table=dtab.ptr, len=dlen.ptr, table_stride=20, max_len=160,
                        prefix_table=dptab.ptr, prefix_len=dplen.ptr, prefix_stride=20, max_prefix=320, scale=0.125)
    L = q.load_library()
    need = L.qmh_paged_attention_ws(ctypes.byref(a))
    ws, ws2 = q.DeviceBuffer(max(need, 1)), q.DeviceBuffer(max(need, 1))
    b = q.AttentionArgs.from_buffer_copy(a)
    b.out = bufs["eager"].ptr
    try:
        assert hip.hipStreamBeginCapture(stream, 1) == 0
        rc = L.qmh_paged_attention(ctypes.byref(a), ws.ptr, need, stream)
        assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
        assert rc == 0, q.last_error()
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for plen, olen in ((320, (160, 1)), (1, (3, 99)), (0, (1, 1)), (300, (160, 160))):
            for name in ("k", "v", "x"):
                h = o.encode(rs.standard_normal(bufs[name].nbytes // 2), dt)
                L.qmh_memcpy_h2d(bufs[name].ptr, h.ctypes.data, h.nbytes)
            for d, h in ((dplen, np.array([plen], np.int32)), (dlen, np.array(olen, np.int32))):
                L.qmh_memcpy_h2d(d.ptr, h.ctypes.data, h.nbytes)
            assert L.qmh_paged_attention(ctypes.byref(b), ws2.ptr, need, None) == 0
            q.sync()
            assert hip.hipGraphLaunch(exe, stream) == 0
            assert hip.hipStreamSynchronize(stream) == 0
            got, want = bufs["out"].to_array(np.uint16), bufs["eager"].to_array(np.uint16)
            assert np.array_equal(got, want)
            assert np.isfinite(o.decode(got, dt)).all()
    finally:
        if exe:
            hip.hipGraphExecDestroy(exe)
        if graph:
            hip.hipGraphDestroy(graph)
        hip.hipStreamDestroy(stream)


def _hip():
    hip = ctypes.CDLL("libamdhip64.so")
    vp = ctypes.c_void_p
    hip.hipStreamCreate.argtypes = [ctypes.POINTER(vp)]
    hip.hipStreamBeginCapture.argtypes = [vp, ctypes.c_int]
    hip.hipStreamEndCapture.argtypes = [vp, ctypes.POINTER(vp)]
    hip.hipGraphInstantiate.argtypes = [ctypes.POINTER(vp), vp, vp, vp, ctypes.c_size_t]
    hip.hipGraphLaunch.argtypes = [vp, vp]
    for f in (hip.hipStreamSynchronize, hip.hipGraphExecDestroy, hip.hipGraphDestroy, hip.hipStreamDestroy):
        f.argtypes = [vp]
    return hip


# ------------------------------------------------------------------------------------- reorder

@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("groups,beams", [(1, 1), (2, 2), (3, 4), (2, 7), (1, 16), (2, 17), (1, 64)])
@pytest.mark.parametrize("KV,hd,ps", [(2, 64, 16), (1, 8, 16), (3, 128, 64), (1, 248, 32)])
def test_paged_reorder(gpu, dtype, groups, beams, KV, hd, ps):
    q, dt = gpu, o.TYPES[dtype]
    rs = np.random.default_rng(groups * 100 + beams + hd)
    B = groups * beams
    length = rs.integers(0, 3 * ps + 2, B).astype(np.int32)
    most = int(length.max()) + 3
    stride = -(-most // ps) + 1
    counts = [-(-most // ps)] * B
    table, n_pages = o.make_tables(rs, counts, stride)
    k, v = (rs.integers(0, 2 ** 16 if dt != o.F32 else 2 ** 31, (n_pages, KV, ps, hd)).astype(np.uint16 if dt != o.F32 else np.uint32)
            for _ in range(2))
    for trial in range(3):
        parent = rs.integers(-1, beams + 1, B).astype(np.int32)
        if trial == 1 and beams > 1:  # a ring: every state moves
            parent = ((np.arange(B) % beams + 1) % beams).astype(np.int32)
        tab = table.copy()
        if trial == 2:  # a page that leads nowhere is left alone
            tab[0, 0] = n_pages
            tab[-1, 0] = -1
        dk, dv = o.Guarded(q, k), o.Guarded(q, v)
        dtab, dlen, dpar = (o.Guarded(q, x) for x in (tab, length, parent))
        p = pages_of(q, dt, KV, hd, ps, n_pages, dk.ptr, dv.ptr)
        q._check(q.load_library().qmh_paged_reorder(ctypes.byref(p), dtab.ptr, stride, dlen.ptr, most, dpar.ptr, groups, beams, None),
                 "reorder")
        q.sync()
        wk, wv = k.copy(), v.copy()
        for i in range(B):
            f = parent[i]
            if f < 0 or f >= beams:
                continue
            f = i - i % beams + f
            for t in range(length[f]):
                a, b = tab[f, t // ps], tab[i, t // ps]
                if 0 <= a < n_pages and 0 <= b < n_pages:
                    wk[b, :, t % ps], wv[b, :, t % ps] = k[a, :, t % ps], v[a, :, t % ps]
        assert np.array_equal(dk.get(), wk) and np.array_equal(dv.get(), wv), trial


# ------------------------------------------------------------------------------------- long caches, graphs, streams

def test_pages_past_4_gib(gpu):
    """Pages at both ends of pools of 5 GiB each: append writes there, attention reads there, the reorder moves them."""
    q, L, KV, hd, ps, H = gpu, gpu.load_library(), 2, 128, 1024, 4
    n_pages = (5 << 30) // (KV * ps * hd * 2)
    rs = np.random.default_rng(12)
    pool = [q.DeviceBuffer(n_pages * KV * ps * hd * 2) for _ in range(2)]
    p = pages_of(q, o.BF16, KV, hd, ps, n_pages, pool[0].ptr, pool[1].ptr)
    table = np.array([[n_pages - 1, 1], [n_pages - 3, n_pages - 2]], np.int32)
    ptable = np.array([[n_pages - 4]], np.int32)
    tabs = np.concatenate([table, np.array([[n_pages - 4, -1]], np.int32)])
    lens = [1030, 1025, 700]
    tok = [(s, t) for s, n in enumerate(lens) for t in range(n)]
    seq, slot = np.array([s for s, _ in tok], np.int32), np.array([t for _, t in tok], np.int32)
    n, width = len(tok), 2 * KV * hd
    x = o.encode(rs.standard_normal((n, width)), o.BF16)
    dx, ds, dl, dt = (q.DeviceBuffer.from_array(a) for a in (x, seq, slot, tabs))
    a = q.AppendArgs(pages=ctypes.pointer(p), n_tokens=n, k=dx.ptr, k_stride=width, v=dx.ptr + 2 * KV * hd, v_stride=width, n_seq=3, table=dt.ptr,
                     table_stride=2, seq=ds.ptr, slot=dl.ptr)
    q._check(L.qmh_paged_append(ctypes.byref(a), None), "append")
    xv = o.decode(x, o.BF16).reshape(n, 2, KV, hd)
    hist = [xv[seq == s] for s in range(3)]
    qx = o.encode(rs.standard_normal((2, H * hd)), o.BF16)
    dq, dout, dtab, dptab = q.DeviceBuffer.from_array(qx), q.DeviceBuffer(2 * H * hd * 2), q.DeviceBuffer.from_array(table), q.DeviceBuffer.from_array(ptable)
    dlen, dplen = q.DeviceBuffer.from_array(np.array(lens[:2], np.int32)), q.DeviceBuffer.from_array(np.array(lens[2:], np.int32))
    t = q.AttentionArgs(pages=ctypes.pointer(p), n_heads=H, n_seq=2, q_len=1, n_groups=1, q=dq.ptr, q_stride=H * hd, out=dout.ptr, out_stride=H * hd,
                        table=dtab.ptr, len=dlen.ptr, table_stride=2, max_len=1100, prefix_table=dptab.ptr, prefix_len=dplen.ptr, prefix_stride=1,
                        max_prefix=700, scale=hd ** -0.5)
    need = L.qmh_paged_attention_ws(ctypes.byref(t))
    ws = q.DeviceBuffer(max(need, 1))

    def check(own):
        q._check(L.qmh_paged_attention(ctypes.byref(t), ws.ptr, need, None), "attention")
        q.sync()
        got = o.decode(dout.to_array(np.uint16), o.BF16).reshape(2, H, hd)
        for i in range(2):
            kk, vv = (np.concatenate([hist[2][:, c], own[i][:, c]]) for c in range(2))
            want, mag, _ = o.attention(o.decode(qx[i], o.BF16).reshape(H, hd), kk, vv, hd ** -0.5)
            o.close(got[i], want, mag * 2 * o.HALF[o.BF16] + np.abs(want) * o.HALF[o.BF16] + 1e-4, f"sequence {i}")
    check(hist[:2])
    dpar, dlen2 = q.DeviceBuffer.from_array(np.array([1, 0], np.int32)), q.DeviceBuffer.from_array(np.array([1025, 1025], np.int32))
    q._check(L.qmh_paged_reorder(ctypes.byref(p), dtab.ptr, 2, dlen2.ptr, 1030, dpar.ptr, 1, 2, None), "reorder")
    check([np.concatenate([hist[1], hist[0][1025:]]), hist[0][:1025]])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_attention_long_queries(gpu, dtype):
    # a suffix of many tokens per sequence: tiles of queries with their own ends
    run_attention(gpu, o.TYPES[dtype], 8, 2, 64, 16, 1, 2, 200, [90], [200, 333], seed=20)
    run_attention(gpu, o.TYPES[dtype], 2, 2, 128, 32, 2, 1, 77, [0, 40], [80, 77], seed=21)
    run_attention(gpu, o.TYPES[dtype], 2, 2, 256, 32, 1, 2, 20, [65], [30, 20], seed=22)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_bounds_above_the_lengths(gpu, dtype):
    # upper bounds far above every length: chunks that hold nothing
    run_attention(gpu, o.TYPES[dtype], 4, 2, 64, 16, 2, 2, 1, [100, 5], [3, 40, 1, 17], seed=23, max_len=3000, max_prefix=9000)
    run_attention(gpu, o.TYPES[dtype], 4, 4, 64, 16, 2, 2, 2, [0, 0], [3, 40, 2, 17], seed=24, max_len=3000, max_prefix=9000)


def test_append_one_gain_only(gpu):
    """Only the keys are normed: queries turn as they are."""
    q, L, H, KV, hd, n = gpu, gpu.load_library(), 2, 1, 64, 5
    rs = np.random.default_rng(31)
    x = rs.standard_normal((n, (H + 2 * KV) * hd)).astype(np.float32)
    g = (1 + 0.2 * rs.standard_normal(hd)).astype(np.float32)
    pool = [o.Guarded(q, np.zeros((1, KV, 16, hd), np.float32)) for _ in range(2)]
    p = pages_of(q, o.F32, KV, hd, 16, 1, pool[0].ptr, pool[1].ptr)
    dx, dg, out = o.Guarded(q, x), o.Guarded(q, g), o.Guarded(q, np.zeros((n, H * hd), np.float32))
    dz, dl, dt = (o.Guarded(q, np.array(a, np.int32)) for a in (np.zeros(n), np.arange(n), [[0]]))
    with q.Rotary(hd, max_pos=64) as r:
        a = q.AppendArgs(pages=ctypes.pointer(p), rotary=r.handle, n_tokens=n, n_heads=H, q=dx.ptr, q_stride=x.shape[1], q_out=out.ptr, q_out_stride=H * hd,
                         k=dx.ptr + 4 * H * hd, k_stride=x.shape[1], v=dx.ptr + 4 * (H + KV) * hd, v_stride=x.shape[1], k_gain=dg.ptr, eps=1e-5, n_seq=1,
                         table=dt.ptr, table_stride=1, seq=dz.ptr, slot=dl.ptr)
        q._check(L.qmh_paged_append(ctypes.byref(a), None), "append")
        q.sync()
    f, at, xv = o.freqs(hd, "none"), np.arange(n), x.astype(np.float64).reshape(n, -1, hd)
    tol = (hd + 12) * o.U32 * 2 * np.abs(xv).max() * 1.5
    o.close(out.get().reshape(n, H, hd), o.rotate(xv[:, :H], at, f, "pairs"), tol, "queries")
    o.close(pool[0].get()[0, :, :n].transpose(1, 0, 2), o.rotate(o.norm(xv[:, H:H + KV], g.astype(np.float64), 1e-5), at, f, "pairs"), tol, "keys")


def test_step_in_a_graph(gpu):
    """Append, attention, selection and reorder of one step captured together, replayed with new contents between eager
    work: every replay leaves what the eager calls leave on the same contents."""
    q, L, hip = gpu, gpu.load_library(), _hip()
    rs = np.random.default_rng(40)
    KV, H, hd, ps, B, V, ml = 2, 4, 64, 16, 4, 5000, 80
    tables, n_pages = o.make_tables(rs, [8] + [5] * B, 8)
    width = (H + 2 * KV) * hd
    sizes = dict(k=n_pages * KV * ps * hd, v=n_pages * KV * ps * hd, x=B * width, logits=B * V)
    dptab, dtab = q.DeviceBuffer.from_array(tables[:1]), q.DeviceBuffer.from_array(tables[1:])
    seq = q.DeviceBuffer.from_array(np.arange(B, dtype=np.int32))
    with q.Rotary(hd, "halves", "linear", factor=4.0, max_pos=1000) as rot:
        sides = []
        for _ in range(2):
            d = {n: q.DeviceBuffer(c * (4 if n == "logits" else 2)) for n, c in sizes.items()}
            d.update(q=q.DeviceBuffer(B * H * hd * 2), out=q.DeviceBuffer(B * H * hd * 2), slot=q.DeviceBuffer(4 * B), pos=q.DeviceBuffer(4 * B),
                     len=q.DeviceBuffer(4 * B), plen=q.DeviceBuffer(4), score=q.DeviceBuffer(4 * B), parent=q.DeviceBuffer(4 * B), token=q.DeviceBuffer(4 * B))
            p = pages_of(q, o.F16, KV, hd, ps, n_pages, d["k"].ptr, d["v"].ptr)
            pp = ctypes.pointer(p)
            a = q.AppendArgs(pages=pp, rotary=rot.handle, n_tokens=B, n_heads=H, q=d["x"].ptr, q_stride=width, q_out=d["q"].ptr, q_out_stride=H * hd,
                             k=d["x"].ptr + 2 * H * hd, k_stride=width, v=d["x"].ptr + 2 * (H + KV) * hd, v_stride=width, n_seq=B, table=dtab.ptr, table_stride=8,
                             seq=seq.ptr, slot=d["slot"].ptr, pos=d["pos"].ptr)
            t = q.AttentionArgs(pages=pp, n_heads=H, n_seq=B, q_len=1, n_groups=1, q=d["q"].ptr, q_stride=H * hd, out=d["out"].ptr, out_stride=H * hd,
                                table=dtab.ptr, len=d["len"].ptr, table_stride=8, max_len=ml, prefix_table=dptab.ptr, prefix_len=d["plen"].ptr, prefix_stride=8,
                                max_prefix=128, scale=0.125)
            s = q.BeamArgs(dtype=o.F32, n_groups=1, n_beams=B, vocab=V, n_out=B, logits=d["logits"].ptr, stride=V, score=d["score"].ptr,
                           out_score=d["score"].ptr, out_parent=d["parent"].ptr, out_token=d["token"].ptr)
            wa, wb = L.qmh_paged_attention_ws(ctypes.byref(t)), L.qmh_beam_select_ws(ctypes.byref(s))
            ws = q.DeviceBuffer(max(wa, 1)), q.DeviceBuffer(wb)

            def step(stream, a=a, t=t, s=s, p=p, d=d, ws=ws, wa=wa, wb=wb):
                assert L.qmh_paged_append(ctypes.byref(a), stream) == 0, q.last_error()
                assert L.qmh_paged_attention(ctypes.byref(t), ws[0].ptr, wa, stream) == 0, q.last_error()
                assert L.qmh_beam_select(ctypes.byref(s), ws[1].ptr, wb, stream) == 0, q.last_error()
                assert L.qmh_paged_reorder(ctypes.byref(p), dtab.ptr, 8, d["len"].ptr, ml, d["parent"].ptr, 1, B, stream) == 0, q.last_error()
            sides.append((d, step, p))
        stream, graph, exe = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        assert hip.hipStreamCreate(ctypes.byref(stream)) == 0
        try:
            assert hip.hipStreamBeginCapture(stream, 1) == 0
            sides[0][1](stream)
            assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
            assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
            for trial in range(5):
                n = int(rs.integers(1, ml + 1))
                vals = dict(slot=np.full(B, n - 1, np.int32), pos=np.full(B, 100 + n, np.int32), len=np.full(B, n, np.int32),
                            plen=np.array([rs.integers(0, 129)], np.int32), score=-rs.random(B).astype(np.float32))
                for name, c in sizes.items():
                    h = rs.standard_normal(c)
                    vals[name] = h.astype(np.float32) if name == "logits" else o.encode(h, o.F16)
                for d, _, _ in sides:
                    for name, h in vals.items():
                        L.qmh_memcpy_h2d(d[name].ptr, h.ctypes.data, h.nbytes)
                sides[1][1](None)
                q.sync()
                assert hip.hipGraphLaunch(exe, stream) == 0
                assert hip.hipStreamSynchronize(stream) == 0
                for name in ("k", "v", "q", "out", "score", "parent", "token"):
                    x, y = (d[name].to_array(np.uint8) for d, _, _ in sides)
                    assert np.array_equal(x, y), (trial, name)
        finally:
            if exe:
                hip.hipGraphExecDestroy(exe)
            if graph:
                hip.hipGraphDestroy(graph)
            hip.hipStreamDestroy(stream)
