"""qmh_beam_select and qmh_beam_reorder against statements in 64 bits: the chosen beams and tokens exactly, the
scores to half a step of f32 (and the 64-bit sums' own error, far below it)."""
import ctypes

import numpy as np
import pytest

import _ops as o

pytestmark = pytest.mark.gpu


def best_of(x, score, done, n_out, eos):
    """[(score, beam, token)] of one group: x [beams, vocab] in 64 bits."""
    K, V = x.shape
    total = np.full((K, V), -np.inf)
    for b in range(K):
        if done is not None and done[b]:
            total[b, eos] = score[b]
            continue
        with np.errstate(all="ignore"):
            m = x[b].max() if not np.isnan(x[b]).any() else np.nan
            lse = m + np.log(np.exp(x[b] - m).sum())
            total[b] = score[b] + (x[b] - lse)
    total = np.where(np.isnan(total), -np.inf, total).reshape(-1)
    order = np.lexsort((np.arange(total.size), -total))[:n_out]
    out = [(total[i], i // V, i % V) for i in order if total[i] > -np.inf]
    return out + [(-np.inf, -1, -1)] * (n_out - len(out))


def run_select(q, x, score, done, n_out, eos=2, dt=o.F32, pad=0, shift=0, inplace=False):
    G, K, V = x.shape
    enc = o.encode(np.pad(x.reshape(G * K, V), ((0, 0), (0, pad)), constant_values=np.nan), dt)
    dx, ds = o.Guarded(q, enc, shift), o.Guarded(q, score.reshape(-1).astype(np.float32))
    dd = o.Guarded(q, done.reshape(-1).astype(np.int32)) if done is not None else None
    dsc = ds if inplace else o.Guarded(q, np.zeros((G, n_out), np.float32))
    dp, dt_ = (o.Guarded(q, np.full((G, n_out), 99, np.int32)) for _ in range(2))
    a = q.BeamArgs(dtype=dt, n_groups=G, n_beams=K, vocab=V, n_out=n_out, eos=eos, logits=dx.ptr, stride=V + pad, score=ds.ptr,
                   done=o.ptr(dd), out_score=dsc.ptr, out_parent=dp.ptr, out_token=dt_.ptr)
    L = q.load_library()
    need = L.qmh_beam_select_ws(ctypes.byref(a))
    ws = o.Guarded(q, np.full(need, 0xFF, np.uint8))
    q._check(L.qmh_beam_select(ctypes.byref(a), ws.ptr, need, None), "select")
    q.sync()
    ws.get()
    got_s, got_p, got_t = dsc.get().reshape(G, n_out), dp.get(), dt_.get()
    xv = o.decode(enc, dt)[:, :V].reshape(G, K, V)
    for g in range(G):
        want = best_of(xv[g], score[g].astype(np.float32).astype(np.float64), done[g] if done is not None else None, n_out, eos)
        assert list(got_p[g]) == [w[1] for w in want], g
        assert list(got_t[g]) == [w[2] for w in want], g
        s = np.array([w[0] for w in want])
        # one rounding to f32; the 64-bit log sum is good to 1e-12
        o.close(got_s[g], s, np.where(np.isfinite(s), np.abs(s) * o.U32 + 1e-12, 0), "scores")
    return got_s, got_p, got_t


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,K,V,n_out", [(1, 1, 1, 1), (1, 4, 32000, 8), (3, 5, 1003, 10), (2, 2, 5, 10), (1, 64, 700, 64), (2, 8, 9000, 16),
                                         (1, 3, 2049, 64), (40, 4, 2047, 4), (1, 1, 128256, 2), (300, 2, 2500, 4)])
def test_select(gpu, dtype, G, K, V, n_out):
    rs = np.random.default_rng(G * 31 + V)
    x = rs.standard_normal((G, K, V)) * 2.5
    done = rs.random((G, K)) < 0.3 if V > 2 else None
    run_select(gpu, x, -3 * rs.random((G, K)), None, n_out, dt=o.TYPES[dtype])
    run_select(gpu, x, -3 * rs.random((G, K)), done, n_out, dt=o.TYPES[dtype])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,shift", [(0, 4), (1, 0), (3, 12), (13, 8)])
def test_select_unaligned_rows(gpu, dtype, pad, shift):
    rs = np.random.default_rng(pad)
    run_select(gpu, rs.standard_normal((2, 3, 4001)), -rs.random((2, 3)), None, 6, dt=o.TYPES[dtype], pad=pad, shift=shift)


@pytest.mark.parametrize("n_out", [1, 7, 64])
@pytest.mark.parametrize("V", [40, 2048, 20000])
def test_select_ties(gpu, n_out, V):
    """Equal values everywhere: the lower beam, then the lower token; and few distinct values."""
    rs = np.random.default_rng(V)
    run_select(gpu, np.zeros((2, 3, V)), np.zeros((2, 3)), None, n_out)
    run_select(gpu, np.full((1, 2, V), -3.4e38), np.zeros((1, 2)), None, n_out)
    run_select(gpu, np.where(rs.random((2, 2, V)) < 0.5, 0.0, -0.0), np.zeros((2, 2)), None, n_out)
    few = rs.integers(0, 3, (2, 1, V)).astype(np.float64)
    run_select(gpu, few.repeat(3, 1), np.zeros((2, 3)), None, n_out)
    run_select(gpu, np.sort(rs.standard_normal((1, 2, V)), -1), np.array([[0.0, -1.0]]), None, n_out)
    run_select(gpu, -np.sort(rs.standard_normal((1, 2, V)), -1), np.array([[0.0, -1.0]]), None, n_out)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G,K,V,n_out", [(1, 12, 57576, 24), (1, 4, 151936, 8), (2, 16, 9000, 32), (3, 2, 40000, 64), (1, 64, 20000, 64), (1, 7, 70001, 1)])
def test_select_many_segments(gpu, dtype, G, K, V, n_out):
    """Few rows cut into many segments, most of which hold none of the best; finished and dead rows, masked stretches,
    the best all in one place, equal values."""
    rs = np.random.default_rng(V + n_out)
    dt = o.TYPES[dtype]
    x = rs.standard_normal((G, K, V)) * 2.5
    s = -3 * rs.random((G, K))
    done = (rs.random((G, K)) < 0.3).astype(np.int32)
    run_select(gpu, x, s, None, n_out, dt=dt)
    run_select(gpu, x, s, done, n_out, eos=V - 1, dt=dt)
    first = np.where(np.arange(K) == K - 1, s, -np.inf)
    run_select(gpu, x, first, None, n_out, dt=dt)
    y = x.copy()
    y[:, 0, : V - V // 16] = -np.inf
    y[:, K // 2, V // 9 :] = -np.inf
    y[:, K - 1, 700:1000] += 40
    run_select(gpu, y, s, None, n_out, dt=dt)
    y[0, 0, V // 2] = np.nan
    y[0, K - 1] = -np.inf
    run_select(gpu, y, s, done, n_out, dt=dt)
    run_select(gpu, rs.integers(0, 2, (G, K, V)).astype(np.float64), np.zeros((G, K)), None, n_out, dt=dt)
    run_select(gpu, np.zeros((G, K, V)), np.zeros((G, K)), done, n_out, dt=dt)


@pytest.mark.parametrize("level", [-710.0, -709.5, 710.0, -3e38])
@pytest.mark.parametrize("K,n_out", [(1, 2), (1, 64), (4, 32)])
def test_select_masked_segments_far_from_zero(gpu, K, n_out, level):
    """Segments without a logit, before, between and behind, in rows whose values lie far from 0."""
    rs = np.random.default_rng(int(abs(level)) % 1000)
    V = 150000
    x = np.full((1, K, V), -np.inf)
    for a in (70000, 90000, 149000):
        x[..., a : a + 800] = level - rs.random((1, K, 800)) * 20
    run_select(gpu, x, np.zeros((1, K)), None, n_out)


def test_select_masked_and_dead(gpu):
    rs = np.random.default_rng(3)
    x = rs.standard_normal((4, 4, 3000))
    x[0, :, 10:] = -np.inf  # ten tokens a beam
    x[1, 0] = -np.inf  # a beam that has none
    x[1, 1, 5] = np.nan
    x[1, 2, 7] = np.inf
    x[2] = -np.inf
    s = -rs.random((4, 4))
    s[3, 1:] = -np.inf  # the first step of a search
    _, p, _ = run_select(gpu, x, s, None, 64)
    assert (p[2] == -1).all() and set(p[1]) == {3} and set(p[3]) == {0}
    s[3, 0] = np.nan
    run_select(gpu, x, s, None, 8)
    done = np.zeros((4, 4))
    done[:, 3] = 1
    done[2] = 1
    run_select(gpu, x, np.where(np.isnan(s), -2.0, s), done, 9, eos=2999)


def test_select_in_place_scores(gpu):
    rs = np.random.default_rng(4)
    run_select(gpu, rs.standard_normal((5, 4, 5000)), -rs.random((5, 4)), None, 4, inplace=True)


def test_select_large_offsets(gpu):
    """A row stride that takes the last row past 2^32 bytes."""
    q, V, rows = gpu, 1000, 5
    stride = (1 << 28) + 64
    rs = np.random.default_rng(5)
    x = rs.standard_normal((1, rows, V)).astype(np.float32)
    buf = q.DeviceBuffer(((rows - 1) * stride + V) * 4)
    L = q.load_library()
    for r in range(rows):
        L.qmh_memcpy_h2d(buf.ptr + 4 * r * stride, x[0, r].ctypes.data, 4 * V)
    score = -rs.random(rows).astype(np.float32)
    ds = q.DeviceBuffer.from_array(score)
    out = [q.DeviceBuffer(32) for _ in range(3)]
    a = q.BeamArgs(dtype=o.F32, n_groups=1, n_beams=rows, vocab=V, n_out=8, eos=0, logits=buf.ptr, stride=stride, score=ds.ptr,
                   out_score=out[0].ptr, out_parent=out[1].ptr, out_token=out[2].ptr)
    need = L.qmh_beam_select_ws(ctypes.byref(a))
    ws = q.DeviceBuffer(need)
    q._check(L.qmh_beam_select(ctypes.byref(a), ws.ptr, need, None), "select")
    q.sync()
    want = best_of(x[0].astype(np.float64), score.astype(np.float64), None, 8, 0)
    assert list(out[1].to_array(np.int32)) == [w[1] for w in want] and list(out[2].to_array(np.int32)) == [w[2] for w in want]


# ------------------------------------------------------------------------------------- reorder

@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("beams", [1, 3, 8, 16, 17, 64])
@pytest.mark.parametrize("outer,rows,row_stride,live,gap,shift", [(1, 1, 64, 64, 0, 0), (2, 5, 48, 41, 16, 0), (3, 2, 37, 30, 3, 1),
                                                                  (1, 7, 1024, 1000, 64, 4), (2, 1, 8192, 8000, 0, 0), (1, 3, 4, 4, 4, 0),
                                                                  (2, 300, 36, 20, 0, 8)])
def test_beam_reorder(gpu, inplace, beams, outer, rows, row_stride, live, gap, shift):
    q = gpu
    rs = np.random.default_rng(beams * 7 + live)
    groups = 3
    B = groups * beams
    seq_stride = rows * row_stride + gap
    src = rs.integers(0, 256, (outer, B, seq_stride)).astype(np.uint8)
    dst = src if inplace else rs.integers(0, 256, src.shape).astype(np.uint8)
    for trial in range(2):
        parent = rs.integers(-1, beams + 1, B).astype(np.int32)
        if trial:
            parent = ((np.arange(B) % beams + 1) % beams).astype(np.int32)
        ds = o.Guarded(q, src, shift)
        dd = ds if inplace else o.Guarded(q, dst, shift)
        dp = o.Guarded(q, parent)
        st = q.BeamState(n_outer=outer, outer_stride=B * seq_stride, seq_stride=seq_stride, n_rows=rows, row_stride=row_stride, live=live)
        q._check(q.load_library().qmh_beam_reorder(ctypes.byref(st), dd.ptr, ds.ptr, dp.ptr, groups, beams, None), "reorder")
        q.sync()
        want = dst.copy()
        for i in range(B):
            f = i - i % beams + parent[i] if 0 <= parent[i] < beams else i
            for r in range(rows):
                want[:, i, r * row_stride:r * row_stride + live] = src[:, f, r * row_stride:r * row_stride + live]
        assert np.array_equal(dd.get(), want)
        if not inplace:
            assert np.array_equal(ds.get(), src)


def test_beam_reorder_of_more_pieces_than_a_launch(gpu):
    """2^24 pieces of a byte for each of two groups: more workgroups than one launch may have."""
    q, outer, groups, beams = gpu, 1 << 24, 2, 2
    rs = np.random.default_rng(9)
    src = rs.integers(0, 256, (outer, groups, beams), dtype=np.uint8)
    ds, dp = q.DeviceBuffer.from_array(src), q.DeviceBuffer.from_array(np.array([1, 1, 1, 0], np.int32))
    st = q.BeamState(n_outer=outer, outer_stride=4, seq_stride=1, n_rows=1, row_stride=1, live=1)
    q._check(q.load_library().qmh_beam_reorder(ctypes.byref(st), ds.ptr, ds.ptr, dp.ptr, groups, beams, None), "reorder")
    q.sync()
    got = ds.to_array(np.uint8).reshape(src.shape)
    assert np.array_equal(got[:, 0], src[:, 0, [1, 1]]) and np.array_equal(got[:, 1], src[:, 1, [1, 0]])


def test_select_on_two_streams_at_once(gpu):
    """Two selections of different sizes under way together, each with its own workspace, again and again."""
    q, L = gpu, gpu.load_library()
    hip = ctypes.CDLL("libamdhip64.so")
    hip.hipStreamCreate.argtypes = [ctypes.POINTER(ctypes.c_void_p)]
    hip.hipStreamSynchronize.argtypes = hip.hipStreamDestroy.argtypes = [ctypes.c_void_p]
    rs = np.random.default_rng(10)
    sides = []
    for G, K, V, n_out in ((2, 5, 60000, 20), (30, 4, 3001, 8)):
        x, score = rs.standard_normal((G, K, V)).astype(np.float32), -rs.random((G, K)).astype(np.float32)
        d = dict(x=q.DeviceBuffer.from_array(x), s=q.DeviceBuffer.from_array(score),
                 out=[q.DeviceBuffer.from_array(np.zeros((G, n_out), t)) for t in (np.float32, np.int32, np.int32)])
        d["a"] = q.BeamArgs(dtype=o.F32, n_groups=G, n_beams=K, vocab=V, n_out=n_out, eos=0, logits=d["x"].ptr, stride=V, score=d["s"].ptr,
                            out_score=d["out"][0].ptr, out_parent=d["out"][1].ptr, out_token=d["out"][2].ptr)
        d["need"] = L.qmh_beam_select_ws(ctypes.byref(d["a"]))
        d["ws"] = q.DeviceBuffer.from_array(np.full(d["need"], 0xFF, np.uint8))
        d["want"] = [best_of(x[g].astype(np.float64), score[g].astype(np.float64), None, n_out, 0) for g in range(G)]
        d["stream"] = ctypes.c_void_p()
        assert hip.hipStreamCreate(ctypes.byref(d["stream"])) == 0
        sides.append(d)
    q.sync()
    try:
        for _ in range(20):
            for d in sides:
                assert L.qmh_beam_select(ctypes.byref(d["a"]), d["ws"].ptr, d["need"], d["stream"]) == 0
        for d in sides:
            assert hip.hipStreamSynchronize(d["stream"]) == 0
            assert [w[1:] for g in d["want"] for w in g] == list(zip(d["out"][1].to_array(np.int32).ravel().tolist(), d["out"][2].to_array(np.int32).ravel().tolist()))
    finally:
        for d in sides:
            hip.hipStreamDestroy(d["stream"])


def test_select_more_rows_than_a_grid_dimension(gpu):
    """80000 rows: the rows pass one launch's limit."""
    q, G, K, V = gpu, 40000, 2, 9
    rs = np.random.default_rng(6)
    x, score = rs.standard_normal((G, K, V)).astype(np.float32), -rs.random((G, K)).astype(np.float32)
    dx, ds = o.Guarded(q, x), o.Guarded(q, score)
    out = [o.Guarded(q, np.zeros((G, 2), t)) for t in (np.float32, np.int32, np.int32)]
    a = q.BeamArgs(dtype=o.F32, n_groups=G, n_beams=K, vocab=V, n_out=2, eos=0, logits=dx.ptr, stride=V, score=ds.ptr, out_score=out[0].ptr,
                   out_parent=out[1].ptr, out_token=out[2].ptr)
    L = q.load_library()
    need = L.qmh_beam_select_ws(ctypes.byref(a))
    ws = o.Guarded(q, np.full(need, 0xFF, np.uint8))
    q._check(L.qmh_beam_select(ctypes.byref(a), ws.ptr, need, None), "select")
    q.sync()
    ws.get()
    p, t = out[1].get(), out[2].get()
    for g in list(range(0, 40)) + list(range(32740, 32800)) + list(range(G - 40, G)):
        want = best_of(x[g].astype(np.float64), score[g].astype(np.float64), None, 2, 0)
        assert list(p[g]) == [w[1] for w in want] and list(t[g]) == [w[2] for w in want], g


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n_out", [1, 16, 64])
def test_select_long_rows(gpu, dtype, n_out):
    """Rows of several pieces a wave (many rows share the chip): rising, falling, sawtooth, repeated and random."""
    rs = np.random.default_rng(n_out)
    V, G = 30011, 100
    kinds = [np.arange(V) * 1e-3, -np.arange(V) * 1e-3, (np.arange(V) % 700) * 0.01, np.zeros(V), np.where(np.arange(V) % 5000 == 4999, 3.0, -1.0)]
    x = rs.standard_normal((G, 2, V)).astype(np.float32) * 2
    for i, k in enumerate(kinds):
        x[i, 0] = k
        x[i + 10, 1] = k
    x[20, :, ::3] = -np.inf
    x[21, 0, 29000] = np.nan
    run_select(gpu, x, -rs.random((G, 2)), None, n_out, dt=o.TYPES[dtype])
