"""qmh_paged_attention with scores far from zero, all of them finite in 32 bits: exact products, so that the softmax
follows from the scores' differences alone."""
import ctypes

import numpy as np
import pytest

import _ops as o
from test_gpu_paged import pages_of

pytestmark = pytest.mark.gpu


def attend(q, dt, k, v, x, prefix, scale, ps=32):
    """out [heads, hd] of one sequence of one query: x [heads, hd] over k, v [n, 1, hd], the first `prefix` of them shared."""
    n, _, hd = k.shape
    H = len(x)
    up = lambda m: -(-m // ps)  # noqa: E731
    own = n - prefix
    pages = up(prefix) + up(own)
    kp, vp = (np.full((max(pages, 1), 1, ps, hd), np.nan) for _ in range(2))
    for pool, rows in ((kp, k), (vp, v)):
        for t in range(prefix):
            pool[t // ps, :, t % ps] = rows[t]
        for t in range(own):
            pool[up(prefix) + t // ps, :, t % ps] = rows[prefix + t]
    dk, dv, dx = (o.Guarded(q, o.encode(a, dt)) for a in (kp, vp, x.reshape(1, -1)))
    dout = o.Guarded(q, o.encode(np.full((1, H * hd), 7.0), dt))
    dtab, dptab = o.Guarded(q, np.arange(up(prefix), pages + 1, dtype=np.int32)), o.Guarded(q, np.arange(up(prefix) + 1, dtype=np.int32))
    dlen, dplen = o.Guarded(q, np.array([own], np.int32)), o.Guarded(q, np.array([prefix], np.int32))
    p = pages_of(q, dt, 1, hd, ps, max(pages, 1), dk.ptr, dv.ptr)
    a = q.AttentionArgs(pages=ctypes.pointer(p), n_heads=H, n_seq=1, q_len=1, n_groups=1, q=dx.ptr, q_stride=H * hd, out=dout.ptr,
                        out_stride=H * hd, table=dtab.ptr, len=dlen.ptr, table_stride=up(own) + 1, max_len=own, prefix_table=dptab.ptr,
                        prefix_len=dplen.ptr, prefix_stride=up(prefix) + 1, max_prefix=prefix, scale=scale)
    L = q.load_library()
    need = L.qmh_paged_attention_ws(ctypes.byref(a))
    ws = o.Guarded(q, np.full(max(need, 16), 0xFF, np.uint8))
    q._check(L.qmh_paged_attention(ctypes.byref(a), ws.ptr, need, None), "attention")
    q.sync()
    ws.get()
    return o.decode(dout.get(), dt).reshape(H, hd)


def build(dt, n, hd, base, j, seed):
    """Keys and queries of two elements each whose products are sign * 2^base + j, exactly: two heads, of either sign."""
    rs = np.random.default_rng(seed)
    k, x = np.zeros((n, 1, hd)), np.zeros((2, hd))
    k[:, 0, 0], k[:, 0, 5] = 2.0 ** (base // 2), j
    x[:, 0], x[:, 5] = [2.0 ** (base - base // 2), -2.0 ** (base - base // 2)], 1.0
    v = o.decode(o.encode(rs.standard_normal((n, 1, hd)) + 2, dt), dt)
    return k, v, x


SPLITS = [(1, 0), (33, 0), (40, 37), (700, 650), (4000, 3500)]  # positions, and how many of them are the prefix's


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,prefix", SPLITS)
@pytest.mark.parametrize("base", [8, 10, 12, 16, 20, 23])
def test_attention_differences_of_far_scores(gpu, dtype, n, prefix, base):
    """Scores of +-2^base and a small whole number: any two of them differ by what those numbers do, whichever wave,
    chunk or part they are seen by."""
    dt = o.TYPES[dtype]
    rs = np.random.default_rng(n + base)
    j = rs.integers(0, 8, n).astype(np.float64)
    k, v, x = build(dt, n, 64, base, j, n)
    for scale in (1.0, 0.5):
        got = attend(gpu, dt, k, v, x, prefix, scale)
        p = np.exp((j - j.max()) * scale)
        p /= p.sum()
        want, mag = p @ v[:, 0], p @ np.abs(v[:, 0])
        # the reference of the exponents (powers of two, up to 2^10 of them) is rounded: 2^-15 of an exponent, for each of the
        # two rows that are compared; differences, products and exponentials to some steps of up to 16 powers; a sum of n terms;
        # 16-bit probabilities and the result round to the type
        tol = mag * (2 * 2.0 ** -15 + (16 + n + 64) * o.U32 + (o.HALF[dt] if dt != o.F32 else 0)) * 1.01 + o.HALF[dt] * mag + o.TINY[dt]
        for h in range(2):
            o.close(got[h], want, tol, f"scale {scale} head {h}")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,prefix", SPLITS)
@pytest.mark.parametrize("scale", [2.0 ** -6, 1.0, 3.0, 1e10, -1e10, -1.0])
def test_attention_one_far_score_takes_all(gpu, dtype, n, prefix, scale):
    """Scores of 2^28 scale, and others lower by a 128th: the largest ones share everything, to the last bit."""
    dt = o.TYPES[dtype]
    rs = np.random.default_rng(n)
    for most in ([n - 1], [0, n // 2]):
        top = np.zeros(n, bool)
        top[most] = True
        k = np.where(top, 128.0, rs.integers(120, 128, n))[:, None, None] * np.eye(1, 64) * 2.0 ** 7
        x = np.eye(1, 64).repeat(2, 0) * [[2.0 ** 14], [-2.0 ** 14]]
        v = o.decode(o.encode(rs.standard_normal((n, 1, 64)) + 2, dt), dt)
        got = attend(gpu, dt, k, v, x, prefix, scale)
        for h in range(2):
            s = k[:, 0, 0] * np.sign(x[h, 0]) * np.sign(scale)
            want = v[s == s.max(), 0].mean(0)
            o.close(got[h], want, (np.count_nonzero(s == s.max()) > 1) * (o.HALF[dt] + 2.0 ** -20) * np.abs(v[s == s.max(), 0]).max(0), f"head {h}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("level", [-3e38, 3e38, -1e30, 1e20])
def test_attention_every_score_at_one_far_value(gpu, dtype, level):
    """A row masked throughout with a finite value, and its opposite: every position weighs the same."""
    dt = o.TYPES[dtype]
    rs = np.random.default_rng(3)
    for n, prefix in SPLITS:
        k, x = np.eye(1, 64)[None].repeat(n, 0) * level, np.eye(1, 64)
        v = o.decode(o.encode(rs.standard_normal((n, 1, 64)) + 2, dt), dt)
        got = attend(gpu, dt, k, v, x, prefix, 1.0)
        mag = np.abs(v[:, 0]).mean(0)
        o.close(got[0], v[:, 0].mean(0), mag * ((n + 64) * o.U32 + 2 * o.HALF[dt]), f"{n} positions")
