"""Shared by the tests of the ops for several continuations of one prompt: element types without torch, guarded
device arrays and 64-bit statements of the operators."""
import ctypes
import math

import numpy as np

F32, F16, BF16 = 0, 1, 4
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}
BYTES = {F32: 4, F16: 2, BF16: 2}
U32 = 2.0 ** -24  # half a step of f32, relative
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}  # half a step of each type, relative
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}  # a step of the smallest values


def encode(x, dt):
    """x rounded to the type (nearest, ties to even), as its bytes' array."""
    x = np.ascontiguousarray(x, np.float32)
    if dt == F32:
        return x
    if dt == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u >> 16) + ((u & 0xFFFF) > 0x8000) + (((u & 0xFFFF) == 0x8000) & ((u >> 16) & 1))).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def decode(a, dt):
    """float64 values of encoded elements."""
    if dt == F32:
        return a.astype(np.float64)
    if dt == F16:
        return a.view(np.float16).astype(np.float64)
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def raw(dt):
    return np.float32 if dt == F32 else np.uint16


class Guarded:
    """A device copy of an array with `pad` bytes of a pattern before and behind it, checked by ok(); `shift`
    bytes move the array off its alignment."""

    def __init__(self, q, a, shift=0, pad=4096):
        a = np.ascontiguousarray(a)
        self.q, self.like, self.pad, self.shift = q, a, pad, shift
        host = np.full(a.nbytes + 2 * pad, 0xA5, np.uint8)
        host[pad + shift:pad + shift + a.nbytes] = a.view(np.uint8).reshape(-1)
        self.buf = q.DeviceBuffer.from_array(host)
        self.ptr = self.buf.ptr + pad + shift

    def get(self):
        host = self.buf.to_array(np.uint8)
        a, b = self.pad + self.shift, self.pad + self.shift + self.like.nbytes
        assert (host[:a] == 0xA5).all() and (host[b:] == 0xA5).all(), "written outside the array"
        return host[a:b].view(self.like.dtype).reshape(self.like.shape)


def close(got, want, tol, what=""):
    """|got - want| <= tol elementwise; where want is NaN or infinite, the same."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (got.shape, want.shape)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)]), f"{what}: infinities"
    tol = np.broadcast_to(tol, want.shape)
    d = np.abs(got - want)
    bad = fin & ~(d <= tol)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, d / np.maximum(tol, 1e-300), 0)), want.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {want.size} off; at {i}: {got[i]} for {want[i]}, tolerance {tol[i]}")


# ------------------------------------------------------------------------------------- rotation

def freqs(rot, scaling, theta=10000.0, factor=8.0, low=1.0, high=4.0, first=8192):
    """Radians per position of each pair, from the declared formulas."""
    out = []
    for i in range(rot // 2):
        th = theta * factor ** (rot / (rot - 2)) if scaling == "ntk" else theta
        f = th ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        if scaling in ("bands", "yarn"):
            if scaling == "bands":
                w = (first * f / (2 * math.pi) - low) / (high - low)
            else:
                c = lambda n: rot * math.log(first / (2 * math.pi * n)) / (2 * math.log(theta))  # noqa: E731
                a, b = max(math.floor(c(high)), 0), min(math.ceil(c(low)), rot - 1)
                w = 1 - (i - a) / max(b - a, 0.001)
            w = min(max(w, 0.0), 1.0)
            f = f * w + f / factor * (1 - w)
        out.append(f)
    return np.array(out)


def rotate(x, pos, f, layout, magnitude=1.0):
    """x [n, heads, hd] turned by pos [n]: the first 2 len(f) elements of each head."""
    half = len(f)
    ang = np.asarray(pos, np.float64)[:, None] * f
    c, w = (np.cos(ang) * magnitude)[:, None], (np.sin(ang) * magnitude)[:, None]
    y = x.copy()
    a, b = (slice(0, half), slice(half, 2 * half)) if layout == "halves" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    y[..., a] = x[..., a] * c - x[..., b] * w
    y[..., b] = x[..., a] * w + x[..., b] * c
    return y


def norm(x, gain, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain


# ------------------------------------------------------------------------------------- pages

def make_tables(rs, counts, stride, spare=2):
    """Tables of distinct shuffled pages; entries behind a sequence's last page lead nowhere. And the pool's size."""
    n = sum(counts) + spare
    perm = rs.permutation(n).astype(np.int32)
    t = rs.choice(np.array([-1, n, 2 ** 31 - 1, -2 ** 31], np.int32), (len(counts), stride)).astype(np.int32)
    at = 0
    for i, c in enumerate(counts):
        t[i, :c] = perm[at:at + c]
        at += c
    return t, n


def rows_of(pool, table, n, ps):
    """[n, kv heads, hd] of a table row's first n positions (pool: [pages, kv heads, page, hd])."""
    t = np.arange(n)
    return pool[table[t // ps], :, t % ps]


def attention(q, k, v, scale):
    """One query's out [heads, hd] over k, v [n, kv heads, hd], sum p |v| beside it and the largest sum |q k| scale."""
    H, KV = q.shape[0], k.shape[1]
    out, mag, reach = np.zeros(q.shape), np.zeros(q.shape), 0.0
    if len(k) == 0:
        return out, mag, reach
    for h in range(H):
        g = h // (H // KV)
        s = k[:, g] @ q[h]
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.where(np.abs(s) > np.finfo(np.float32).max, s * np.inf, s) * scale  # scores are held in 32 bits
        reach = max(reach, (np.abs(k[:, g]) @ np.abs(q[h])).max() * abs(scale))
        with np.errstate(invalid="ignore"):
            e = np.exp(s - max(s.max(), -1e300))  # no score above -inf: nothing is seen
        if e.sum() == 0:
            continue
        p = e / e.sum()
        out[h], mag[h] = p @ v[:, g], p @ np.abs(v[:, g])
    return out, mag, reach


def ptr(x):
    return x.ptr if x is not None else None


def byref(x):
    return ctypes.byref(x)
