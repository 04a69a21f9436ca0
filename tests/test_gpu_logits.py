"""Edited logits (qmh_logits_edit) against a statement in 64 bits. Where logits and parameters are quarters and powers of two the
edits are exact, and results and best tokens are equal; elsewhere the tolerance counts the roundings."""
import ctypes

import numpy as np
import pytest

import _ops as o
import _trees as tr

pytestmark = pytest.mark.gpu


def run(q, dt, V, seqs=2, per=1, rows=None, exact=True, history=60, biases=7, grammar=True, trees=None, out="other", best=True, shift=0, pad=0, seed=0,
        penalties="rpf", prompt=True, change=None, chain=False, n_allow=None, row_map=True, counts=None, gap=0):
    """counts: rows of each sequence (ragged), at most per."""
    rs = np.random.default_rng(seed)
    ragged = counts is not None
    counts = counts if ragged else [per] * seqs
    seqs = len(counts)
    first = tr.starts(counts) + gap
    at = first if ragged else np.arange(seqs + 1) * per
    n_rows = rows or (int(at[-1]) + 3 if ragged else seqs * per)
    x = rs.integers(-24, 25, (n_rows, V)) / 4 if exact else rs.standard_normal((n_rows, V)) * 3
    d = dict(x=x, hist=rs.integers(0, max(V // 4, 1), (seqs, history)), hlen=rs.integers(0, history + 1, seqs),
             rep=rs.choice([0.5, 1, 2, 4], seqs) if exact else 0.7 + rs.random(seqs), pres=rs.integers(0, 4, seqs) / 4 if exact else rs.random(seqs),
             freq=rs.integers(0, 3, seqs) / 4 if exact else rs.random(seqs) / 3, btok=rs.integers(0, V, (seqs, biases or 1)),
             bias=rs.integers(-8, 9, (seqs, biases or 1)) / 4 if exact else rs.standard_normal((seqs, biases or 1)),
             blen=rs.integers(0, biases + 1, seqs))
    d["plen"] = (d["hlen"] * rs.random(seqs)).astype(int)
    words = -(-V // 32)
    m = n_allow if n_allow is not None else (n_rows if not row_map else 5)
    d["allow"] = rs.random((max(m, 1), V)) < np.array([0.02, 0.5, 0.98, 1.0, 0.5])[np.arange(max(m, 1)) % 5][:, None]
    d["rowmap"] = rs.integers(-1, m + 1, n_rows) if row_map else np.arange(n_rows)
    d["node"] = rs.integers(0, V, (seqs, per)) if V < 40 else np.concatenate([d["hist"], rs.integers(0, V, (seqs, per))], 1)[:, rs.permutation(per + history)[:per]]
    see = np.zeros((seqs, per, per), bool)
    for i in range(seqs):
        see[i] = np.tril(np.ones((per, per), bool)) if chain else tr.ancestors(tr.tree(rs, per))
    d["see"], d["first"] = see, first
    if change:
        change(d)
    enc = o.encode(d["x"], dt)
    xv = o.decode(enc, dt)
    stride = V + pad
    host = np.full((n_rows, stride), 0x3B3B, o.raw(dt)) if dt != o.F32 else np.full((n_rows, stride), 7.5, np.float32)
    host[:, :V] = enc
    i32 = lambda a: q.DeviceBuffer.from_array(np.asarray(a, np.int32))  # noqa: E731
    f32 = lambda a: q.DeviceBuffer.from_array(np.asarray(a, np.float32))  # noqa: E731
    dx = o.Guarded(q, host, shift=shift)
    blank = np.full((n_rows, stride), 0x77, o.raw(dt))
    dout = dx if out == "inplace" else o.Guarded(q, blank, shift=(shift * 3) % 16) if out == "other" else None
    dbest = o.Guarded(q, np.full(n_rows, 777, np.int32)) if best else None
    a = q.LogitsArgs(dtype=dt, n_rows=n_rows, vocab=V, logits=dx.ptr, stride=stride, out=o.ptr(dout), out_stride=stride, best=o.ptr(dbest),
                     n_seq=seqs, rows_per_seq=per)
    keep = []

    def put(name, buf):
        keep.append(buf)
        setattr(a, name, buf.ptr)

    if ragged:
        put("first", i32(d["first"]))
    if history:
        put("history", i32(d["hist"]))
        put("history_len", i32(d["hlen"]))
        a.history_stride = history
        if prompt:
            put("prompt_len", i32(d["plen"]))
    for name, key in (("repetition", "rep"), ("presence", "pres"), ("frequency", "freq")):
        if name[0] in penalties:
            put(name, f32(d[key]))
    if biases:
        put("bias_token", i32(d["btok"]))
        put("bias", f32(d["bias"]))
        put("bias_len", i32(d["blen"]))
        a.bias_stride = biases
    if grammar:
        put("allow", q.DeviceBuffer.from_array(tr.pack(d["allow"], words + 1, rs)))
        a.allow_stride, a.n_allow = words + 1, m
        if row_map:
            put("allow_row", i32(d["rowmap"]))
    if trees:
        w = -(-per // 32) + 1
        put("node_token", i32(d["node"]))
        a.node_stride = per
        if not chain:
            put("mask", q.DeviceBuffer.from_array(tr.pack(see, w, rs)))
            a.mask_words, a.mask_stride = w, per * w
    L = q.load_library()
    need = L.qmh_logits_edit_ws(ctypes.byref(a))
    ws = o.Guarded(q, np.full(max(need, 16), 0x5A, np.uint8))
    q._check(L.qmh_logits_edit(ctypes.byref(a), ws.ptr, need, None), "logits")
    q.sync()
    ws.get()
    got = dout.get() if dout else None
    gbest = dbest.get() if best else None
    if out != "inplace":
        assert np.array_equal(dx.get(), host, equal_nan=dt == o.F32)
    # ---- the statement
    if got is not None:
        tail = host if out == "inplace" else blank
        assert np.array_equal(got[:, V:], tail[:, V:]), "written behind the rows"
    covered = np.zeros(n_rows, int)
    spans = [(int(d["first"][i]), int(d["first"][i + 1]) - int(d["first"][i])) if ragged else (i * per, per) for i in range(seqs)]
    spans = [(t0, n) if t0 >= 0 and 0 <= n <= per and t0 + n <= n_rows else (0, 0) for t0, n in spans]
    for t0, n in spans:
        covered[t0:t0 + n] += 1
    for i, (t0, n) in enumerate(spans):
        c, told = np.zeros(V), np.zeros(V, bool)
        h = min(max(d["hlen"][i], 0), history)
        for k in range(h if history else 0):
            t = d["hist"][i, k]
            if 0 <= t < V:
                if prompt and k < d["plen"][i]:
                    told[t] = True
                else:
                    c[t] += 1
        bias = np.zeros(V)
        for k in range(min(max(d["blen"][i], 0), biases) if biases else 0):
            if 0 <= d["btok"][i, k] < V:
                bias[d["btok"][i, k]] = np.float32(d["bias"][i, k])
        r, p, f = (float(np.float32(d[k][i])) if s in penalties else z for k, s, z in (("rep", "r", 1.0), ("pres", "p", 0.0), ("freq", "f", 0.0)))
        r = r if r > 0 else 1.0
        for j in range(n):
            if covered[t0 + j] > 1:
                continue  # what rows of two sequences hold is not defined
            cc = c.copy()
            if trees:
                for k in range(n):
                    if see[i, j, k] and 0 <= d["node"][i, k] < V:
                        cc[d["node"][i, k]] += 1
            v = xv[t0 + j]
            seen = (cc > 0) | told
            with np.errstate(invalid="ignore", over="ignore"):
                y = np.where(seen, np.where(v > 0, v / r, v * r), v)
                mag = np.abs(y) + f * cc + p + np.abs(bias)
                y = y - (f * cc + p * (cc > 0)) + bias
            row = d["rowmap"][t0 + j]
            ok = np.ones(V, bool)
            if grammar and 0 <= row < m:
                ok = d["allow"][row]
            y = np.where(ok, y, -np.inf)
            if got is not None:
                g = o.decode(got[t0 + j, :V], dt)
                if exact:
                    with np.errstate(invalid="ignore"):
                        want = o.decode(o.encode(y, dt), dt)
                    bad = ~((g == want) | (np.isnan(g) & np.isnan(want)))
                    assert not bad.any(), (i, j, np.argwhere(bad)[:5], g[bad][:5], want[bad][:5])
                else:
                    # a division or product, f c, its sum with p, the difference and the bias: five roundings
                    o.close(g, y, 5 * o.U32 * np.nan_to_num(mag) + o.HALF[dt] * np.abs(np.nan_to_num(y, neginf=0)) + o.TINY[dt], f"row {t0 + j}")
            if best:
                z = np.where(np.isnan(y), -np.inf, y)
                want = int(np.argmax(z)) if z.max() > -np.inf else -1
                if exact or want < 0 or np.ptp(np.nan_to_num(np.sort(z)[-2:], neginf=-1e30)) > 1e-5:
                    assert gbest[t0 + j] == want, (i, j, gbest[t0 + j], want, z[gbest[t0 + j]], z[want])
    covered = covered > 0
    if best:
        assert (gbest[~covered] == 777).all()
    if got is not None:
        assert np.array_equal(got[~covered], (host if out == "inplace" else blank)[~covered], equal_nan=dt == o.F32), "rows that are nobody's"
    return gbest


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 33, 300, 4095, 4096, 4097, 8197, 32003])
def test_vocabularies(gpu, dtype, V):
    run(gpu, o.TYPES[dtype], V, seed=V)
    run(gpu, o.TYPES[dtype], V, seqs=1, per=5, trees=True, seed=V + 1, out="none")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out,best", [("other", True), ("other", False), ("inplace", True), ("inplace", False), ("none", True)])
@pytest.mark.parametrize("grammar", [True, False])
def test_outputs(gpu, dtype, out, best, grammar):
    run(gpu, o.TYPES[dtype], 5003, seqs=3, per=4, trees=True, out=out, best=best, grammar=grammar, seed=2)
    run(gpu, o.TYPES[dtype], 9000, seqs=2, out=out, best=best, grammar=grammar, exact=False, seed=3)


@pytest.mark.parametrize("dtype,shift,pad", [("f32", 4, 1), ("f16", 2, 3), ("bf16", 6, 1), ("bf16", 0, 5), ("f32", 12, 3), ("f16", 8, 0)])
def test_alignment(gpu, dtype, shift, pad):
    for out in ("other", "inplace"):
        run(gpu, o.TYPES[dtype], 4101, seqs=2, per=2, out=out, shift=shift, pad=pad, seed=4)


@pytest.mark.parametrize("parts", [dict(history=0), dict(biases=0), dict(penalties=""), dict(penalties="r"), dict(penalties="p"), dict(penalties="f"),
                                   dict(prompt=False), dict(history=0, biases=0, penalties="", grammar=False), dict(row_map=False),
                                   dict(n_allow=0)])
def test_parts(gpu, parts):
    for out in ("other", "inplace"):
        run(gpu, o.F32, 4500, seqs=3, per=3, trees=True, out=out, seed=5, **parts)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("chain", [True, False])
@pytest.mark.parametrize("per", [1, 2, 31, 32, 33, 64, 65, 130])
def test_trees(gpu, dtype, chain, per):
    run(gpu, o.TYPES[dtype], 700, seqs=2, per=per, trees=True, chain=chain, seed=per)


@pytest.mark.parametrize("counts", [[3, 0, 5, 1], [0, 0], [40, 1, 33]])
def test_ragged(gpu, counts):
    run(gpu, o.F32, 4600, per=40, counts=counts, trees=True, gap=2, seed=6)


@pytest.mark.parametrize("first", [[0, 4, 3, 8], [-1, 2, 4, 5], [0, 2, 5, 2 ** 31 - 1], [0, 7, 8, 9], [-2 ** 31, 2 ** 31 - 1, 3, 4]])
def test_bad_rows_are_left_out(gpu, first):
    def change(d):
        d["first"][:] = first
    run(gpu, o.F32, 4600, per=5, counts=[2, 2, 2], trees=True, change=change, seed=7)


def test_numbers_that_are_none(gpu):
    def change(d):
        V = d["x"].shape[1]
        d["hist"][:, ::3] = [[-1], [V], [2 ** 31 - 1]]
        d["btok"][:, ::2] = [[-1], [V], [-2 ** 31]]
        d["hlen"][:] = [-5, 1000, 60]
        d["blen"][:] = [1000, -1, 7]
        d["plen"][:] = [5, -1, 2000]
        d["node"][:, ::2] = [[-1], [V], [2 ** 31 - 1]]
        d["rep"][:] = [0.0, -2.0, np.nan]
    run(gpu, o.F32, 4500, seqs=3, per=6, trees=True, change=change, seed=8)


def test_a_bias_that_is_there_twice(gpu):
    def change(d):
        d["btok"][:] = 17
        d["blen"][:] = [40, 3, 1]
    run(gpu, o.F32, 64, seqs=3, biases=40, change=change, grammar=False, seed=9)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_infinite_and_nan_logits(gpu, dtype):
    def change(d):
        d["x"][0, ::3], d["x"][1, ::5], d["x"][2, :] = np.nan, -np.inf, np.nan
        d["x"][3, 100], d["x"][4, :], d["x"][5, ::2] = np.inf, -np.inf, -np.inf
        d["rowmap"][:] = [0, 1, 1, 2, 3, 4]
        d["allow"][4] = False  # nothing may follow
    for out in ("other", "inplace"):
        best = run(gpu, o.TYPES[dtype], 4200, seqs=2, per=3, out=out, change=change, seed=10)
        assert best[2] == best[4] == best[5] == -1


def test_zeros_of_both_signs_tie(gpu):
    def change(d):
        d["x"][:] = -1.0
        d["x"][0, [900, 5000]] = [-0.0, 0.0]
        d["x"][1, [900, 5000]] = [0.0, -0.0]
        d["x"][2, [4, 5, 6, 7]] = [-1, -0.0, 0.0, -0.0]
    for dt in (o.F32, o.BF16):
        best = run(gpu, dt, 9000, seqs=3, change=change, history=0, biases=0, grammar=False, seed=11)
        assert list(best) == [900, 900, 5]


def test_repeated_tokens_by_the_thousand(gpu):
    def change(d):
        d["hist"][:] = d["hist"] % 5
        d["freq"][:] = 0.25
        d["hlen"][:] = 9000
    run(gpu, o.F32, 4100, seqs=2, history=9000, change=change, seed=12)


def test_many_rows_and_segments(gpu):
    run(gpu, o.BF16, 128256, seqs=2, per=3, trees=True, history=3000, biases=300, seed=13)
    run(gpu, o.F32, 600, seqs=300, per=1, history=20, seed=14)
    run(gpu, o.F16, 40, seqs=3, per=200, history=20, seed=15, trees=True)


def test_the_workspace_holds_what_other_calls_left(gpu):
    """The same call after others on the same workspace, and rows past 2 GiB of elements apart."""
    q, L = gpu, gpu.load_library()
    V, stride = 5000, (1 << 29) + 3
    x = q.DeviceBuffer(4 * (stride * 2 + V))
    row = (np.random.default_rng(0).integers(-99, 99, V) / 4).astype(np.float32)
    for r in range(3):
        row[r * 1111] = 50.0
        q._check(L.qmh_memcpy_h2d(x.ptr + 4 * stride * r, row.ctypes.data, row.nbytes), "copy")
        row[r * 1111] = -60.0
    best = q.DeviceBuffer(12)
    a = q.LogitsArgs(dtype=o.F32, n_rows=3, vocab=V, logits=x.ptr, stride=stride, best=best.ptr, n_seq=1, rows_per_seq=3)
    need = L.qmh_logits_edit_ws(ctypes.byref(a))
    ws = q.DeviceBuffer.from_array(np.full(need, 0xFF, np.uint8))
    for _ in range(2):
        q._check(L.qmh_logits_edit(ctypes.byref(a), ws.ptr, need, None), "logits")
        q.sync()
        assert list(best.to_array(np.int32)) == [0, 1111, 2222]
