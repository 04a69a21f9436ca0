"""The path of a drafted tree that the model agrees with, and its keys and values moved to follow the context (qmh_tree_accept),
against a walk on the host. Everything is whole numbers or copies: results are equal."""
import ctypes

import numpy as np
import pytest

import _ops as o
import _trees as tr

pytestmark = pytest.mark.gpu


def run(q, nodes, size=None, ragged=True, context=None, dt=o.F32, KV=2, hd=16, ps=16, layers=1, gap=0, move=True, agree=0.85, V=50, room=None, seed=0,
        static=False, spoil=None, path=True, history=True, twice=False):
    rs = np.random.default_rng(seed)
    B = len(nodes)
    size = size or max(max(nodes), 1)
    context = context if context is not None else rs.integers(0, 70, B)
    length = (np.array(nodes) + context).astype(np.int32)
    counts = [-(-int(n) // ps) for n in length]
    table, n_pages = o.make_tables(rs, counts, max(counts) + 1)
    first = tr.starts(nodes)
    rows = int(first[-1]) + 2 if ragged else B * size
    at = first if ragged else np.arange(B + 1) * size
    T = 1 if static else B
    parent = np.stack([tr.tree(rs, size) for _ in range(T)])
    token = rs.integers(0, V, (T, size)).astype(np.int32)
    choice = rs.integers(0, V, rows).astype(np.int32)
    for i in range(B):
        for c in rs.permutation(np.arange(1, max(nodes[i], 1))):
            if rs.random() < agree:
                choice[at[i] + parent[i % T][c]] = token[i % T][c]
    room = room or 40
    hlen = rs.integers(0, room + 1, B).astype(np.int32)
    hist = rs.integers(0, V, (B, room)).astype(np.int32)
    es = o.BYTES[dt]
    stride = n_pages * KV * ps * hd + gap * (16 // es)
    pools = [rs.integers(0, 2 ** 16, layers * stride * es // 2).astype(np.uint16) for _ in range(2)]
    if spoil:
        spoil(dict(parent=parent, token=token, choice=choice, first=first, len=length, table=table, hlen=hlen, n_pages=n_pages))
    G = lambda a: o.Guarded(q, a)  # noqa: E731
    dev = {k: G(a) for k, a in dict(parent=parent, token=token, choice=choice, first=first, len=length, table=table).items()}
    io = {k: G(a) for k, a in dict(count=np.full(B, 9, np.int32), path=np.full((B, size), 9, np.int32), next=np.full(B, 9, np.int32),
                                   keep=np.full(B, 9, np.int32), history=hist, hlen=hlen, k=pools[0], v=pools[1]).items()}
    pages = q.Pages(dtype=dt, n_kv_heads=KV, head_dim=hd, page_size=ps, n_pages=n_pages, k=io["k"].ptr, v=io["v"].ptr)
    a = q.AcceptArgs(n_seq=B, tree_size=size, parent=dev["parent"].ptr, parent_stride=0 if static else size, token=dev["token"].ptr,
                     token_stride=0 if static else size, n_rows=rows, first=dev["first"].ptr if ragged else None, choice=dev["choice"].ptr,
                     len=dev["len"].ptr, count=io["count"].ptr, path=io["path"].ptr if path else None, next=io["next"].ptr, keep=io["keep"].ptr,
                     history=io["history"].ptr if history else None, history_stride=room, history_len=io["hlen"].ptr if history else None,
                     pages=ctypes.pointer(pages) if move else None, n_layers=layers, layer_stride=stride, table=dev["table"].ptr,
                     table_stride=table.shape[1])
    q._check(q.load_library().qmh_tree_accept(ctypes.byref(a), None), "accept")
    q.sync()
    # ---- the walk
    want = dict(count=np.zeros(B, np.int32), path=np.full((B, size), -1, np.int32), next=np.full(B, -1, np.int32), keep=np.full(B, -1, np.int32),
                history=hist.copy(), hlen=hlen.copy(), k=pools[0].copy(), v=pools[1].copy())
    views = [want[n].reshape(-1)[l * stride * es // 2:][:n_pages * KV * ps * hd * es // 2].reshape(n_pages, KV, ps, -1) for n in "kv" for l in range(layers)]
    for i in range(B):
        t0, n = (int(first[i]), int(first[i + 1]) - int(first[i])) if ragged else (i * size, size)
        if not (0 <= t0 and 0 <= n <= size and t0 + n <= rows and n <= length[i] and (not move or length[i] <= table.shape[1] * ps)):
            continue
        line, p = [], parent[i % T]
        x = 0 if n else None
        while x is not None:
            line.append(x)
            x = next((c for c in range(x + 1, n) if p[c] == x and token[i % T][c] >= 0 and token[i % T][c] == choice[t0 + x]), None)
        begin = int(length[i]) - n
        want["count"][i], want["keep"][i] = len(line), begin + len(line)
        if line:
            want["path"][i, :len(line)] = line
            want["next"][i] = choice[t0 + line[-1]]
        if history and 0 <= hlen[i] < room:
            m = min(len(line), room - hlen[i])
            want["history"][i, hlen[i]:hlen[i] + m] = token[i % T][line[:m]]
            want["hlen"][i] += m
        for k, x in enumerate(line if move else []):
            s, d = begin + x, begin + k
            ps_, pd = table[i, s // ps], table[i, d // ps]
            if x != k and 0 <= ps_ < n_pages and 0 <= pd < n_pages:
                for y in views:
                    y[pd, :, d % ps] = y[ps_, :, s % ps]
    if not path:
        want["path"][:] = 9
    for name, w in want.items():
        assert np.array_equal(io[name].get(), w), (name, np.argwhere(io[name].get() != w)[:6])
    for d in dev.values():
        assert np.array_equal(d.get(), d.like)
    return want


@pytest.mark.parametrize("n", [1, 2, 8, 33, 64, 65, 257, 1024])
@pytest.mark.parametrize("ragged", [False, True])
def test_sizes(gpu, n, ragged):
    nodes = [n] * 3 if not ragged else [n, max(n // 3, 1), 0, n, 1]
    w = run(gpu, nodes, ragged=ragged, seed=n)
    run(gpu, nodes, ragged=ragged, agree=1.0, V=3, ps=32, seed=n)  # siblings with the same token
    assert n < 8 or w["count"].max() > 2


@pytest.mark.parametrize("dt", [o.F32, o.F16, o.BF16])
@pytest.mark.parametrize("KV,hd,ps,layers,gap", [(1, 8, 16, 1, 0), (4, 64, 32, 3, 5), (32, 128, 64, 2, 0), (3, 248, 16, 2, 1), (2, 80, 1024, 1, 0)])
def test_pages(gpu, dt, KV, hd, ps, layers, gap):
    run(gpu, [20, 7, 31], dt=dt, KV=KV, hd=hd, ps=ps, layers=layers, gap=gap, agree=0.95, seed=hd)


def test_long_paths(gpu):
    """Chains with a node left out here and there: every position moves, over pages, more than eight at a time."""
    def spoil(d):
        p = np.arange(-1, 199)
        for k in range(5, 200, 7):
            p[k] = p[k - 1]
        d["parent"][:] = p
        d["token"][:] = np.arange(200)
        for i in range(3):
            for c in range(1, 200):
                d["choice"][200 * i + p[c]] = c  # the last child
    w = run(gpu, [200] * 3, ragged=False, context=np.array([3, 16, 40]), spoil=spoil, room=300, seed=1)
    assert (w["count"] > 150).all()


def test_shared_tree_and_parts(gpu):
    run(gpu, [12, 12, 5, 12], static=True, seed=2)
    run(gpu, [12, 12, 5, 12], move=False, seed=2)
    run(gpu, [12, 12, 5, 12], path=False, seed=2)
    run(gpu, [12, 12, 5, 12], history=False, seed=2)
    run(gpu, [300] * 70, size=300, seed=5)


def test_choices_that_are_none(gpu):
    def spoil(d):
        d["choice"][::3] = -1
        d["token"][:, ::2] = -1
    run(gpu, [30, 30, 2], spoil=spoil, seed=3)


def test_bad_pages_rows_and_lengths(gpu):
    def pages(d):
        d["table"][0, 1], d["table"][1, 2], d["table"][2, 0] = -1, d["n_pages"], 2 ** 31 - 1
    run(gpu, [60, 60, 60, 60], spoil=pages, agree=1.0, seed=4)

    def lengths(d):
        d["len"][0], d["len"][1], d["len"][2] = 59, -1, d["table"].shape[1] * 16 + 1
    run(gpu, [60, 60, 60, 60], spoil=lengths, seed=4)

    for bad in ([0, 70, 80, 90, 100], [-1, 10, 20, 30, 40], [0, 5, 3, 9, 9], [0, 60, 120, 180, 2 ** 31 - 1], [-2 ** 31, 2 ** 31 - 1, 0, 1, 2]):
        def rows(d):
            d["first"][:] = bad
        run(gpu, [60, 60, 60, 60], spoil=rows, seed=6)

    def parents(d):
        d["parent"][:, 0] = 3
        d["parent"][:, 4:9] = [4, 7, -9, 2 ** 31 - 1, 8]
    run(gpu, [60, 60], spoil=parents, agree=1.0, seed=7)

    def histories(d):
        d["hlen"][:] = [-1, 40, 41, 38]
    run(gpu, [60, 60, 60, 60], spoil=histories, agree=1.0, seed=8)
