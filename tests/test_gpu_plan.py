"""Pages, rows, slots and masks made on the device (qmh_paged_plan) against a statement of the declaration that goes over the
sequences one by one: single calls, refusals, and walks of many calls in which no page may be lost or given twice."""
import ctypes

import numpy as np
import pytest

import _ops as o
import _trees as tr

pytestmark = pytest.mark.gpu
PAD = 5


class State:
    """Tables, lengths and the ring, on the device and as the statement has them."""

    def __init__(self, q, n, ps, stride, size, spare, turn=0, seed=0):
        self.q, self.n, self.ps, self.size = q, n, ps, size
        rs = np.random.default_rng(seed)
        self.table = rs.integers(-9, 0, (n, stride)).astype(np.int32)
        self.len = np.zeros(n, np.int32)
        self.ring = np.full(size, -7, np.int32)
        self.ring[(turn + np.arange(spare)) % size] = rs.permutation(size)[:spare]
        self.state = np.array([turn, spare], np.int32)

    def upload(self):
        self.dev = {k: o.Guarded(self.q, getattr(self, k)) for k in ("table", "len", "ring", "state")}

    def same(self):
        for k, d in self.dev.items():
            got = d.get()
            assert np.array_equal(got, getattr(self, k)), (k, np.argwhere(got != getattr(self, k))[:5])

    def plan(self, keep, add, tokens, parent=None, tree=0):
        """What the declaration says of one call; returns refused, first, rows of (seq, slot, depth)."""
        cap, ps = self.table.shape[1] * self.ps, self.ps
        at, count = (int(x) for x in self.state)
        good = 0 <= at < self.size and 0 <= count <= self.size
        if not good:
            at = count = 0
        room = self.size - count if good else 0
        why, rows, first, freed = [], [], [0], []
        asked = took = back = spent = 0
        for i in range(self.n):
            n, k, a = int(self.len[i]), int(self.len[i] if keep is None else keep[i]), int(0 if add is None else add[i])
            w, got = 0, 0
            if not (0 <= n <= cap and 0 <= k <= n and a >= 0 and k + a <= cap and (parent is None or a <= tree)):
                w = 3
            else:
                have, need = -(-n // ps), -(-(k + a) // ps)
                asked, back = asked + max(need - have, 0), back + max(have - need, 0)
                if (need > have and asked > count) or (need < have and back > room):
                    w = 1
                else:
                    spent += a
                    if a and spent > tokens:
                        w = 2
            if w == 0:
                for j in range(have, need):
                    self.table[i, j] = self.ring[(at + took) % self.size]
                    took += 1
                for j in range(need, have):
                    freed.append(self.table[i, j])
                    self.table[i, j] = -1
                d = np.arange(a) if parent is None else tr.depths(parent[i][:a])
                rows += [(i, k + j, k + int(d[j])) for j in range(a)]
                self.len[i], got = k + a, a
            why.append(w)
            first.append(first[-1] + got)
        for j, page in enumerate(freed):
            self.ring[(at + count + j) % self.size] = page
        if good:
            self.state[:] = (at + took) % self.size, count - took + len(freed)
        return np.array(why, np.int32), np.array(first, np.int32), rows


def call(q, s, keep, add, tokens, base=None, parent=None, tree=0, static=False, mask=True, stream=None):
    """One call on both sides, everything compared. parent: [n][tree]."""
    dev = lambda a: q.DeviceBuffer.from_array(np.asarray(a, np.int32)) if a is not None else None  # noqa: E731
    d = [dev(a) for a in (keep, add, base)]
    dpar = dev(parent[0] if static else parent) if parent is not None else None
    out = {k: o.Guarded(q, np.full(n, 77, np.int32)) for k, n in dict(first=s.n + 1, seq=tokens, slot=tokens, pos=tokens, refused=s.n).items()}
    words = -(-tree // 32)
    dmask = o.Guarded(q, np.full((s.n, tree, words), 0x12345678, np.uint32)) if parent is not None and mask else None
    a = q.PlanArgs(n_seq=s.n, page_size=s.ps, table=s.dev["table"].ptr, table_stride=s.table.shape[1], len=s.dev["len"].ptr, keep=o.ptr(d[0]),
                   add=o.ptr(d[1]), free_pages=s.dev["ring"].ptr, free_size=s.size, free_state=s.dev["state"].ptr, base=o.ptr(d[2]),
                   n_tokens=tokens, first=out["first"].ptr, seq=out["seq"].ptr, slot=out["slot"].ptr, pos=out["pos"].ptr,
                   refused=out["refused"].ptr, parent=o.ptr(dpar), parent_stride=0 if static else tree, tree_size=tree, mask=o.ptr(dmask))
    L = q.load_library()
    need = L.qmh_paged_plan_ws(ctypes.byref(a))
    ws = o.Guarded(q, np.full(max(need, 16), 0x3C, np.uint8))
    q._check(L.qmh_paged_plan(ctypes.byref(a), ws.ptr, need, None), "plan")
    q.sync()
    ws.get()
    why, first, rows = s.plan(keep, add, tokens, parent, tree)
    s.same()
    assert np.array_equal(out["refused"].get(), why), (out["refused"].get()[:20], why[:20])
    if tokens == 0:
        assert (out["first"].get() == 77).all()
        return why, first
    assert np.array_equal(out["first"].get(), first)
    want = np.full((3, tokens), -1, np.int32)
    if rows:
        r = np.array(rows, np.int32).T
        if base is not None:
            r[2] += np.asarray(base, np.int32)[r[0]]
        want[:, :r.shape[1]] = r
    for name, w in zip(("seq", "slot", "pos"), want):
        got = out[name].get()
        assert np.array_equal(got, w), (name, np.argwhere(got != w)[:5], got[got != w][:5], w[got != w][:5])
    if dmask is not None:
        m = np.full((s.n, tree, words), 0x12345678, np.uint32)
        for i in range(s.n):
            n = first[i + 1] - first[i]
            if n:
                m[i, :n] = tr.pack(tr.ancestors(parent[i][:n]), words)
        assert np.array_equal(dmask.get(), m)
    return why, first


def trees(rs, n, size):
    return np.stack([tr.tree(rs, size) for _ in range(n)])


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 1024, 1025, 2100])
@pytest.mark.parametrize("ps", [16, 128])
def test_counts(gpu, n, ps):
    rs = np.random.default_rng(n)
    stride = 700 // ps + 2
    s = State(gpu, n, ps, stride, n * stride, n * stride, turn=n * stride - 1, seed=n)
    s.upload()
    most = 40 if n < 1000 else 3
    add = rs.integers(0, most, n)
    why, _ = call(gpu, s, None, add, int(add.sum()) + PAD, base=rs.integers(0, 5000, n))
    assert (why == 0).all()
    add = rs.integers(0, most, n)
    call(gpu, s, (s.len * rs.random(n)).astype(np.int32), add, int(add.sum()), seq_base(rs, n))
    call(gpu, s, np.zeros(n, np.int32), None, 0)
    assert s.state[1] == s.size and sorted(s.ring) == list(range(s.size))


def seq_base(rs, n):
    return rs.integers(-3, 100, n)


@pytest.mark.parametrize("tokens", [4090, 4096, 4097, 9000, 40000])
def test_long_prompts(gpu, tokens):
    rs = np.random.default_rng(tokens)
    s = State(gpu, 7, 16, 3000, 7 * 3000, 4000, turn=19000, seed=1)
    s.upload()
    cuts = np.sort(rs.integers(0, tokens, 6))
    add = np.diff(np.concatenate([[0], cuts, [tokens]]))
    add[2] = 0
    call(gpu, s, None, add, tokens, base=rs.integers(0, 9, 7))
    call(gpu, s, s.len // 2, None, 0)


@pytest.mark.parametrize("size", [1, 2, 31, 32, 33, 64, 65, 100, 1024])
@pytest.mark.parametrize("n,static", [(3, False), (40, False), (5, True), (1100, False)])
def test_trees(gpu, size, n, static):
    if n * size > 120000:
        size = 100 + n % 7
    rs = np.random.default_rng(size)
    s = State(gpu, n, 32, 40, n * 40, n * 40, turn=3, seed=size)
    s.upload()
    par = trees(rs, 1 if static else n, size)
    par = np.repeat(par, n, 0) if static else par
    add = rs.integers(0, size + 1, n)
    add[n // 2] = size
    call(gpu, s, None, add, int(add.sum()) + PAD, base=seq_base(rs, n), parent=par, tree=size, static=static)
    call(gpu, s, (s.len * 0.7).astype(np.int32), add[::-1].copy(), int(add.sum()), parent=par, tree=size, static=static, mask=False)


def test_parents_that_are_none(gpu):
    rs = np.random.default_rng(0)
    s = State(gpu, 4, 16, 8, 40, 40)
    s.upload()
    par = np.array([[-1, 0, 1, 2, 3, 4], [5, 0, 2, 3, -1, 9], [2 ** 31 - 1, -2 ** 31, 0, 1, 2, 6], [0, 1, 2, 3, 4, 5]], np.int32)
    call(gpu, s, None, [6, 6, 6, 5], 23, parent=par, tree=6, base=seq_base(rs, 4))


@pytest.mark.parametrize("n", [40, 1300])
def test_refusals_one_by_one(gpu, n):
    """Numbers outside their range, too few pages, too few rows, in any mixture: the others are served as if these were not there."""
    rs = np.random.default_rng(n)
    s = State(gpu, n, 16, 6, 6 * n, 2 * n, turn=6 * n - 5, seed=n)
    s.upload()
    call(gpu, s, None, rs.integers(0, 30, n), 30 * n)
    for step in range(6):
        keep = (s.len * rs.random(n)).astype(np.int32)
        add = rs.integers(0, 40, n).astype(np.int32)
        for k, v in ((keep, -1), (keep, 97), (add, -1), (add, 97), (add, 2 ** 31 - 1), (keep, -2 ** 31)):
            k[rs.integers(0, n)] = v
        if step == 3:
            s.len[[1, 7]] = -1, 6 * 16 + 1
            s.upload()
        why, _ = call(gpu, s, keep, add, int(np.clip(add, 0, 96).sum()) * (3 if step % 2 else 1) // 2)
    assert 1 in why or 2 in why


def test_rings_that_are_none(gpu):
    for state in ([-1, 3], [10, 3], [0, -1], [0, 11], [2 ** 31 - 1, 2 ** 31 - 1]):
        s = State(gpu, 3, 16, 4, 10, 5)
        s.len[:] = 5, 20, 0
        s.state[:] = state
        s.upload()
        why, _ = call(gpu, s, [5, 3, 0], [3, 0, 9], 20)
        assert list(why) == [0, 1, 1]


@pytest.mark.parametrize("n,size", [(5, 7), (30, 40)])
def test_walk(gpu, n, size):
    """Many steps of drafting and keeping, in a pool that is nearly used up: the ring goes round, and every page is
    in one place at all times."""
    rs = np.random.default_rng(n)
    stride = 12
    s = State(gpu, n, 16, stride, n * 6, n * 6, seed=n)
    s.table[:] = -1
    s.upload()
    for step in range(25):
        keep = np.maximum(s.len - rs.integers(0, size, n), 0).astype(np.int32)
        if step % 5 == 4:
            keep[rs.integers(0, n, 3)] = 0  # these have ended
        add = np.minimum(rs.integers(1, size + 1, n), stride * 16 - keep)
        call(gpu, s, keep, add, int(add.sum()) + 2, parent=trees(rs, n, size), tree=size)
        at, count = s.state
        held = [p for i in range(n) for p in s.table[i, :-(-s.len[i] // 16)]]
        free = list(s.ring[(at + np.arange(count)) % s.size])
        assert sorted(held + free) == list(range(s.size))


def test_no_sequences(gpu):
    s = State(gpu, 0, 16, 4, 10, 5)
    s.table = np.zeros((1, 4), np.int32)
    s.len = np.zeros(1, np.int32)
    s.upload()
    s.table, s.len = s.table, s.len
    call(gpu, s, None, None, 9)
