"""Plans (qmh_paged_plan) whose work could grow with what asks for nothing: times of two calls that should take the same, far enough
apart where they do not that a busy machine does not matter; and what they write."""
import ctypes
import time

import numpy as np
import pytest

import _trees as tr
from test_gpu_plan import State, call

pytestmark = pytest.mark.gpu


def least(q, add, tokens, parent=None, tree=0, mask=False, ps=16):
    """Seconds of a call, the least of some, and its seq, slot and pos."""
    n, dev = len(add), q.DeviceBuffer.from_array
    full = lambda k: np.full(k, -1, np.int32)  # noqa: E731
    stride = -(-int(max(add)) // ps)
    d = {k: dev(a) for k, a in dict(table=full(n * stride), len=np.zeros(n, np.int32), keep=np.zeros(n, np.int32), add=np.asarray(add, np.int32),
                                    ring=np.arange(4096, dtype=np.int32), state=np.array([0, 4096], np.int32), first=full(n + 1), seq=full(tokens),
                                    slot=full(tokens), pos=full(tokens), mask=full(max(n * tree * (-(-tree // 32)), 1))).items()}
    par = dev(np.asarray(parent, np.int32)) if parent is not None else None
    a = q.PlanArgs(n_seq=n, page_size=ps, table=d["table"].ptr, table_stride=stride, len=d["len"].ptr, keep=d["keep"].ptr, add=d["add"].ptr,
                   free_pages=d["ring"].ptr, free_size=4096, free_state=d["state"].ptr, n_tokens=tokens, first=d["first"].ptr, seq=d["seq"].ptr,
                   slot=d["slot"].ptr, pos=d["pos"].ptr, parent=par.ptr if par else None, parent_stride=0, tree_size=tree,
                   mask=d["mask"].ptr if mask else None)
    L = q.load_library()
    need = L.qmh_paged_plan_ws(ctypes.byref(a))
    ws = q.DeviceBuffer(max(need, 16))
    best = 1e9
    for _ in range(12):  # from the second call on every sequence keeps nothing and gets the same again
        q.sync()
        t = time.perf_counter()
        q._check(L.qmh_paged_plan(ctypes.byref(a), ws.ptr, need, None), "plan")
        q.sync()
        best = min(best, time.perf_counter() - t)
    return best, [d[k].to_array(np.int32) for k in ("seq", "slot", "pos")]


@pytest.mark.parametrize("n", [1000, 65535])
def test_rows_before_many_sequences_without_any(gpu, n):
    """The last rows of a call, not a whole vector of them, before sequences that ask for none: as fast as where they are one."""
    times = []
    for rows in (40, 41, 42, 43):
        add = np.zeros(n, np.int32)
        add[:3] = 17, 3, rows - 20
        t, (seq, slot, pos) = least(gpu, add, 48)
        times.append(t)
        want = np.full((2, 48), -1)
        want[:, :rows] = np.repeat([0, 1, 2], add[:3]), np.concatenate([np.arange(x) for x in add[:3]])
        assert np.array_equal(seq, want[0]) and np.array_equal(slot, want[1]) and np.array_equal(pos, want[1])
    assert max(times[1:]) < 3 * times[0], times


@pytest.mark.parametrize("gap", [0, 1, 2, 5, 70])
@pytest.mark.parametrize("n", [40, 300, 2100])
def test_sequences_without_rows_between_others(gpu, gap, n):
    """Rows of one to six a sequence, `gap` sequences without any between them, more than what asks refused at the end."""
    rs = np.random.default_rng(gap)
    add = np.zeros(n, np.int64)
    add[::gap + 1] = rs.integers(1, 7, len(add[::gap + 1]))
    s = State(gpu, n, 16, 2, 2 * n, 2 * n, seed=gap)
    s.upload()
    call(gpu, s, None, add, max(int(add.sum()) * 2 // 3, 1))


@pytest.mark.parametrize("mask", [False, True])
def test_trees_with_room_for_more_nodes(gpu, mask):
    """A chain of 256 nodes takes as long where trees may have 1024 as where they may have 256."""
    times = []
    for size in (256, 1024):
        t, (seq, slot, pos) = least(gpu, [256], 256, parent=np.arange(-1, size - 1), tree=size, mask=mask)
        times.append(t)
        assert (seq == 0).all() and np.array_equal(slot, np.arange(256)) and np.array_equal(pos, slot)
    assert times[1] < 2 * times[0], times


@pytest.mark.parametrize("size", [1, 31, 32, 33, 63, 64, 65, 96, 97, 129, 1000, 1024])
@pytest.mark.parametrize("shape", ["chain", "star", "teeth", "any"])
def test_masks_word_by_word(gpu, size, shape):
    """Ancestors in every word, in the first and last ones alone, and in some."""
    j = np.arange(size)
    rs = np.random.default_rng(size)
    par = {"chain": j - 1, "star": np.where(j, 0, -1), "teeth": np.maximum(j - 70, -1), "any": tr.tree(rs, size, 0.2)}[shape]
    for n, mask in ((1, True), (5, True), (5, False)):
        s = State(gpu, n, 16, -(-size // 16), n * 64, n * 64, seed=size)
        s.upload()
        add = rs.integers(0, size + 1, n)
        add[0] = size
        call(gpu, s, None, add, int(add.sum()) + 3, parent=np.tile(par, (n, 1)).astype(np.int32), tree=size, static=True, mask=mask)
