"""Shared by the tests of the ops for drafted trees: random trees, masks and rows."""
import numpy as np


def tree(rs, n, chainy=0.5):
    """Parents of n nodes: node 0 the root, others below any earlier one."""
    p = [-1]
    for j in range(1, n):
        p.append(j - 1 if rs.random() < chainy else int(rs.integers(0, j)))
    return np.array(p[:n], np.int32)


def ancestors(parent):
    """Truth values [n, n]: a node's row has itself and its ancestors. A parent that is none counts as -1."""
    n = len(parent)
    see = np.zeros((n, n), bool)
    for j in range(n):
        if 0 <= parent[j] < j:
            see[j] = see[parent[j]]
        see[j, j] = True
    return see


def depths(parent):
    return ancestors(parent).sum(1) - 1


def pack(see, words, rs=None):
    """Rows of truth values as words of 32 bits; bits behind them are 0, or anything if rs is given."""
    see = np.asarray(see, bool)
    n = see.shape[-1]
    bits = np.zeros(see.shape[:-1] + (32 * words,), bool)
    if rs is not None:
        bits = rs.random(bits.shape) < 0.5
    bits[..., :n] = see
    w = (bits.reshape(see.shape[:-1] + (words, 32)).astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(-1)
    return w.astype(np.uint32)


def starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
