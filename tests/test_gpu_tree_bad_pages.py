"""Pages of drafted nodes that are outside the pool (qmh_tree_attention): the nodes that see them are NaN, the others are what they
are with good pages, whatever else the tree holds."""
import numpy as np
import pytest

import _ops as o
from test_gpu_tree_attention import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("masks,H,KV,hd,own,prefix,q_len", [
    ("chain", 2, 1, 64, [52, 52], None, 20), ("tree", 4, 2, 64, [70, 52], [40, 0], 36), ("tree", 32, 4, 64, [1070, 700], [900, 300], 36),
    ("random", 2, 2, 128, [1300, 61], None, 45), ("tree", 3, 3, 256, [64, 90], None, 36)])
def test_a_page_that_only_some_nodes_see(gpu, dtype, odd, masks, H, KV, hd, own, prefix, q_len):
    dt, ps = o.TYPES[dtype], 16
    nodes = [q_len, min(q_len, 20)]
    at = [(own[0] - 1) // ps, (own[0] - nodes[0] + ps) // ps]  # the last page, and the first one of nodes alone
    seen = {}

    def touch(pool, table, lens, n, see):
        seen["see"] = see
        seen["size"] = np.linalg.norm(pool[0], axis=-1).max(), np.abs(pool[1]).max()
        if odd:  # a node before the pages that are none
            t = own[0] - nodes[0] + 1
            pool[1][table[0][t // ps], :, t % ps, 3] = np.inf

    want, first = run(gpu, dt, H, KV, hd, ps, 2, nodes, own, prefix=prefix, q_len=q_len, masks=masks, touch=touch, seed=hd)
    keys, values = seen["size"]
    # either side: 16-bit weights and results are off by half a step each, 32-bit scores by hd + 4 roundings of the largest sum of
    # products (at most the norms' product; a query's, 1.5 times normal numbers, is hardly ever above 1.5 (hd^0.5 + 6)), sums by a
    # rounding a term; f16 weights also by a smallest step a term
    reach, terms = 1.5 * (hd ** 0.5 + 6) * keys * hd ** -0.5, max(own) + max(prefix or [0]) + 64
    tol = 2 * 1.01 * values * (2 * o.HALF[dt] + 2 * ((hd + 4) * o.U32 * reach + 4 * o.U32) + terms * (o.U32 + (o.TINY[dt] if dt == o.F16 else 0)))
    some = False
    for page in at:
        for number in (-1, 2 ** 30):
            def spoil(table, lens, first, bad):
                table[0, page] = number
            got, _ = run(gpu, dt, H, KV, hd, ps, 2, nodes, own, prefix=prefix, q_len=q_len, masks=masks, touch=touch, spoil=spoil, check=False, seed=hd)
            node = np.arange(nodes[0])
            there = (own[0] - nodes[0] + node) // ps == page
            assert there.any() and own[0] - nodes[0] <= page * ps
            lost = (seen["see"][0][:nodes[0], :nodes[0]] & there).any(1)
            some |= 0 < lost.sum() < nodes[0]
            assert np.isnan(got[:nodes[0]][lost]).all()
            o.close(got[:nodes[0]][~lost], want[:nodes[0]][~lost], tol, f"page {page}")
            o.close(got[first[1]:first[2]], want[first[1]:first[2]], tol, "the other sequence")
    assert some


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_page_of_the_context_or_the_prefix_is_seen_by_all(gpu, dtype):
    """The page before the nodes, one that holds the context's end and the first node, and (not a node's at all) the prefix's."""
    for page in (0, 1):
        def spoil(table, own, first, bad):
            table[0, page] = -1
            bad[0] = True
        run(gpu, o.TYPES[dtype], 4, 2, 64, 16, 2, [20, 20], [40, 52], prefix=[30, 0], spoil=spoil, seed=page)
        run(gpu, o.TYPES[dtype], 4, 2, 64, 16, 2, [20, 20], [40, 1052], prefix=[30, 900], spoil=spoil, seed=page)
