"""qmh_paged_attention where many workgroups share a row's positions: every number of partial results that the
division of the work can give, each of them with its share of the values."""
import ctypes

import pytest

import _ops as o
from test_gpu_paged import run_attention

pytestmark = pytest.mark.gpu

P = 1 << 20  # an address: sizes are asked for, nothing is read


def parts_of(q, dt, H, KV, hd, ps, groups, per, prefix, own):
    """Partial results of a row, from the workspace's size: head_dim floats and two statistics each."""
    stride = max(prefix, own) // ps + 1
    p = q.Pages(dtype=dt, n_kv_heads=KV, head_dim=hd, page_size=ps, n_pages=8, k=P, v=P)
    a = q.AttentionArgs(pages=ctypes.pointer(p), n_heads=H, n_seq=groups * per, q_len=1, n_groups=groups, q=P, q_stride=H * hd, out=2 * P,
                        out_stride=H * hd, table=P, len=P, table_stride=stride, max_len=own, prefix_table=P, prefix_len=P, prefix_stride=stride,
                        max_prefix=prefix, scale=1.0)
    need = q.load_library().qmh_paged_attention_ws(ctypes.byref(a))
    each = groups * per * H * (hd * 4 + 8)
    assert need % each == 0
    return need // each


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [40, 64, 96, 128, 200])
def test_attention_every_number_of_parts(gpu, dtype, hd):
    """One sequence, as many chunks of prefix (up to 40) and own positions (up to 24) as make 5 to 64 parts. Keys are
    equal, so each position weighs the same and a part left out shows as its share of the values."""
    dt = o.TYPES[dtype]
    chunk = 64 if dt == o.F32 else 128  # positions of one step of a workgroup
    seen = set()
    for want in range(5, 65):
        n = min(want - 1, 40)
        prefix, own = n * chunk - 5, (want - n) * chunk - 3
        got = parts_of(gpu, dt, 2, 1, hd, 64, 1, 1, prefix, own)
        seen.add(got)
        if got > 1:
            run_attention(gpu, dt, 2, 1, hd, 64, 1, 1, 1, [prefix], [own], seed=want, keys=lambda k: k * 0, values=lambda v, *_: v + 4)
    assert seen >= set(range(6, 65)), sorted(set(range(6, 65)) - seen)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups,KV,prefix,own,parts", [(16, 16, 700, 700, 2), (17, 10, 1400, 700, 3), (8, 16, 700, 700, 4)])
def test_attention_few_parts(gpu, dtype, groups, KV, prefix, own, parts):
    dt = o.TYPES[dtype]
    assert parts_of(gpu, dt, KV, KV, 64, 64, groups, 1, prefix, own) == parts
    run_attention(gpu, dt, KV, KV, 64, 64, groups, 1, 1, [prefix] * groups, [own] * groups, seed=parts, values=lambda v, *_: v + 4)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("groups,per,q_len,prefix,own", [(1, 1, 1, 3584, 2), (2, 2, 2, 10501, 157), (1, 1, 1, 7936, 3000), (1, 3, 3, 5800, 900)])
def test_attention_parts_of_random_scores(gpu, dtype, groups, per, q_len, prefix, own):
    run_attention(gpu, o.TYPES[dtype], 8, 2, 64, 32, groups, per, q_len, [prefix] * groups, [own] * (groups * per), seed=own)
