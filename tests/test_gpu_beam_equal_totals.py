"""qmh_beam_select where 64 bits do not tell totals apart although the logits differ: the lower beam, then the lower
token, as the declaration says, whichever of the logits is larger."""
import numpy as np
import pytest

import _ops as o
from test_gpu_beam import run_select

pytestmark = pytest.mark.gpu

SHAPES = [(2, 4, 3000, 8), (1, 4, 60000, 8), (1, 12, 57576, 24), (3, 2, 700, 64), (1, 1, 128256, 5), (1, 20, 2500, 33)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,K,V,n_out", SHAPES)
def test_select_scores_that_swallow_the_logits(gpu, dtype, G, K, V, n_out):
    """Beams at a score of the type's lowest value, say, in the place of none: each of their continuations stands at it."""
    dt = o.TYPES[dtype]
    rs = np.random.default_rng(V)
    x = rs.standard_normal((G, K, V)) * 2.5
    for far in (-3.4e38, -1e30, -1e17):
        run_select(gpu, x, np.full((G, K), far), None, n_out, dt=dt)
        s = np.full((G, K), far)
        s[:, 0] = 0.0
        y = x.copy()
        y[:, 0, 3:] = -np.inf  # the one live beam has three continuations
        run_select(gpu, y, s, None, n_out, dt=dt)
        y[:, 1:, : V // 2] = -np.inf
        y[:, K - 1, 5] = 1.0
        done = np.zeros((G, K), np.int32)
        done[:, K // 2] = 1
        run_select(gpu, y, s, done, n_out, eos=V - 1, dt=dt)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G,K,V,n_out", SHAPES)
def test_select_log_sums_that_swallow_the_logits(gpu, dtype, G, K, V, n_out):
    """One logit far above ordinary others: these come to a few distinct totals, or to one."""
    rs = np.random.default_rng(V + 1)
    x = rs.standard_normal((G, K, V)) * 2.5
    for far in (1e13, 1e16, 1e30):
        y = x.copy()
        y[:, :, V // 2] = far
        run_select(gpu, y, -rs.random((G, K)), None, n_out, dt=o.TYPES[dtype])
        run_select(gpu, y, np.where(np.arange(K) == K - 1, -1.0, -np.inf)[None].repeat(G, 0), None, n_out, dt=o.TYPES[dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G,K,V,n_out", SHAPES)
def test_select_logits_next_to_zero(gpu, dtype, G, K, V, n_out):
    rs = np.random.default_rng(V + 2)
    s = -rs.random((G, K))
    run_select(gpu, rs.standard_normal((G, K, V)) * 1e-20, s, None, n_out, dt=o.TYPES[dtype])
    x = np.where(rs.random((G, K, V)) < 0.01, rs.standard_normal((G, K, V)) * 1e-25, -rs.random((G, K, V)) - 0.5)
    x[..., :4] = -np.inf
    run_select(gpu, x, s, None, n_out, dt=o.TYPES[dtype])
    x = np.where(rs.random((G, K, V)) < 0.5, 0.0, -1e-30)
    run_select(gpu, x, np.zeros((G, K)), None, n_out, dt=o.TYPES[dtype])
    few = np.full((G, K, V), -4.0)  # fewer that are equal than places
    few[:, :, V // 2 : V // 2 + 3] = [1e-30, 2e-30, 0.0]
    run_select(gpu, few, s, None, 2, dt=o.TYPES[dtype])
