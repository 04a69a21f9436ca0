"""qmh_paged_attention where few positions outweigh each of very many others, which together still count."""
import numpy as np
import pytest

import _ops as o
from test_gpu_paged_scores import attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block", [0, 896])
@pytest.mark.parametrize("powers", [12.0, 18.0, 23.7, 24.6, 25.5, 28.0])
def test_attention_many_small_weights(gpu, dtype, block, powers):
    """60000 positions. In every 1024 there are four of the largest score, 32 apart, whose values are 0; the others' scores are
    `powers` powers of two lower and their values large."""
    dt, n, hd = o.TYPES[dtype], 60000, 64
    rs = np.random.default_rng(int(powers))
    top = np.isin(np.arange(n) % 1024, block + np.array([0, 32, 64, 96]))
    k, x = np.zeros((n, 1, hd)), np.zeros((1, hd))
    k[:, 0, 3], x[0, 3] = ~top, -powers
    v = np.where(top[:, None, None], 0.0, o.decode(o.encode(3e4 * (1 + rs.random((n, 1, hd))), dt), dt))
    scale = float(np.float32(np.log(2.0)))
    x = o.decode(o.encode(x, dt), dt)
    got = attend(gpu, dt, k, v, x, n - 500, scale, ps=1024)
    p = np.exp(x[0, 3] * k[:, 0, 3] * scale)
    p /= p.sum()
    want = p @ v[:, 0]
    # scores, exponents and sums in 32 bits: some steps of the exponent each, a sum of n terms; 16-bit probabilities and
    # the result round to the type, and no f16 probability is off by more than 2^-32 of the largest
    tol = want * (8 * powers * o.U32 + (n + 64) * o.U32 + 2 * (o.HALF[dt] if dt != o.F32 else o.U32)) + o.TINY[dt]
    if dt == o.F16:
        tol = tol + n * 2.0 ** -32 * np.abs(v).max() / np.count_nonzero(top)
    o.close(got[0], want, tol, f"2^-{powers}")
