"""qmh_paged_attention's largest scales: taken up to 2^127, refused beyond."""
import ctypes

import numpy as np
import pytest

import _ops as o
from test_gpu_paged_scores import attend
from test_paged_refusals import P, attention_args, refused


@pytest.mark.parametrize("scale", [2.0 ** 127 * 1.01, -3e38, float("inf"), float("nan")])
def test_scales_refused(qmh, scale):
    L = qmh.load_library()
    a = attention_args(qmh, scale=scale)
    assert L.qmh_paged_attention_ws(ctypes.byref(a)) == 0
    refused(qmh, L.qmh_paged_attention(ctypes.byref(a), P, 1 << 40, None), "scale")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [2.0 ** 127, -2.0 ** 127, 1e38])
def test_largest_scales(gpu, dtype, scale):
    """One score above the others takes all, however far above."""
    dt = o.TYPES[dtype]
    rs = np.random.default_rng(2)
    for n, prefix in ((1, 0), (40, 37), (900, 700)):
        k, x = np.zeros((n, 1, 64)), np.zeros((1, 64))
        k[:, 0, 1], x[0, 1] = 0.25, np.sign(scale)
        k[n // 2, 0, 1] = 0.5
        v = o.decode(o.encode(rs.standard_normal((n, 1, 64)), dt), dt)
        o.close(attend(gpu, dt, k, v, x, prefix, scale)[0], v[n // 2, 0], 0, f"{n} positions")
