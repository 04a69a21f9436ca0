"""qmh_beam_select with logits far from zero, all of them finite: masks of other values than the type's lowest, rows
that lie far out as a whole, maxima whose neighbours are more than 600 away."""
import numpy as np
import pytest

import _ops as o
from test_gpu_beam import run_select

pytestmark = pytest.mark.gpu

LEVELS = [3e4, 1e5, 3e9, 1e10, 1e12, 1e13, 1e16, 1e19, 3e19, 1e20, 3.4e24, 8e24, 1.5e25, 2e25, 1e30, 3e38]


def rounded(x, dt):
    return float(o.decode(o.encode(np.array([x]), dt), dt)[0])


def step(x, dt):
    """The distance of neighbouring values of the type at x."""
    return 2.0 ** (np.floor(np.log2(abs(x))) - (23 if dt == o.F32 else 7))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("level", [-x for x in LEVELS])
def test_select_segments_masked_with_a_far_value(gpu, dtype, level):
    """Stretches of rows, whole segments among them, hold a finite mask; the rest are ordinary logits."""
    dt = o.TYPES[dtype]
    rs = np.random.default_rng(7)
    for K, V, n_out in ((1, 100000, 4), (4, 32000, 8), (3, 9000, 40)):
        x = rs.standard_normal((2, K, V)) * 2.5
        x[0, :, : V // 2] = level
        x[0, 0, V // 2 : V - 700] = level
        x[1, :, V // 3 :] = level
        s = -rs.random((2, K))
        run_select(gpu, x, s, None, n_out, dt=dt)
        done = np.zeros((2, K), np.int32)
        done[:, K - 1] = 1
        run_select(gpu, x, s, done, n_out, dt=dt)
    # fewer ordinary tokens than places: masked ones take the rest
    x = np.full((1, 2, 5000), rounded(level, dt))
    x[0, 0, 4000:4003] = [1.0, 2.0, 3.0]
    run_select(gpu, x, np.array([[0.0, -np.inf]]), None, 6, dt=dt)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("level", LEVELS)
def test_select_rows_far_out(gpu, dtype, sign, level):
    """Rows of one far value; with others a few steps away and lower ones, ruled out ones and rising runs."""
    dt = o.TYPES[dtype]
    rs = np.random.default_rng(8)
    at = rounded(sign * level, dt)
    h = step(at, dt)
    for K, V, n_out in ((1, 30000, 5), (4, 3001, 8), (3, 600, 64)):
        s = -rs.random((1, K))
        run_select(gpu, np.full((1, K, V), at), s, None, n_out, dt=dt)
        x = at - h * rs.integers(0, 9, (1, K, V))
        run_select(gpu, x, s, None, n_out, dt=dt)
        x[..., ::3] = -np.inf
        x[..., 1::7] = at - abs(at)
        run_select(gpu, x, s, None, n_out, dt=dt)
        run_select(gpu, np.sort(at - h * rs.integers(0, 9, (1, K, V)), -1), s, None, n_out, dt=dt)
        x = np.full((1, K, V), -np.inf)
        x[..., V // 2] = at
        run_select(gpu, x, s, None, n_out, dt=dt)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("level", [-60000.0, -17000.0, -16384.0, -16000.0, 16000.0, 16384.0, 17000.0, 60000.0])
def test_select_rows_around_ordinary_far_values(gpu, dtype, level):
    """Ordinary differences at an offset, on both sides of where exponents are made another way."""
    rs = np.random.default_rng(9)
    x = level + rs.standard_normal((2, 3, 20011)) * 2.5 * np.array([1.0, 40.0]).reshape(2, 1, 1)
    run_select(gpu, x, -rs.random((2, 3)), None, 12, dt=o.TYPES[dtype])


def test_select_no_done_flags_and_an_end_token_outside(gpu):
    """Without finished flags the end token is not looked at, whatever the logits."""
    x = np.full((1, 2, 4000), -2e25)
    x[0, 0, :2000] = np.random.default_rng(1).standard_normal(2000)
    run_select(gpu, x, np.zeros((1, 2)), None, 8, eos=-7)
