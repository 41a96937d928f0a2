"""Group norm of data with values far from all others, against numpy in 64 bits.

The variance is a sum of squares of deviations from a value near the data: a deviation is off by half a step e of itself, its square by
three, and a run adds up to 32 of them, 35 e of the run's sum of squares.  Deviations from another value than the mean are larger
than those from the mean by that value's own, a few of them at most: twice 35, and half of that for 1 / sqrt of it, 35 e; 64 e are
allowed.  A value far away is in one run, where the others' squares vanish beside its own, within the same bound.  The mean takes 32 e of
a run's deviations and a rounding of its own.  y takes the errors of both and three roundings."""
import numpy as np
import pytest

from test_gpu_state_space import F, STEP, near

pytestmark = pytest.mark.gpu

# clusters; one group of a CTA; blocks of a large sample; groups wider than a CTA; values one at a time
SHAPES = [(4, 300, 96, 8), (1, 4096, 256, 1), (1, 4097, 512, 2), (2, 500, 2048, 1), (3, 1000, 33, 3), (64, 49, 96, 8)]


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("samples,positions,channels,groups", SHAPES)
@pytest.mark.parametrize("far", [1e3, -1e4, 1e6])
@pytest.mark.parametrize("where", ["first", "last", "first position", "a channel", "two"])
def test_single_values_far_from_all_others(engine, dtype, samples, positions, channels, groups, far, where):
    e, f, r = engine, F[dtype], np.random.default_rng(positions)
    x = r.standard_normal((samples, positions, groups, channels // groups)).astype(f)
    if where in ("first", "two"):
        x[:, 0, :, 0] = far
    if where == "last":
        x[:, -1, :, -1] = far
    if where == "two":
        x[:, positions // 2, :, -1] = -far
    if where == "first position":
        x[:, 0] *= far
    if where == "a channel":
        x[:, :, :, 0] += far
    wide = x.astype(np.float64)
    mean = wide.mean((1, 3))
    away = np.abs(wide - mean[:, None, :, None])
    rstd = 1 / np.sqrt((away ** 2).mean((1, 3)) + 1e-5)
    want = (wide - mean[:, None, :, None]) * rstd[:, None, :, None]
    y, m, s = e.group_norm_forward(e.upload(x.reshape(-1, channels)), groups, positions=positions)
    step = STEP[dtype]
    near(s.numpy(), rstd, 64 * step * rstd, f"far value, rstd {dtype}")
    of_mean = (40 * away.mean((1, 3)) + 2 * np.abs(mean)) * step
    near(m.numpy(), mean, of_mean, f"far value, mean {dtype}")
    limit = 68 * step * np.abs(want) + (of_mean * rstd)[:, None, :, None] * (1 + 68 * step)
    near(y.numpy().reshape(x.shape), want, limit, f"far value, y {dtype}")


def test_sums_over_many_samples(engine):
    """One value per group, so many groups that each has one place on the device: 5000 equal gradients, whose sum in one float would be
    off by more than 1000 half steps. At most 512 are added up before they go into a double: 512 half steps, and one of the result."""
    e, f, samples, channels = engine, np.float32, 5000, 80000
    if e.device_info()["free_bytes"] < 8 << 30:
        pytest.skip("needs 5 GB of device memory")
    c = f(1.518797)
    assert abs(float(np.cumsum(np.full(samples, c, f), dtype=f)[-1]) / (samples * float(c)) - 1) > 1000 * 2.0 ** -24
    zero, dy = e.zeros((samples, channels), f), e.upload(np.full((samples, channels), c, f))
    _, _, dbeta = e.group_norm_backward(zero, zero, zero, dy, channels, out=(dy, e.empty((channels,), f), e.empty((channels,), f)))
    want = np.full(channels, samples * float(c))
    near(dbeta.numpy(), want, 513 * 2.0 ** -24 * want, "sums over many samples")
