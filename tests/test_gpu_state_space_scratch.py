"""What the state space operators need beside their matrices: scratch that does not grow past what the batch itself takes."""
import numpy as np
import pytest

from parallelreverseautodiff_b200 import engine as E
from test_gpu_state_space import check_scan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("sequences,each,d,n,q", [(4500, 1, 3, 2, 1), (4001, 2, 5, 3, 1), (1501, 3, 70, 2, 2), (300, 7, 700, 2, 1)])
def test_many_short_sequences_of_equal_length(engine, dtype, sequences, each, d, n, q):
    """More sequences than the device takes at a time, so that a span has several, and with the last span shorter."""
    check_scan(engine, dtype, [each] * sequences, d, n, q, packed=False)


def _scan(e, f, sequences, each, d, n):
    T, r = sequences * each, np.random.default_rng(0)
    m = lambda *s: e.upload(r.standard_normal(s, dtype=np.float32).astype(f))  # noqa: E731
    of = dict(u=m(T, d), delta=m(T, d), A=e.upload(-np.ones((d, n), f)), B=m(T, n), C=m(T, n), sequences=sequences)
    saved, y = e.empty((e.selective_scan_saved(T, d, n, f),), f), e.empty((T, d), f)
    out = {k: e.empty(of[k].shape, f) for k in ("u", "delta", "A", "B", "C")}
    return of, saved, y, out


def _scratch_of_a_training_step(f, sequences, each, d, n):
    """Bytes by which the device's free memory falls over a forward and a backward in a context of its own."""
    with E.Engine(0) as e:
        of, saved, y, out = _scan(e, f, sequences, each, d, n)
        free = e.device_info()["free_bytes"]
        e.selective_scan_forward(**of, out=y, save=saved)
        e.selective_scan_backward(**of, saved=saved, dy=y, out=out)
        e.sync()
        return free - e.device_info()["free_bytes"]


def test_scratch_of_many_sequences():
    """4096 sequences of two tokens, 512 channels of 16 states.  u has 17 MB; a span for every sequence would leave 134 MB of sums.  The
    device holds less than 2048 CTAs, so there are at most 4096 of them, which leave 1024 values each, 17 MB, and the sums of dB and dC
    over the groups of 64 channels take 8 MB; scratch is a quarter more than what is asked for, and comes in blocks of 2 MB."""
    assert _scratch_of_a_training_step(np.float32, 4096, 2, 512, 16) < 1.25 * 26e6 + 4 * 2 ** 21


def test_gradients_of_rows_that_come_in_several_launches(engine):
    """2100 tokens of 1000 double channels with 128 states: 125 groups of channels leave 4.3 MB of sums of dB and dC each, more than
    256 MB, so they come in three launches.  Against calls on 200 channels each, which come in one: dB and dC are their sums, the other
    gradients theirs.  The spans differ, so a result differs by as many roundings as the module's bound counts for 2100 tokens
    (2100 x (16 + 10 x 3.4) x 2 x 2^-53 = 2.3e-11) of the sum of its terms' magnitudes, which here is below 40 times the largest
    result; a launch that is missing or comes twice is off by the size of the results."""
    e, f, r = engine, np.float64, np.random.default_rng(3)
    T, d, n, part = 2100, 1000, 128, 200
    x = dict(u=r.standard_normal((T, d)), delta=r.standard_normal((T, d)) * 0.2 - 2, A=-r.uniform(0.5, 8, (d, n)), B=r.standard_normal((T, n)),
             C=r.standard_normal((T, n)), D=r.standard_normal(d), z=r.standard_normal((T, d)), delta_bias=r.standard_normal(d) * 0.1)
    dy = r.standard_normal((T, d))

    def run(columns):
        own = {k: v if k in "BC" else np.ascontiguousarray(v[columns] if k in ("A", "D", "delta_bias") else v[:, columns]) for k, v in x.items()}
        dev, off = {k: e.upload(v) for k, v in own.items()}, e.sequence_offsets([700, 0, 1393, 7])
        _, _, saved = e.selective_scan_forward(**dev, offsets=off, sequences=4, save=True)
        g = e.selective_scan_backward(**dev, offsets=off, sequences=4, saved=saved, dy=e.upload(np.ascontiguousarray(dy[:, columns])))
        return {k: m.numpy() for k, m in g.items()}

    got, parts = run(slice(0, d)), [run(slice(i, i + part)) for i in range(0, d, part)]
    for k, m in got.items():
        want = sum(p[k] for p in parts) if k in "BC" else np.concatenate([p[k] for p in parts], 0 if k in ("A", "D", "delta_bias") else 1)
        assert np.abs(m - want).max() <= 40 * 2.3e-11 * np.abs(want).max(), k


def test_scratch_of_many_states():
    """8192 float tokens of 1024 channels with 128 states: 128 groups of channels, 8.4 MB of sums of dB and dC each.  256 MB hold 32 of
    them, so that the device, which takes less than 2048 CTAs at a time, has at most 64 spans, each with 131072 values for dA, as many
    for the states between them and the bit that goes with them."""
    assert _scratch_of_a_training_step(np.float32, 1, 8192, 1024, 128) < 1.25 * (256 + 2.1 * 64 * 0.5) * 2 ** 20 + 4 * 2 ** 21
