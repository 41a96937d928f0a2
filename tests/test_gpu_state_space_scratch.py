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
