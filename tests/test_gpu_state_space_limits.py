"""State space operators at the limits of their inputs, against numpy in 64 bits."""
import numpy as np
import pytest

import state_space_reference as R
from test_gpu_state_space import F, STEP, near, scan_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("lowest", [-np.inf, "lowest"])
@pytest.mark.parametrize("lengths,d,n", [([5, 0, 40, 33], 6, 4), ([301], 34, 16), ([1, 2, 70], 5, 9)])
def test_states_that_forget_everything(engine, dtype, lowest, lengths, d, n):
    """A = -inf (or the type's lowest value) makes a state of its last token alone, whatever rows without a token lie beside it in a
    tile: as A = -1e30 in the reference, whose decays are 0 too. The limit is that of the operators' other tests, 2 T (16 + 10 |dt A|)
    + T + 64 roundings of a magnitude, with dt |A| of the states that remember: at most 3 x 3."""
    e, f, r = engine, F[dtype], np.random.default_rng(d)
    T, S = sum(lengths), len(lengths)
    x = scan_case(r, f, T, d, n, 1, S)
    x["delta"] = np.minimum(x["delta"], 1).astype(f)
    x["delta_bias"] = np.minimum(x["delta_bias"], 1).astype(f)
    forgets = r.random((d, n)) < 0.4
    dy = r.standard_normal((T, d)).astype(f)
    want, size = (R.scan(**{**x, "A": np.where(forgets, -1e30, x["A"])}, lengths=lengths, dy=dy, magnitude=m) for m in (False, True))
    x["A"][forgets] = np.finfo(f).min if lowest == "lowest" else lowest
    of = dict({k: e.upload(v) for k, v in x.items()}, offsets=e.sequence_offsets(lengths), sequences=S)
    y, last, saved = e.selective_scan_forward(**of, h_last=True, save=True)
    grads = e.selective_scan_backward(**of, saved=saved, dy=e.upload(dy))
    limit = (max(lengths) * (16 + 90) * 2 + T + 64) * STEP[dtype]
    near(y.numpy(), want["y"], limit * size["y"], f"forgetting scan y {dtype}")
    near(last.numpy(), want["last"], limit * size["last"], f"forgetting scan last {dtype}")
    for k, m in grads.items():
        near(m.numpy(), want[k].reshape(m.shape), limit * size[k].reshape(m.shape), f"forgetting scan d{k} {dtype}")
    # and single tokens
    one = {k: e.upload(x[k][:S] if k in ("u", "delta", "z", "B", "C") else x[k]) for k in x if k != "h0"}
    h = e.upload(x["h0"])
    y = e.selective_scan_step(**one, h=h)
    want, size = (R.scan(**{**x, **{k: x[k][:S] for k in ("u", "delta", "z", "B", "C")}, "A": np.where(forgets, -1e30, x["A"])}, lengths=[1] * S,
                         magnitude=m) for m in (False, True))
    near(y.numpy(), want["y"], 256 * STEP[dtype] * size["y"], f"forgetting step y {dtype}")
    near(h.numpy(), want["last"], 256 * STEP[dtype] * size["last"], f"forgetting step h {dtype}")
