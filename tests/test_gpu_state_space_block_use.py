"""A state space block as programs use it: calls between a forward and its backward, padded batches, results that are kept."""
import numpy as np
import pytest

from test_gpu_state_space_block import _block

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences", [2, 9])
def test_single_tokens_between_forward_and_backward(engine, sequences):
    """The same gradients, bit by bit, as without them, whether there are fewer sequences than tokens or as many."""
    e, f, r = engine, np.float64, np.random.default_rng(4)
    b, _ = _block(e, f, r)
    x, d_out, more = (e.upload(r.standard_normal((n, b.dim))) for n in (9, 9, sequences))
    states = b.new_states(sequences)
    got = []
    for stepped in (False, True):
        b.forward(x, sequences=3)
        for _ in range(2 if stepped else 0):
            b.step(more, states)
        got.append({"x": b.backward(d_out).numpy(), **{k: v.numpy() for k, v in b.g.items()}})
    for k in got[0]:
        assert np.array_equal(got[0][k], got[1][k]), k
