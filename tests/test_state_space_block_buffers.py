"""Which buffers the calls of a state space block work on: what one call keeps for another is not written by a third."""
import numpy as np
import pytest

from parallelreverseautodiff_b200.networks import StateSpaceBlock
from recording_library import recording_engine

F = np.dtype(np.float32)


def _block(width=4):
    e = recording_engine()
    b = StateSpaceBlock(e, F, 8, 12, 4, 1, 2, width, 2)
    return e, b, {m.ptr for m in (*b.p.values(), *b.g.values())}


@pytest.mark.parametrize("width", [1, 4])
@pytest.mark.parametrize("sequences", [2, 9])
def test_single_tokens_use_buffers_of_their_own(sequences, width):
    """Between a forward and its backward, with fewer sequences than tokens and with as many."""
    e, b, parameters = _block(width)
    b.forward(e.empty((9, 8), F), sequences=3)
    kept, norm = e.lib.touched() - parameters, b.norm
    b.step(e.empty((sequences, 8), F), b.new_states(sequences))
    assert not kept & (e.lib.touched() - parameters) and b.norm is norm
    b.backward(e.empty((9, 8), F))
    assert {b.uz.ptr, b.c.ptr, b.dbc.ptr, b.delta.ptr, b.y.ptr, b.saved.ptr, *(m.ptr for m in norm)} <= e.lib.touched() & kept
