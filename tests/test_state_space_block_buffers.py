"""Which buffers the calls of a state space block work on: what one call keeps for another is not written by a third."""
import numpy as np
import pytest

from parallelreverseautodiff_b200 import _lib
from parallelreverseautodiff_b200.networks import StateSpaceBlock, SwinBlock
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


def test_a_backward_that_no_forward_fits_is_refused_before_its_first_launch():
    e, b, _ = _block()
    x, d_out = e.empty((9, 8), F), e.empty((9, 8), F)
    e.lib.taken()

    def refused(call, status):
        with pytest.raises(_lib.PradError) as err:
            call()
        assert err.value.status == status and not e.lib.taken()

    refused(lambda: b.backward(d_out), _lib.ERR_INVALID)
    for bad, status in ((e.empty((9, 7), F), _lib.ERR_SHAPE), (e.empty((9, 8), np.float64), _lib.ERR_INVALID)):
        refused(lambda: b.forward(bad), status)
        refused(lambda: b.step(bad, {}), status)
    b.forward(x, sequences=3)
    e.lib.taken()
    for bad in ((10, 8), (8, 8), (8, 9)):
        refused(lambda: b.backward(e.empty(bad, F)), _lib.ERR_SHAPE)
    refused(lambda: b.backward(e.empty((9, 8), np.float64)), _lib.ERR_SHAPE)
    b.backward(d_out)
    # an answer that keeps nothing, and a forward that was refused half way
    b.forward(x, sequences=3, training=False)
    e.lib.taken()
    refused(lambda: b.backward(d_out), _lib.ERR_INVALID)
    b.forward(x, sequences=3)
    with pytest.raises(_lib.PradError):
        b.forward(x, sequences=3, states={"conv": None, "h": e.empty((2, 48), F)})
    e.lib.taken()
    refused(lambda: b.backward(d_out), _lib.ERR_INVALID)


@pytest.mark.parametrize("recorded", ["step", "backward"])
def test_a_recorded_step_keeps_its_buffers(recorded):
    """Calls of other sizes behind a recording: what it was recorded with stays allocated until the sequence is closed."""
    e, b, parameters = _block()
    x, d_out, states = e.empty((9, 8), F), e.empty((9, 8), F), b.new_states(3)

    def train():
        b.forward(x, sequences=3, states=states)
        b.backward(d_out)

    train()
    e.lib.taken()
    sequence = e.record(train if recorded == "step" else lambda: b.backward(d_out))
    used = e.lib.touched()
    assert len(used - parameters) > 15
    for n in (12, 5):
        b.forward(e.empty((n, 8), F), sequences=1)
        b.step(e.empty((n, 8), F), b.new_states(n))
        b.backward(e.empty((n, 8), F))
    assert used <= set(e.lib.live)
    sequence.close()
    assert not used <= set(e.lib.live)


def test_a_recorded_attention_block_keeps_its_buffers():
    e = recording_engine()
    b = SwinBlock(e, F, 32, 2, 4)
    x, d_out = e.empty((8, 32), F), e.empty((8, 32), F)

    def train():
        b.forward(x)
        b.backward(d_out)

    train()
    e.lib.taken()
    sequence = e.record(train)
    used = e.lib.touched()
    b.forward(e.empty((12, 32), F))
    b.backward(e.empty((12, 32), F))
    assert used <= set(e.lib.live)
    sequence.close()


def test_results_are_the_callers_to_keep():
    """Several prompts and tokens in a row: none of the outputs is written again."""
    e, b, _ = _block()
    x, states = e.empty((9, 8), F), b.new_states(9)
    results = [*(b.forward(x, sequences=3, training=t) for t in (True, False)), *(b.step(x, states) for _ in range(3))]
    assert len({m.ptr for m in results}) == 5
