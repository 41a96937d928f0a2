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


def test_a_recorded_step_after_calls_of_other_sizes(engine):
    """Replayed behind them, with new allocations where the block's old buffers would be, it gives what it gave before them."""
    e, f, r = engine, np.float32, np.random.default_rng(6)
    b, _ = _block(e, f, r)
    x, d_out = (e.upload(r.standard_normal((9, b.dim)).astype(f)) for _ in range(2))

    def train():
        b.forward(x, sequences=3)
        b.backward(d_out)

    train()
    sequence = e.record(train)
    out, d_x = b.out, b.d_x
    sequence.launch()
    want = [m.numpy() for m in (out, d_x, *b.g.values())]
    for n in (6, 12):
        more = e.upload(r.standard_normal((n, b.dim)).astype(f))
        b.forward(more, sequences=1)
        b.step(more, b.new_states(n))
        b.backward(more)
    others = [e.upload(np.full(s, 7, f)) for s in ((9, b.inner), (9, 2 * b.inner), (9, b.dim), (9, b.columns), (9, b.norm_groups)) for _ in range(4)]
    sequence.launch()
    for m, w in zip((out, d_x, *b.g.values()), want):
        assert np.array_equal(m.numpy(), w)
    assert all((m.numpy() == 7).all() for m in others)
    sequence.close()


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
def test_padded_batches(engine, dtype):
    """Rows in front of the first sequence and behind the last: out and every gradient are those of the batch without them, whatever a
    batch before it left in the buffers.  The sums are the same, over some zeros more and in other tiles: a result is a sum of fewer
    than 100 products that have passed at most 60 roundings each, and the results here are sums of values of about their size."""
    e, r = engine, np.random.default_rng(15)
    b, p = _block(e, dtype, r)
    lengths, front, back = [12, 0, 7], 3, 5
    T = sum(lengths)
    rows = T + front + back
    full, padded = (e._upload_raw(np.array(m, np.int32)) for m in ([0, 9, 9, rows], np.cumsum([front] + lengths)))
    x, d_out = r.standard_normal((rows, b.dim)).astype(dtype), r.standard_normal((rows, b.dim)).astype(dtype)
    d_out[:front] = d_out[front + T:] = 0
    up = lambda a: e.upload(np.ascontiguousarray(a))  # noqa: E731

    def run(x, d_out, offsets):
        out = b.forward(up(x), offsets, 3)
        return {"out": out.numpy(), "x": b.backward(up(d_out)).numpy(), **{k: v.numpy() for k, v in b.g.items()}}

    inside = slice(front, front + T)
    want = run(x[inside], d_out[inside], e.sequence_offsets(lengths))
    run(x * 3, d_out + 1, full)          # every row of every buffer holds something
    for _ in range(2):
        got = run(x, d_out, padded)
        assert (got["x"][:front] == 0).all() and (got["x"][front + T:] == 0).all()
        got["out"], got["x"] = got["out"][inside], got["x"][inside]
        for k in want:
            assert np.abs(got[k] - want[k]).max() <= 6000 * np.finfo(dtype).eps / 2 * (1 + np.abs(want[k]).max()), k


def test_a_single_token_of_width_one(engine):
    e, r = engine, np.random.default_rng(2)
    x, w = r.standard_normal((5, 12)), r.standard_normal((12, 1))
    y = e.causal_conv_step(e.upload(x), e.upload(w), None, swish=False).numpy()
    assert np.array_equal(y, x * w[:, 0])
