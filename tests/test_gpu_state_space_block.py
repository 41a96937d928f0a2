"""The operators together, as a layer: forward, backward, a prompt continued token by token, and training steps from a recording."""
import numpy as np
import pytest

import state_space_reference as R
from parallelreverseautodiff_b200 import engine as E
from parallelreverseautodiff_b200.networks import StateSpaceBlock

pytestmark = pytest.mark.gpu


def _block(e, dtype, r, dim=12, inner=20, state=6, groups=2, width=3, norm_groups=4, dropout=0.0):
    b = StateSpaceBlock(e, dtype, dim, inner, state, groups, 5, width, norm_groups, dropout, seed=77)
    p = {k: r.standard_normal(v.shape) * (v.shape[0] ** -0.5 if k.startswith("W") else 0.3) for k, v in b.p.items()}
    p["A"] = -r.uniform(0.1, 2, p["A"].shape)
    p["gamma"] += 1
    p["Wc"] = r.standard_normal(p["Wc"].shape) * 0.5
    b.set_parameters(p)
    return b, p


def _reference(b, p, x, lengths, states=None, keep=None):
    """The layer in 64 bits from the operators' references."""
    n = b.groups * b.state
    uz = x @ p["Win"]
    u, z = uz[:, :b.inner], uz[:, b.inner:]
    c = R.conv(u, p["Wc"], p["bc"], states and states["conv"], lengths)["y"]
    dbc = c @ p["Wx"]
    y = R.scan(c, dbc[:, :b.rank] @ p["Wdt"], p["A"], dbc[:, b.rank:b.rank + n], dbc[:, b.rank + n:], p["D"], z, p["bdt"],
               states and states["h"], lengths, b.groups)["y"]
    v = R.group_norm(y, len(x), 1, b.norm_groups, p["gamma"], p["beta"])[0]["y"] @ p["Wout"]
    if keep is not None:
        v = np.where(keep, v / (1 - b.p_drop), 0)
    return x + v


def test_forward_and_gradients(engine):
    """Forward against the references; every gradient against central differences of them, along a random direction: h = 1e-5 leaves
    about h^2 = 1e-10 from third derivatives and 1e-16 / h = 1e-11 from rounding, relative to values of order one to a hundred here."""
    e, r = engine, np.random.default_rng(21)
    lengths = [5, 0, 37, 1]
    b, p = _block(e, np.float64, r, dropout=0.25)
    T = sum(lengths)
    x, d_out = r.standard_normal((T, b.dim)), r.standard_normal((T, b.dim))
    states = {"conv": r.standard_normal((4, 2 * b.inner)), "h": r.standard_normal((4, b.inner * b.state))}
    keep = (R.philox(T * b.dim, 77, 3) < np.floor(0.75 * 2 ** 32 + 0.5)).reshape(T, b.dim)
    step = e.dropout_step(3)
    out = b.forward(e.upload(x), e.sequence_offsets(lengths), 4, {k: e.upload(v) for k, v in states.items()}, step=step)
    want = _reference(b, p, x, lengths, states, keep)
    assert np.abs(out.numpy() - want).max() < 1e-11 * (1 + np.abs(want).max())
    d_x = b.backward(e.upload(d_out)).numpy()
    got = {**{k: v.numpy() for k, v in b.g.items()}, "x": d_x, "conv": b.d_states["conv"].numpy(), "h": b.d_states["h"].numpy()}
    for k in got:
        src = x if k == "x" else states[k] if k in states else p[k]
        dv = r.standard_normal(src.shape)

        def value(h):
            at = {**p, **states, "x": x, k: src + h * dv}
            return (_reference(b, at, at["x"], lengths, {q: at[q] for q in states}, keep) * d_out).sum()

        along, scale = (got[k].reshape(src.shape) * dv).sum(), np.abs(got[k].reshape(src.shape) * dv).sum()
        assert abs(along - (value(1e-5) - value(-1e-5)) / 2e-5) < 1e-7 * (scale + 1), k


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("width", [1, 4])
def test_tokens_one_by_one_continue_a_prompt(engine, dtype, width):
    """The same rows in one call and as a prompt and single tokens: each token's value takes a few hundred roundings over the layer and
    four in front of it, values of order ten."""
    e, r = engine, np.random.default_rng(8)
    b, p = _block(e, dtype, r, width=width)
    S, P, more = 3, 6, 4
    x = r.standard_normal((S, P + more, b.dim)).astype(dtype)
    up = lambda a: e.upload(np.ascontiguousarray(a.reshape(-1, b.dim)))  # noqa: E731
    whole = b.forward(up(x), sequences=S, training=False).numpy().reshape(x.shape)
    states = b.new_states(S)
    y = b.forward(up(x[:, :P]), sequences=S, states_out=states, training=False).numpy().reshape(S, P, b.dim)
    limit = 4000 * np.finfo(dtype).eps * 10
    assert np.abs(y - whole[:, :P]).max() < limit
    for t in range(P, P + more):
        y = b.step(up(x[:, t]), states).numpy()
        assert np.abs(y - whole[:, t]).max() < limit, t


def test_recorded_training_steps(engine):
    """Forward, backward and Adam recorded once and replayed with the step counted on, against the same steps called one by one."""
    r0 = 5
    results = []
    for recorded in (False, True):
        with E.Engine(0) as e:
            r = np.random.default_rng(r0)
            b, _ = _block(e, np.float32, r, dim=32, inner=64, state=16, groups=1, width=4, norm_groups=2, dropout=0.1)
            lengths = [50, 3, 200]
            x, d_out = (e.upload(r.standard_normal((253, 32)).astype(np.float32)) for _ in range(2))
            off, step = e.sequence_offsets(lengths), e.dropout_step(0)
            names = list(b.p)
            m, v = ([e.zeros(b.p[k].shape, np.float32) for k in names] for _ in range(2))

            def train():
                b.forward(x, off, 3, step=step)
                b.backward(d_out)
                e.adam([b.p[k] for k in names], [b.g[k] for k in names], m, v, 1e-3, 0.9, 0.999, 1e-8, 1.0)

            def count(k):
                e.copy(step, e.dropout_step(k))

            train()
            e.sync()
            sequence = e.record(train) if recorded else None
            for k in range(1, 4):
                count(k)
                sequence.launch() if recorded else train()
            results.append({k: b.p[k].numpy() for k in names})
            if recorded:
                sequence.close()
    for k in results[0]:
        assert np.array_equal(results[0][k], results[1][k]), k
