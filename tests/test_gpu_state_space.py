"""State space operators on the GPU against numpy in 64 bits.

Tolerances.  A result is a sum of products; its magnitude M is that sum with every term's absolute value (the reference computes
it).  A term's factors and the additions above it are each off by half a step e (2^-24, 2^-53), so a result is off by at most
K e M with K the number of roundings on the longest way from an input to it:
  scan      a token's decay exp(dt A): dt (8: bias, softplus), the product and the factor log2 e (2 |dt A|), the exponential (4, and
            its argument's error, 8 |dt A|); times the state and added to it, 2.  Over T tokens both ways T (16 + 10 max|dt A|) x 2, the
            rest (products, gate, sums over channels, states and tokens in a tree) within 64 + T.
  conv      width + 12 roundings, sums over T tokens T more.
  norm      16, and the sums over n values: at most n / 32 + 16 additions in a row.
"""
import ctypes as C

import numpy as np
import pytest

import state_space_reference as R
from parallelreverseautodiff_b200 import _lib
from parallelreverseautodiff_b200 import engine as E
from util import HEADROOM

pytestmark = pytest.mark.gpu
F = {"f32": np.float32, "f64": np.float64}
STEP = {"f32": 2.0 ** -24, "f64": 2.0 ** -53}


def near(got, want, limit, what):
    got = got.astype(np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    limit = np.broadcast_to(limit, want.shape)
    err = np.abs(got - want)
    if err.size:
        HEADROOM[what] = max(HEADROOM.get(what, 0.0), float((err / np.maximum(limit, 1e-300)).max()))
    bad = ~(err <= limit)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, worst {err[bad].max():.3e} at {np.argwhere(bad)[0]}"


def scan_case(r, f, T, d, n, q, S, z=True, D=True, bias=True, h0=True):
    x = dict(u=r.standard_normal((T, d)), delta=r.standard_normal((T, d)) * 0.7 - 1, A=-r.uniform(0.05, 3, (d, n)),
             B=r.standard_normal((T, q * n)), C=r.standard_normal((T, q * n)))
    if D:
        x["D"] = r.standard_normal(d)
    if z:
        x["z"] = r.standard_normal((T, d))
    if bias:
        x["delta_bias"] = r.standard_normal(d) * 0.5
    if h0:
        x["h0"] = r.standard_normal((S, d * n))
    return {k: v.astype(f) for k, v in x.items()}


def check_scan(e, dtype, lengths, d, n, q=1, packed=True, softplus=True, **options):
    f, T, S = F[dtype], sum(lengths), len(lengths)
    r = np.random.default_rng(T * 131 + d * 7 + n + q)
    x = scan_case(r, f, T, d, n, q, S, **options)
    if not softplus:
        x["delta"] = np.abs(x["delta"]).astype(f)
        if "delta_bias" in x:
            x["delta_bias"] = np.abs(x["delta_bias"]).astype(f)
    dy = r.standard_normal((T, d)).astype(f)
    want = R.scan(**x, lengths=lengths, groups=q, delta_softplus=softplus, dy=dy)
    size = R.scan(**x, lengths=lengths, groups=q, delta_softplus=softplus, dy=dy, magnitude=True)
    raw = x["delta"].astype(np.float64) + x.get("delta_bias", 0)
    most = float(np.abs((R.softplus(raw) if softplus else raw).max() * x["A"].min()))
    longest = max(lengths)
    limit = (longest * (16 + 10 * most) * 2 + T + 64) * STEP[dtype]
    dev = {k: e.upload(v) for k, v in x.items()}
    of = dict(dev, sequences=S, groups=q, delta_softplus=softplus)
    if packed:
        of["offsets"] = e.sequence_offsets(lengths)
    y, last, saved = e.selective_scan_forward(**of, h_last=True, save=True)
    grads = e.selective_scan_backward(**of, saved=saved, dy=e.upload(dy))
    near(y.numpy(), want["y"], limit * size["y"], f"scan y {dtype}")
    near(last.numpy(), want["last"], limit * size["last"], f"scan last {dtype}")
    assert set(grads) == set(x)
    for k, m in grads.items():
        near(m.numpy(), want[k].reshape(m.shape), limit * size[k].reshape(m.shape), f"scan d{k} {dtype}")
    y2, none, no_saved = e.selective_scan_forward(**of)       # the same without what it need not leave
    assert none is None and no_saved is None and np.array_equal(y2.numpy(), y.numpy())


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("lengths", [[1], [2, 1], [31], [32], [33], [64, 0, 1], [5, 0, 0, 40, 33, 1], [0, 0, 7, 0], [16, 16, 17, 15]])
@pytest.mark.parametrize("d,n,q", [(5, 1, 1), (33, 16, 1), (40, 3, 2)])
def test_scan_of_packed_sequences(engine, dtype, lengths, d, n, q):
    check_scan(engine, dtype, lengths, d, n, q)


@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_many_sequences_of_a_token_or_two(engine, dtype):
    lengths = [1] * 40 + [0] * 3 + [2] * 30 + [0, 3, 0, 0, 1]
    check_scan(engine, dtype, lengths, 70, 16)
    check_scan(engine, dtype, [1] * 90, 24, 5, 3, packed=False)
    e, f, r = engine, F[dtype], np.random.default_rng(1)
    T, S, d = sum(lengths), len(lengths), 20
    x = {k: r.standard_normal(s).astype(f) for k, s in (("x", (T, d)), ("w", (d, 4)), ("bias", (d,)), ("state", (S, 3 * d)))}
    dy = r.standard_normal((T, d)).astype(f)
    want, size = (R.conv(**x, lengths=lengths, dy=dy, magnitude=m) for m in (False, True))
    of = dict({k: e.upload(v) for k, v in x.items()}, offsets=e.sequence_offsets(lengths), sequences=S)
    y, last = e.causal_conv_forward(**of, state_out=True)
    near(y.numpy(), want["y"], 16 * STEP[dtype] * size["y"], f"conv y {dtype}")
    assert np.array_equal(last.numpy(), want["last"].astype(f))
    for k, m in e.causal_conv_backward(**of, dy=e.upload(dy)).items():
        near(m.numpy(), want[k], (16 + (T if k in ("w", "bias") else 0)) * STEP[dtype] * size[k], f"conv d{k} {dtype}")


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("n", [1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 128])
@pytest.mark.parametrize("d,q", [(1, 1), (66, 2)])
def test_scan_of_every_number_of_states(engine, dtype, n, d, q):
    check_scan(engine, dtype, [37, 3], d, n, q)


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("lengths", [[700], [301, 1, 0, 260], [129] * 5])
def test_scan_in_spans(engine, dtype, lengths):
    """Few channels and many tokens: spans that begin inside sequences, with and without offsets."""
    check_scan(engine, dtype, lengths, 20, 8, 2)
    if len(set(lengths)) == 1:
        check_scan(engine, dtype, lengths, 20, 8, 2, packed=False)


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("n", [8, 16, 32, 64, 128])
def test_scan_of_many_channels_in_spans(engine, dtype, n):
    """Sums of dB and dC over several CTAs' channels, tile by tile, where the states fill the lanes."""
    check_scan(engine, dtype, [3, 700, 45, 0, 301], 150, n)


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("lengths,d", [([50] * 3, 33), ([1] * 9, 64), ([7] * 40, 5), ([100] * 30, 700)])
def test_scan_of_equal_sequences(engine, dtype, lengths, d):
    check_scan(engine, dtype, lengths, d, 6, packed=False)


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("absent", ["z", "D", "bias", "h0"])
@pytest.mark.parametrize("softplus", [True, False])
def test_scan_without_some_inputs(engine, dtype, absent, softplus):
    check_scan(engine, dtype, [40, 3, 20], 34, 10, 2, softplus=softplus, **{absent: False})


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("lengths,d,n", [([40, 0, 3], 5, 3), ([700], 33, 16), ([1500, 900], 9, 70)])
def test_steps_of_no_time_leave_the_states_as_they_are(engine, dtype, lengths, d, n):
    """A decay over no time is 1 exactly, however many tokens it is repeated for, and both ways."""
    e, f, T, S = engine, F[dtype], sum(lengths), len(lengths)
    x = scan_case(np.random.default_rng(T), f, T, d, n, 1, S, z=False, D=False, bias=False)
    x["delta"][:] = 0
    x["C"][:] = 0
    dev = {k: e.upload(v) for k, v in x.items()}
    of = dict(dev, sequences=S, offsets=e.sequence_offsets(lengths), delta_softplus=False)
    _, last, saved = e.selective_scan_forward(**of, h_last=True, save=True)
    assert np.array_equal(last.numpy(), x["h0"])
    # only the last tokens ask for a state: its gradient reaches the first one unchanged
    ends = np.cumsum(lengths) - 1
    x["C"][ends] = 1
    dy = np.zeros((T, d), f)
    dy[ends] = 0.375
    grads = e.selective_scan_backward(**dict(of, C=e.upload(x["C"])), saved=saved, dy=e.upload(dy))
    want = np.repeat([0.375 if m else 0.0 for m in lengths], d * n).reshape(S, d * n)
    assert np.array_equal(grads["h0"].numpy(), want.astype(f))


def test_scan_gradients_against_differences(engine):
    """The double kernels against central differences of their own forward, along one random direction in all inputs at once.
    With h = 1e-5 the third derivatives leave about h^2 = 1e-10 of the functional's scale, rounding 1e-16 / h = 1e-11 of it."""
    e, r = engine, np.random.default_rng(11)
    lengths, d, n, q = [70, 0, 33, 1], 37, 12, 1
    T = sum(lengths)
    x = scan_case(r, np.float64, T, d, n, q, 4)
    dy = r.standard_normal((T, d))
    dx = {k: r.standard_normal(v.shape) for k, v in x.items()}
    off = e.sequence_offsets(lengths)

    def value(h):
        return float((e.selective_scan_forward(**{k: e.upload(v + h * dx[k]) for k, v in x.items()}, offsets=off, sequences=4)[0].numpy() * dy).sum())

    dev = {k: e.upload(v) for k, v in x.items()}
    _, _, saved = e.selective_scan_forward(**dev, offsets=off, sequences=4, save=True)
    g = e.selective_scan_backward(**dev, offsets=off, sequences=4, saved=saved, dy=e.upload(dy))
    along = sum((g[k].numpy() * dx[k]).sum() for k in x)
    scale = sum(np.abs(g[k].numpy() * dx[k]).sum() for k in x)
    assert abs(along - (value(1e-5) - value(-1e-5)) / 2e-5) < 1e-7 * scale


@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_columns_of_wider_matrices_and_rows_of_no_sequence(engine, dtype):
    """u and z are the halves of one matrix, delta, B and C columns of another; rows in front of the first sequence and behind the
    last hold NaN, are not read, and results there stay as they were."""
    e, f, r = engine, F[dtype], np.random.default_rng(3)
    lengths, front, back, d, n = [40, 2, 60], 5, 9, 36, 7
    T = sum(lengths)
    x = scan_case(r, f, T, d, n, 1, 3)
    dy = r.standard_normal((T, d)).astype(f)
    pad = lambda m: np.concatenate([np.full((front, m.shape[1]), np.nan, f), m, np.full((back, m.shape[1]), np.nan, f)])  # noqa: E731
    uz = e.upload(np.concatenate([pad(x["u"]), pad(x["z"])], 1))
    dbc = e.upload(np.concatenate([pad(x["delta"]), pad(x["B"]), pad(x["C"])], 1))
    rows, wide = T + front + back, d + 2 * n
    off = e._upload_raw((np.concatenate([[0], np.cumsum(lengths)]) + front).astype(np.int32))
    of = dict(u=uz.view((rows, d)), z=uz.view((rows, d), d), delta=dbc.view((rows, d)), B=dbc.view((rows, n), d),
              C=dbc.view((rows, n), d + n), **{k: e.upload(x[k]) for k in ("A", "D", "delta_bias", "h0")}, offsets=off, sequences=3,
              pitches=dict(u=2 * d, z=2 * d, delta=wide, B=wide, C=wide))
    marked = lambda *shape: e.upload(np.full(shape, 7.0, f))  # noqa: E731
    y = marked(rows, d + 3)
    _, last, saved = e.selective_scan_forward(**of, out=y, ld_y=d + 3, h_last=True, save=True)
    duz, ddbc = marked(rows, 2 * d), marked(rows, wide)
    out = dict(u=duz.view((rows, d)), z=duz.view((rows, d), d), delta=ddbc.view((rows, d)), B=ddbc.view((rows, n), d),
               C=ddbc.view((rows, n), d + n), **{k: e.empty(x[k].shape, f) for k in ("A", "D", "delta_bias", "h0")})
    dyp = e.upload(pad(dy))
    e.selective_scan_backward(**of, saved=saved, dy=dyp, out=out, gradient_pitches=dict(u=2 * d, z=2 * d, delta=wide, B=wide, C=wide))
    dense = {k: e.upload(v) for k, v in x.items()}
    off0 = e.sequence_offsets(lengths)
    y0, last0, saved0 = e.selective_scan_forward(**dense, offsets=off0, sequences=3, h_last=True, save=True)
    g0 = {k: m.numpy() for k, m in e.selective_scan_backward(**dense, offsets=off0, sequences=3, saved=saved0, dy=e.upload(dy)).items()}
    e2 = 400 * 100 * STEP[dtype]       # other tiles, the same sums: as in the module's bound with T = 102
    got = y.numpy()
    assert (got[:front] == 7).all() and (got[front + T:] == 7).all() and (got[:, d:] == 7).all()
    near(got[front:front + T, :d], y0.numpy().astype(np.float64), e2 * (1 + np.abs(y0.numpy()).max()), f"padded scan {dtype}")
    near(last.numpy(), last0.numpy().astype(np.float64), e2 * (1 + np.abs(last0.numpy()).max()), f"padded scan {dtype}")
    guz, gdbc = duz.numpy(), ddbc.numpy()
    for m in (guz, gdbc):
        assert (m[:front] == 7).all() and (m[front + T:] == 7).all()
    got = dict(u=guz[front:front + T, :d], z=guz[front:front + T, d:], delta=gdbc[front:front + T, :d], B=gdbc[front:front + T, d:d + n],
               C=gdbc[front:front + T, d + n:], **{k: out[k].numpy() for k in ("A", "D", "delta_bias", "h0")})
    for k in got:
        near(got[k], g0[k].astype(np.float64).reshape(got[k].shape), e2 * (1 + np.abs(g0[k]).max()), f"padded scan {dtype}")


def test_a_sequence_of_infinities_stays_alone(engine):
    e, f, r = engine, np.float32, np.random.default_rng(9)
    lengths, d, n = [70, 50, 90], 12, 4
    x = scan_case(r, f, 210, d, n, 1, 3)
    dy = r.standard_normal((210, d)).astype(f)
    off = e.sequence_offsets(lengths)

    def run(x):
        dev = {k: e.upload(v) for k, v in x.items()}
        y, last, saved = e.selective_scan_forward(**dev, offsets=off, sequences=3, h_last=True, save=True)
        g = e.selective_scan_backward(**dev, offsets=off, sequences=3, saved=saved, dy=e.upload(dy))
        return {"y": y.numpy(), "last": last.numpy(), **{k: g[k].numpy() for k in ("u", "delta", "z", "B", "C", "h0")}}

    clean = run(x)
    bad = {k: v.copy() for k, v in x.items()}
    bad["u"][70:120:7] = np.inf
    bad["delta"][75] = np.nan
    bad["h0"][1] = -np.inf
    got = run(bad)
    for k, v in got.items():
        rows = np.r_[0:70, 120:210] if v.shape[0] == 210 else np.r_[0, 2]
        assert np.array_equal(v[rows], clean[k][rows]), k
    assert not np.isfinite(got["y"][70:120]).all()


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("batch,d,n,q,width", [(1, 1, 1, 1, 1), (3, 40, 16, 1, 4), (5, 33, 10, 3, 3), (2, 18, 128, 2, 8), (1, 260, 33, 1, 2)])
def test_single_tokens_continue_a_prompt(engine, dtype, batch, d, n, q, width):
    """A prompt, then three tokens one by one, the states in place: the rows of the whole sequences in one call, as near as the
    orders of their sums allow."""
    e, f, r = engine, F[dtype], np.random.default_rng(batch + d)
    P, more = 9, 3
    T = P + more
    x = scan_case(r, f, batch * T, d, n, q, batch)
    w, cb = (r.standard_normal((d, width)) * 0.5).astype(f), r.standard_normal(d).astype(f)
    cs = r.standard_normal((batch, (width - 1) * d)).astype(f) if width > 1 else None
    up = lambda a: None if a is None else e.upload(np.ascontiguousarray(a))  # noqa: E731
    fixed = {k: up(x[k]) for k in ("A", "D", "delta_bias")}

    def part(k, a, b):
        return up(x[k].reshape(batch, T, -1)[:, a:b].reshape(batch * (b - a), -1))

    def prompt(length, conv_state, h0):
        u, cs1 = e.causal_conv_forward(part("u", 0, length), up(w), up(cb), conv_state, sequences=batch, state_out=width > 1 or None)
        y, h, _ = e.selective_scan_forward(u, **{k: part(k, 0, length) for k in ("delta", "B", "C", "z")}, **fixed, h0=h0, sequences=batch,
                                           groups=q, h_last=True)
        return y, cs1, h

    whole, cs_end, h_end = prompt(T, up(cs), up(x["h0"]))
    y, state, h = prompt(P, up(cs), up(x["h0"]))
    whole = whole.numpy().reshape(batch, T, d).astype(np.float64)
    size = R.scan(**{**x, "u": np.abs(whole.reshape(-1, d)) + 10}, lengths=[T] * batch, groups=q, magnitude=True)["y"].max()
    limit = 2 * (T * (16 + 10 * 9) * 2 + 64) * STEP[dtype] * size
    near(y.numpy().reshape(batch, P, d), whole[:, :P], limit, f"prompt {dtype}")
    state = state if state is not None else e.zeros((batch, 1), f)
    for t in range(P, T):
        u = e.causal_conv_step(part("u", t, t + 1), up(w), state, bias=up(cb))
        y = e.selective_scan_step(u, **{k: part(k, t, t + 1) for k in ("delta", "B", "C", "z")}, **fixed, h=h, groups=q)
        near(y.numpy(), whole[:, t], limit, f"step {dtype}")
    near(h.numpy(), h_end.numpy().astype(np.float64), limit, f"step state {dtype}")
    if cs_end is not None:
        assert np.array_equal(state.numpy(), cs_end.numpy())


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("lengths,d", [([1], 1), ([3, 0, 2, 1, 40, 0], 12), ([31, 32, 33, 257], 33), ([600, 0], 132)])
@pytest.mark.parametrize("swish", [True, False])
def test_conv(engine, dtype, width, lengths, d, swish):
    e, f, r = engine, F[dtype], np.random.default_rng(d + width)
    T, S = sum(lengths), len(lengths)
    x = dict(x=r.standard_normal((T, d)), w=r.standard_normal((d, width)))
    if width % 2 == 0:
        x["bias"] = r.standard_normal(d)
        x["state"] = r.standard_normal((S, (width - 1) * d))
    x = {k: v.astype(f) for k, v in x.items()}
    dy = r.standard_normal((T, d)).astype(f)
    want, size = (R.conv(**x, lengths=lengths, swish_=swish, dy=dy, magnitude=m) for m in (False, True))
    dev = {k: e.upload(v) for k, v in x.items()}
    of = dict(dev, offsets=e.sequence_offsets(lengths), sequences=S, swish=swish)
    y, last = e.causal_conv_forward(**of, state_out=width > 1 or None)
    g = e.causal_conv_backward(**of, dy=e.upload(dy))
    limit = (width + 12) * STEP[dtype]
    near(y.numpy(), want["y"], limit * size["y"], f"conv y {dtype}")
    if width > 1:
        assert np.array_equal(last.numpy(), want["last"].astype(f))
    for k, m in g.items():
        near(m.numpy(), want[k], (limit + (T * STEP[dtype] if k in ("w", "bias") else 0)) * size[k], f"conv d{k} {dtype}")


@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_conv_of_equal_sequences_in_wider_matrices(engine, dtype):
    e, f, r = engine, F[dtype], np.random.default_rng(2)
    S, n, d, W = 5, 21, 24, 4
    wide = r.standard_normal((S * n, 2 * d)).astype(f)
    w, dy = r.standard_normal((d, W)).astype(f), r.standard_normal((S * n, d)).astype(f)
    m, y, dx = e.upload(wide), e.upload(np.full((S * n, d + 4), 7, f)), e.upload(np.full((S * n, 2 * d), 7, f))
    x = m.view((S * n, d), d)
    e.causal_conv_forward(x, e.upload(w), sequences=S, out=y, ld_x=2 * d, ld_y=d + 4)
    out = {"x": dx.view((S * n, d), d), "w": e.empty((d, W), f)}
    e.causal_conv_backward(x, e.upload(w), e.upload(dy), sequences=S, out=out, ld_x=2 * d, ld_dx=2 * d)
    want, size = (R.conv(wide[:, d:], w, lengths=[n] * S, dy=dy, magnitude=k) for k in (False, True))
    limit = 16 * STEP[dtype]
    near(y.numpy()[:, :d], want["y"], limit * size["y"], f"conv y {dtype}")
    near(dx.numpy()[:, d:], want["x"], limit * size["x"], f"conv dx {dtype}")
    near(out["w"].numpy(), want["w"], (limit + S * n * STEP[dtype]) * size["w"], f"conv dw {dtype}")
    assert (y.numpy()[:, d:] == 7).all() and (dx.numpy()[:, :d] == 7).all()


NORMS = [(1, 1, 1, 1), (3, 1, 12, 4), (70, 1, 96, 8), (5, 1, 130, 1), (33, 1, 2048, 16), (2, 1, 1024, 1), (2, 1, 4100, 2), (7, 1, 36, 12),
         (1, 5, 7, 7), (3, 49, 60, 5), (4, 300, 96, 8), (2, 1000, 33, 3), (2, 9, 3000, 2), (1, 4000, 4, 2), (300, 2, 16, 4), (1, 64, 520, 130)]


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("samples,positions,channels,groups", NORMS)
@pytest.mark.parametrize("swish,plain", [(True, False), (False, True)])
def test_group_norm(engine, dtype, samples, positions, channels, groups, swish, plain):
    e, f, r = engine, F[dtype], np.random.default_rng(channels + positions)
    x = (r.standard_normal((samples * positions, channels)) * 2 + 0.5).astype(f)
    dy = r.standard_normal(x.shape).astype(f)
    gamma, beta = (None, None) if plain else (r.standard_normal(channels).astype(f), r.standard_normal(channels).astype(f))
    want, size = R.group_norm(x, samples, positions, groups, gamma, beta, swish_=swish, dy=dy)
    up = lambda a: None if a is None else e.upload(a)  # noqa: E731
    dev, g, b = e.upload(x), up(gamma), up(beta)
    y, mean, rstd = e.group_norm_forward(dev, groups, g, b, positions=positions, swish=swish)
    dx, dgamma, dbeta = e.group_norm_backward(dev, mean, rstd, e.upload(dy), groups, g, b, positions=positions, swish=swish)
    n = positions * channels // groups
    limit = (16 + 16 + n / 32) * STEP[dtype]
    columns = limit + (samples * positions / 8 + 16) * STEP[dtype]
    for k, m, lim in (("y", y, limit), ("mean", mean, limit), ("rstd", rstd, limit), ("x", dx, 2 * limit), ("gamma", dgamma, 2 * columns),
                      ("beta", dbeta, 2 * columns)):
        near(m.numpy(), want[k], lim * size[k], f"norm {k} {dtype}")


@pytest.mark.parametrize("positions", [1, 200])
def test_group_norm_far_from_zero(engine, positions):
    """A mean a thousand deviations away: xhat's error stays that of x itself (2^-24 of 1000) and of some additions."""
    e, r = engine, np.random.default_rng(0)
    x = (r.standard_normal((4 * positions, 64)) + 1000).astype(np.float32)
    want, size = R.group_norm(x, 4, positions, 4)
    y, mean, rstd = e.group_norm_forward(e.upload(x), 4, positions=positions)
    n = positions * 16
    # mean: one rounding, 6e-5; the variance around it: as of values of size one
    near(y.numpy(), want["y"], (4 + n / 32) * 2.0 ** -24 * size["y"], "norm far from zero")
    near(rstd.numpy(), want["rstd"], 64 * 2.0 ** -24 * want["rstd"] * (1 + n / 32), "norm far from zero, rstd")


def test_group_norm_of_a_group_with_nan(engine):
    e, r = engine, np.random.default_rng(0)
    for positions in (1, 30):
        x = r.standard_normal((3 * positions, 24)).astype(np.float32)
        clean = e.group_norm_forward(e.upload(x), 4, positions=positions)[0].numpy()
        x[positions, 7] = np.inf         # sample 1, group 1
        y = e.group_norm_forward(e.upload(x), 4, positions=positions)[0].numpy().reshape(3, positions, 4, 6)
        assert np.isnan(y[1, :, 1]).any()
        y[1, :, 1] = clean.reshape(y.shape)[1, :, 1]
        assert np.array_equal(y.reshape(clean.shape), clean)


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("n", [1, 3, 4, 5, 1023, 4096])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(engine, dtype, n, p):
    """The mask is the generator's, bit by bit; a kept value is the product with 1 / (1 - p) rounded to the type, one rounding, or two
    with the residual; a dropped one 0 whatever it was."""
    e, f, r = engine, F[dtype], np.random.default_rng(n)
    x, res = r.standard_normal(n).astype(f), r.standard_normal(n).astype(f)
    seed, offset = (1 << 63) + 12345, (1 << 40) + 7
    keep = R.philox(n, seed, offset) < np.floor((1 - p) * 2.0 ** 32 + 0.5)
    x[~keep] = np.where(np.arange((~keep).sum()) % 2, np.nan, np.inf)
    with np.errstate(divide="ignore", invalid="ignore"):
        want = np.where(keep, x.astype(np.float64) / (1 - p), 0)
    y = e.dropout(e.upload(x), p, seed, offset).numpy()
    assert (y[~keep] == 0).all()
    near(y, want, 3 * STEP[dtype] * np.abs(want), f"dropout {dtype}")
    y = e.dropout(e.upload(x), p, seed, offset, residual=e.upload(res)).numpy()
    near(y, want + res, 4 * STEP[dtype] * (np.abs(want) + np.abs(res)), f"dropout {dtype}")
    # the same words from an odd address, in place, and with the offset divided between the call and the device
    m = e.upload(np.concatenate([[0], x]).astype(f))
    view = m.view((n,), 1)
    e.dropout(view, p, seed, offset - 5, step=e.dropout_step(5), out=view)
    assert np.array_equal(m.numpy()[1:], e.dropout(e.upload(x), p, seed, offset).numpy())


def test_dropout_keeps_the_share_it_says(engine):
    """Among 2^20 independent words the share kept lies within six standard deviations (one in 10^9 by chance; the seed is fixed)."""
    e, n, p = engine, 1 << 20, 0.3
    y = e.dropout(e.upload(np.ones(n, np.float32)), p, 3, 1).numpy()
    assert abs((y != 0).mean() - 0.7) < 6 * np.sqrt(0.21 / n)
    z = e.dropout(e.upload(np.ones(n, np.float32)), p, 3, 2).numpy()
    assert abs(((y != 0) & (z != 0)).mean() - 0.49) < 6 * np.sqrt(0.25 / n)


def test_matrices_that_do_not_fit_are_refused(engine):
    e, f = engine, np.float32
    m = lambda *s: e.zeros(s, f)  # noqa: E731
    u, A, B = m(6, 8), m(8, 4), m(6, 4)
    off, last = e.sequence_offsets([6]), m(1, 32)
    good = dict(u=u, delta=u, A=A, B=B, C=B)
    for bad in (dict(delta=m(5, 8)), dict(B=m(6, 3)), dict(C=m(6, 5)), dict(D=m(7)), dict(z=m(6, 7)), dict(delta_bias=m(9)), dict(h0=m(1, 31)),
                dict(offsets=off, sequences=2), dict(out=m(6, 7)), dict(h_last=m(2, 32)), dict(save=m(31))):
        with pytest.raises(_lib.PradError) as err:
            e.selective_scan_forward(**{**good, **bad})
        assert err.value.status == _lib.ERR_SHAPE, bad
    _, _, saved = e.selective_scan_forward(**good, save=True)
    for bad in (dict(dy=m(6, 7)), dict(out=dict(u=u, delta=u, A=m(8, 3), B=B, C=B)), dict(out=dict(u=m(5, 8), delta=u, A=A, B=B, C=B))):
        with pytest.raises(_lib.PradError):
            e.selective_scan_backward(**{**good, "saved": saved, "dy": u, **bad})
    for call in (lambda: e.selective_scan_step(u, u, A, B, B, m(5, 32)), lambda: e.causal_conv_forward(u, m(7, 4)),
                 lambda: e.causal_conv_forward(u, m(8, 4), state=m(2, 24)), lambda: e.causal_conv_backward(u, m(8, 4), m(6, 9)),
                 lambda: e.causal_conv_step(u, m(8, 4), m(6, 16)), lambda: e.group_norm_forward(u, 2, gamma=m(7)),
                 lambda: e.group_norm_forward(u, 2, positions=4), lambda: e.group_norm_backward(u, m(6, 2), m(5, 2), u, 2),
                 lambda: e.dropout(u, 0.1, 1, residual=m(6, 7))):
        with pytest.raises(_lib.PradError) as err:
            call()
        assert err.value.status == _lib.ERR_SHAPE
    other = e.zeros((6, 8), np.float64)
    for call in (lambda: e.dropout(u, 0.1, 1, step=u), lambda: e.dropout(u, 0.1, 1, residual=other),
                 lambda: e.selective_scan_forward(**{**good, "delta": other}), lambda: e.selective_scan_forward(**good, offsets=m(2)),
                 lambda: e.causal_conv_forward(u, e.zeros((8, 4), np.float64)), lambda: e.group_norm_forward(u, 2, out=(other, m(6, 2), m(6, 2)))):
        with pytest.raises(_lib.PradError) as err:
            call()
        assert err.value.status == _lib.ERR_INVALID
    with pytest.raises(ValueError):
        e.sequence_offsets([3, -1])
    assert last.numpy().shape == (1, 32)


def test_what_was_not_saved_and_pitches_of_nothing_are_refused(engine):
    e = engine
    m = lambda *s: e.zeros(s, np.float32)  # noqa: E731
    u, A, B = m(20, 8), m(8, 4), m(20, 4)
    scan = dict(u=u, delta=u, A=A, B=B, C=B)
    _, _, saved = e.selective_scan_forward(**scan, save=True)
    assert saved.size == e.selective_scan_saved(20, 8, 4, np.float32)
    with pytest.raises(_lib.PradError) as err:          # what a shorter batch saved
        e.selective_scan_backward(**scan, saved=e.empty((saved.size - 1,), np.float32), dy=u)
    assert err.value.status == _lib.ERR_SHAPE
    with pytest.raises(_lib.PradError) as err:          # a forward that kept nothing
        e.selective_scan_backward(**scan, saved=None, dy=u)
    assert err.value.status == _lib.ERR_INVALID
    for call in (lambda: e.selective_scan_forward(**scan, pitches={"y": 8}), lambda: e.selective_scan_step(u, u, A, B, B, m(20, 32), pitches={"Z": 8}),
                 lambda: e.selective_scan_backward(**scan, saved=saved, dy=u, gradient_pitches={"dz": 8})):
        with pytest.raises(_lib.PradError) as err:
            call()
        assert err.value.status == _lib.ERR_INVALID


@pytest.mark.parametrize("dtype", ["f32", "f64"])
def test_matrices_at_odd_addresses(engine, dtype):
    """One value behind an allocation's start nothing can be read sixteen bytes at a time: the same values as at its start."""
    e, f, r = engine, F[dtype], np.random.default_rng(13)

    owners = []                          # (a view does not keep its matrix)

    def shifted(a):
        owners.append(e.upload(np.concatenate([[0], a.reshape(-1)]).astype(f)))
        return owners[-1].view(a.shape, 1)

    T, d, n = 75, 36, 8
    x = scan_case(r, f, T, d, n, 1, 2)
    dy, off = r.standard_normal((T, d)).astype(f), e.sequence_offsets([40, 35])
    w = r.standard_normal((d, 4)).astype(f)
    gamma = r.standard_normal(d).astype(f)
    limit = 400 * 75 * STEP[dtype]       # the same sums in another order: as in the module's bound with T = 75

    def run(up):
        dev = {k: up(v) for k, v in x.items()}
        y, last, saved = e.selective_scan_forward(**dev, offsets=off, sequences=2, h_last=True, save=True)
        g = e.selective_scan_backward(**dev, offsets=off, sequences=2, saved=saved, dy=up(dy))
        c, _ = e.causal_conv_forward(dev["u"], up(w), offsets=off, sequences=2)
        gc = e.causal_conv_backward(dev["u"], up(w), up(dy), offsets=off, sequences=2)
        out = [y, last, *(g[k] for k in sorted(g)), c, gc["x"], gc["w"]]
        for positions in (1, 25):
            v, mean, rstd = e.group_norm_forward(dev["u"], 3, up(gamma), positions=positions, swish=True)
            out += [v, mean, rstd, *e.group_norm_backward(dev["u"], mean, rstd, up(dy), 3, up(gamma), positions=positions, swish=True)]
        return [m.numpy().astype(np.float64) for m in out]

    for got, want in zip(run(shifted), run(e.upload)):
        near(got, want, limit * (1 + np.abs(want).max()), f"odd addresses {dtype}")


def test_empty_calls(engine):
    e, f = engine, np.float32
    x = e.empty((0, 8), f)
    A, B = e.upload(-np.ones((8, 4), f)), e.empty((0, 4), f)
    h0 = np.arange(64, dtype=f).reshape(2, 32)
    off = e.sequence_offsets([0, 0])
    y, last, saved = e.selective_scan_forward(x, x, A, B, B, h0=e.upload(h0), offsets=off, sequences=2, h_last=True, save=True)
    assert np.array_equal(last.numpy(), h0)
    g = e.selective_scan_backward(x, x, A, B, B, saved, x, h0=e.upload(h0), offsets=off, sequences=2)
    assert (g["A"].numpy() == 0).all() and (g["h0"].numpy() == 0).all()
    y, s = e.causal_conv_forward(x, e.upload(np.ones((8, 4), f)), state=e.upload(h0[:, :24].copy()), offsets=off, sequences=2, state_out=True)
    assert np.array_equal(s.numpy(), h0[:, :24])
    g = e.causal_conv_backward(x, e.upload(np.ones((8, 4), f)), x, state=e.upload(h0[:, :24].copy()), offsets=off, sequences=2)
    assert (g["w"].numpy() == 0).all() and (g["state"].numpy() == 0).all()
    dx, dg, db = e.group_norm_backward(x, e.empty((0, 2), f), e.empty((0, 2), f), x, 2)
    assert (dg.numpy() == 0).all() and (db.numpy() == 0).all()
    e.dropout(x, 0.5, 1)
    assert e.selective_scan_step(x, x, A, B, B, e.empty((0, 32), f)).shape == (0, 8)


def test_offsets_that_do_not_ascend_stay_inside(engine):
    """Wrong offsets give wrong rows, but every access stays inside: the call returns and neighbours of the results are untouched."""
    e, f, r = engine, np.float32, np.random.default_rng(1)
    T, d, n = 200, 8, 4
    x = scan_case(r, f, T, d, n, 1, 4)
    for marks in ([0, 150, 20, 90, 200], [-50, 30, 9999, 100, 400], [200, 100, 50, 20, 0], [0, 0, -7, 300, 300]):
        off = e._upload_raw(np.array(marks, np.int32))
        dev = {k: e.upload(v) for k, v in x.items()}
        y = e.upload(np.full((T + 2, d), 7, f))
        _, last, saved = e.selective_scan_forward(**dev, offsets=off, sequences=4, out=y.view((T, d), d), h_last=True, save=True)
        e.selective_scan_backward(**dev, offsets=off, sequences=4, saved=saved, dy=dev["u"])
        state = e.zeros((4, 3 * d), f)
        e.causal_conv_forward(dev["u"], e.zeros((d, 4), f), state=state, offsets=off, sequences=4, state_out=True)
        e.causal_conv_backward(dev["u"], e.zeros((d, 4), f), dev["z"], state=state, offsets=off, sequences=4)
        e.sync()
        got = y.numpy()
        assert (got[0] == 7).all() and (got[-1] == 7).all()


def test_recorded_layers_share_scratch_and_draw_new_masks(engine):
    """Two recordings of different sizes, replayed in turn with other inputs in their buffers, against the same calls unrecorded."""
    f, r = np.float32, np.random.default_rng(4)
    with E.Engine(0) as e:
        jobs = []
        for lengths, d, n in (([300, 41], 24, 8), ([90, 0, 20], 50, 16)):
            T = sum(lengths)
            dev = {k: e.upload(v) for k, v in scan_case(r, f, T, d, n, 1, len(lengths)).items()}
            w, dy, off, step = e.upload(r.standard_normal((d, 4)).astype(f)), e.upload(r.standard_normal((T, d)).astype(f)), e.sequence_offsets(lengths), e.dropout_step(0)

            def run(dev=dev, w=w, dy=dy, off=off, step=step, S=len(lengths)):
                c, _ = e.causal_conv_forward(dev["u"], w, offsets=off, sequences=S)
                of = {**dev, "u": c, "offsets": off, "sequences": S}
                y, last, saved = e.selective_scan_forward(**of, h_last=True, save=True)
                v, mean, rstd = e.group_norm_forward(y, 2)
                out = e.dropout(v, 0.3, 99, 0, residual=dev["u"], step=step)
                dv = e.dropout(dy, 0.3, 99, 0, step=step)
                dyn, _, _ = e.group_norm_backward(y, mean, rstd, dv, 2)
                g = e.selective_scan_backward(**of, saved=saved, dy=dyn)
                gc = e.causal_conv_backward(dev["u"], w, g["u"], offsets=off, sequences=S)
                return [out, last, gc["x"], gc["w"], g["A"], g["B"]]

            run()
            jobs.append((run, dev, step, T, d))
        recorded = []
        for run, dev, step, T, d in jobs:
            kept = []
            recorded.append((e.record(lambda: kept.extend(run())), kept))
        for turn in range(3):
            for (run, dev, step, T, d), (sequence, kept) in zip(jobs, recorded):
                e.upload(r.standard_normal((T, d)).astype(f), out=dev["u"])
                check = e._upload_raw(np.array([turn], np.uint64))
                e.copy(step, check)
                sequence.launch()
                got = [m.numpy() for m in kept]
                want = [m.numpy() for m in run()]
                for a, b in zip(got, want):
                    assert np.array_equal(a, b)
        for sequence, _ in recorded:
            sequence.close()


def test_two_contexts_at_once(engine):
    """Each context has its own stream and scratch: calls that overlap give what they give alone."""
    f, r = np.float32, np.random.default_rng(6)
    with E.Engine(0) as a, E.Engine(0) as b:
        x = scan_case(r, f, 1000, 64, 16, 1, 1)
        devs = [{k: e.upload(v) for k, v in x.items()} for e in (a, b)]
        alone = a.selective_scan_forward(**devs[0])[0].numpy()
        for _ in range(5):
            ys = [e.selective_scan_forward(**dev)[0] for e, dev in zip((a, b), devs)]
            assert all(np.array_equal(y.numpy(), alone) for y in ys)


def test_rows_beyond_the_first_four_gigabytes(engine):
    """A pitch that puts the last rows past 2^32 bytes and elements past 2^31: the same results as in a dense matrix."""
    e, f, r = engine, np.float32, np.random.default_rng(8)
    T, d, ld = 40, 8, 60_000_000
    if e.device_info()["free_bytes"] < 24 << 30:
        pytest.skip("needs 20 GB of device memory")
    x, w = r.standard_normal((T, d)).astype(f), r.standard_normal((d, 4)).astype(f)
    big = e.empty((T * ld,), f)
    dense = e.upload(x)
    _lib.check(e.lib.prad_copy_2d(e.ctx, big.ptr, ld * 4, dense.ptr, d * 4, d * 4, T))
    wd = e.upload(w)
    want = e.causal_conv_forward(dense, wd)[0].numpy()
    assert np.array_equal(e.causal_conv_forward(big.view((T, d)), wd, ld_x=ld)[0].numpy(), want)
    A, B = e.upload(-np.ones((d, 4), f)), e.upload(r.standard_normal((T, 4)).astype(f))
    want = e.selective_scan_forward(dense, dense, A, B, B)[0].numpy()
    got = e.selective_scan_forward(big.view((T, d)), big.view((T, d)), A, B, B, pitches=dict(u=ld, delta=ld))[0].numpy()
    assert np.array_equal(got, want)
