"""How far a selective scan computed in a type of half step `e` may be off, result by result.

Every rounding is followed to where it ends up: a state's error decays with the state, so that the bound forgets as the scan does
instead of growing with the longest sequence.  Roundings of a value, each half a step (an approximate function of 2 units in the
last place counts four):
  raw = delta + bias     1
  dt = softplus(raw)     16 of its own (two approximate functions, a polynomial, products) and 2 |raw| of the exponential's argument
  swish, its slope, the sigmoid of x     12 of their own and 2 |x| of the argument
  decay = exp(dt A)      8 of its own, and its argument's: dt's, and 3 for the factor log2 e and the products; where spans are strung
                         together the argument is a sum over up to SPAN tokens, as many roundings of it
  state                  3 for dt u B, 1 for the sum
  sums over states       12: a lane's, the lanes'
  sums over channels     12 + channels / 8: a thread's, a warp's, the warps', the CTAs'
  sums over tokens       SPAN + 16 within a span, the spans in double
"""
import numpy as np

import state_space_reference as R

SPAN = 64        # tokens of a span: the least a float span has, and what the sizes that are compared with these bounds have


def scan_bounds(e, u, delta, A, B, C, D=None, z=None, delta_bias=None, h0=None, lengths=(), groups=1, delta_softplus=True, dy=None):
    """Largest errors of y, last and the gradients by name."""
    f = lambda x: None if x is None else np.asarray(x, np.float64)  # noqa: E731
    u, delta, A, B, C, D, z, bias, h0, dy = map(f, (u, delta, A, B, C, D, z, delta_bias, h0, dy))
    (T, d), n = u.shape, A.shape[1]
    ab = np.abs
    raw = delta + (bias if bias is not None else 0)
    e_raw = e * ab(raw) * (bias is not None)
    dt = R.softplus(raw) if delta_softplus else raw
    e_dt = e_raw * R.sigmoid(raw) + e * dt * (16 + 2 * ab(raw)) if delta_softplus else e_raw
    x, e_x = dt * u, e_dt * ab(u) + e * ab(dt * u)
    a = np.exp(dt[:, :, None] * A)
    r_a = 8 * e + ab(A) * (e_dt + (3 + SPAN) * e * ab(dt))[:, :, None]
    expand = lambda m: np.repeat(m.reshape(T, groups, n), d // groups, 1)  # noqa: E731
    Bd, Cd = expand(B), expand(C)
    h0 = h0.reshape(-1, d, n) if h0 is not None else np.zeros((len(lengths), d, n))
    h, before, e_h, e_before = (np.zeros((T, d, n)) for _ in range(4))
    last, at = np.zeros(h0.shape), 0
    for s, length in enumerate(lengths):
        now, off = h0[s], np.zeros((d, n))
        for t in range(at, at + length):
            before[t], e_before[t] = now, off
            off = a[t] * (off * (1 + r_a[t]) + r_a[t] * ab(now)) + (e_x[t][:, None] + 3 * e * ab(x[t])[:, None]) * ab(Bd[t])
            now = a[t] * now + x[t][:, None] * Bd[t]
            off = off + e * ab(now)
            h[t], e_h[t] = now, off
        last[s] = off
        at += length
    Dv = D if D is not None else np.zeros(d)
    r = (h * Cd).sum(2) + Dv * u
    e_r = (e_h * ab(Cd)).sum(2) + 12 * e * (ab(h * Cd)).sum(2) + 3 * e * ab(Dv * u)
    gate = R.swish(z) if z is not None else np.ones((T, d))
    k_z = e * (12 + 2 * ab(z)) if z is not None else np.zeros((T, d))
    out = {"y": ab(gate) * e_r + ab(r * gate) * (k_z + e), "last": last.reshape(len(lengths), d * n)}
    if dy is None:
        return out
    v = dy * gate
    e_v = ab(v) * (k_z + e)
    g, e_g, back, e_back = (np.zeros((T, d, n)) for _ in range(4))       # back: a g, what the token in front is handed
    dh0, at = np.zeros(h0.shape), 0
    for s, length in enumerate(lengths):
        now, off = np.zeros((d, n)), np.zeros((d, n))
        for t in range(at + length - 1, at - 1, -1):
            g[t] = Cd[t] * v[t][:, None] + now
            e_g[t] = ab(Cd[t]) * e_v[t][:, None] + off + 2 * e * (ab(Cd[t] * v[t][:, None]) + ab(now))
            now = a[t] * g[t]
            off = a[t] * (e_g[t] * (1 + r_a[t]) + r_a[t] * ab(g[t])) + e * ab(now)
            back[t], e_back[t] = now, off
        dh0[s] = off
        at += length
    w, e_w = back * before, e_back * ab(before) + ab(back) * e_before + e * ab(back * before)
    gB, e_gB = (g * Bd).sum(2), (e_g * ab(Bd)).sum(2) + 12 * e * ab(g * Bd).sum(2)
    wA, e_wA = (w * A).sum(2), (e_w * ab(A)).sum(2) + 15 * e * ab(w * A).sum(2)
    ddt, e_ddt = u * gB + wA, ab(u) * e_gB + e_wA + 3 * e * (ab(u * gB) + ab(wA))
    slope = R.sigmoid(raw) if delta_softplus else np.ones(raw.shape)
    ddelta = ddt * slope
    e_ddelta = e_ddt * slope + (e * ab(ddelta) * (12 + 2 * ab(raw)) + ab(ddt) * slope * (1 - slope) * e_raw) * delta_softplus
    rows = lambda m: m.reshape(T, groups, d // groups, n).sum(2).reshape(T, groups * n)  # noqa: E731
    over_tokens, over_channels = (SPAN + 16) * e, (12 + d / groups / 8) * e
    x3, v3 = x[:, :, None], v[:, :, None]
    out.update(u=ab(dt) * e_gB + e_dt * ab(gB) + ab(Dv) * e_v + 3 * e * (ab(dt * gB) + ab(Dv * v)), delta=e_ddelta,
               A=(e_w * ab(dt)[:, :, None] + ab(w) * e_dt[:, :, None] + over_tokens * ab(w * dt[:, :, None])).sum(0),
               B=rows(e_g * ab(x3) + ab(g) * e_x[:, :, None] + over_channels * ab(g * x3)),
               C=rows(e_h * ab(v3) + ab(h) * e_v[:, :, None] + over_channels * ab(h * v3)),
               D=(e_v * ab(u) + over_tokens * ab(v * u)).sum(0), delta_bias=(e_ddelta + over_tokens * ab(ddelta)).sum(0),
               h0=dh0.reshape(len(lengths), d * n))
    if z is not None:
        s = R.sigmoid(z)
        out["z"] = ab(dy) * (e_r * ab(R.swish_slope(z)) + ab(r) * s * (1 + ab(z)) * (k_z + 6 * e))
    return out
