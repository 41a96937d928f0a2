"""The state space operators in numpy and 64 bits, sequence by sequence and token by token, with the scale of their roundings.

Every function takes `magnitude`: with it, every term counts with its absolute value and nothing is subtracted, which gives for
each result the sum of the magnitudes of what was added up to get it.  A result computed in another order and precision is off by
at most (roundings along the longest chain of operations that ends in it) x (half a step) x (that magnitude), as every term is a
product of factors each off by a number of half steps."""
import numpy as np


def sigmoid(x):
    return np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))


def swish(x):
    return x * sigmoid(x)


def swish_slope(x, magnitude=False):
    s = sigmoid(x)
    return s * (1 + (np.abs(x) if magnitude else x) * (1 - s))


def softplus(x):
    return np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, h0=None, lengths=(), groups=1, delta_softplus=True, dy=None,
         magnitude=False):
    """y, last and, with dy, the gradients by name."""
    m = np.abs if magnitude else (lambda x: x)
    f = lambda x: None if x is None else np.asarray(x, np.float64)  # noqa: E731
    u, delta, A, B, C, D, z, bias, h0, dy = map(f, (u, delta, A, B, C, D, z, delta_bias, h0, dy))
    (T, d), n = u.shape, A.shape[1]
    raw = delta + (bias if bias is not None else 0)
    dt = softplus(raw) if delta_softplus else raw
    decay = np.exp(dt[:, :, None] * A)
    dtm, u = m(dt), m(u)
    expand = lambda x: np.repeat(m(x).reshape(T, groups, n), d // groups, 1)  # noqa: E731
    Bd, Cd = expand(B), expand(C)
    Dv = m(D) if D is not None else np.zeros(d)
    h0 = m(h0).reshape(-1, d, n) if h0 is not None else np.zeros((len(lengths), d, n))
    h, before = np.zeros((T, d, n)), np.zeros((T, d, n))
    last, at = h0.copy(), 0
    for s, length in enumerate(lengths):
        now = h0[s]
        for t in range(at, at + length):
            before[t] = now
            now = decay[t] * now + (dtm[t] * u[t])[:, None] * Bd[t]
            h[t] = now
        last[s] = now
        at += length
    r = (h * Cd).sum(2) + Dv * u
    y = r * m(swish(z)) if z is not None else r
    out = {"y": y, "last": last.reshape(len(lengths), d * n)}
    if dy is None:
        return out
    dy = m(dy)
    v = dy * m(swish(z)) if z is not None else dy
    g, dh0, at = np.zeros((T, d, n)), np.zeros((len(lengths), d, n)), 0
    for s, length in enumerate(lengths):
        e = np.zeros((d, n))
        for t in range(at + length - 1, at - 1, -1):
            g[t] = Cd[t] * v[t][:, None] + e
            e = decay[t] * g[t]
        dh0[s] = e
        at += length
    gah = g * decay * before
    gB = (g * Bd).sum(2)
    ddt = u * gB + (gah * m(A)).sum(2)
    ddelta = ddt * sigmoid(raw) if delta_softplus else ddt
    rows = lambda x: x.reshape(T, groups, d // groups, n).sum(2).reshape(T, groups * n)  # noqa: E731
    out.update(u=dtm * gB + Dv * v, delta=ddelta, A=(gah * dtm[:, :, None]).sum(0), B=rows(g * (dtm * u)[:, :, None]),
               C=rows(h * v[:, :, None]), D=(v * u).sum(0), delta_bias=ddelta.sum(0), h0=dh0.reshape(len(lengths), d * n))
    if z is not None:
        out["z"] = dy * r * (swish_slope(z, True) if magnitude else swish_slope(z))
    return out


def conv(x, w, bias=None, state=None, lengths=(), swish_=True, dy=None, magnitude=False):
    m = np.abs if magnitude else (lambda a: a)
    f = lambda a: None if a is None else np.asarray(a, np.float64)  # noqa: E731
    x, w, bias, state, dy = map(f, (x, w, bias, state, dy))
    (T, d), W = x.shape, w.shape[1]
    state = state.reshape(len(lengths), W - 1, d) if state is not None else np.zeros((len(lengths), W - 1, d))
    y, last, dx, dw, db, ds = np.zeros((T, d)), [], np.zeros((T, d)), np.zeros((d, W)), np.zeros(d), np.zeros(state.shape)
    at = 0
    for s, n in enumerate(lengths):
        rows = np.concatenate([state[s], x[at:at + n]])
        last.append(rows[n:])
        drows = np.zeros_like(rows)
        for t in range(n):
            p = (rows[t:t + W] * w.T).sum(0) + (bias if bias is not None else 0)
            pm = (m(rows[t:t + W]) * m(w.T)).sum(0) + (m(bias) if bias is not None else 0)
            y[at + t] = m(swish(p)) + (pm if magnitude else 0) if swish_ else pm
            if dy is None:
                continue
            g = m(dy[at + t]) * ((swish_slope(p, magnitude) + (pm if magnitude else 0)) if swish_ else 1)
            db += g
            dw += g[:, None] * m(rows[t:t + W]).T
            drows[t:t + W] += g * m(w.T)
        ds[s], dx[at:at + n] = drows[:W - 1], drows[W - 1:]
        at += n
    out = {"y": y, "last": np.stack(last).reshape(len(lengths), (W - 1) * d) if lengths else np.zeros((0, (W - 1) * d))}
    if dy is not None:
        out.update(x=dx, w=dw, bias=db, state=ds.reshape(len(lengths), (W - 1) * d))
    return out


def group_norm(x, samples, positions, groups, gamma=None, beta=None, eps=1e-5, swish_=False, dy=None):
    """Results and their magnitudes: (out, scale)."""
    f = lambda a: None if a is None else np.asarray(a, np.float64)  # noqa: E731
    x, gamma, beta, dy = map(f, (x, gamma, beta, dy))
    channels = x.shape[-1]
    shape = (samples, positions, groups, channels // groups)
    gam = (gamma if gamma is not None else np.ones(channels)).reshape(shape[2:])
    bet = (beta if beta is not None else np.zeros(channels)).reshape(shape[2:])
    v = x.reshape(shape)
    ax = (1, 3)
    mean = v.mean(ax, keepdims=True)
    var = ((v - mean) ** 2).mean(ax, keepdims=True)
    rstd = 1 / np.sqrt(var + eps)
    xhat = (v - mean) * rstd
    # What xhat's roundings are proportional to.  The mean is a sum over n values, so each of its roundings is half a step of a
    # partial sum, which sum |x| bounds: the mean is off by a multiple of mean |x|, however near to zero it is itself.
    xm = (np.abs(v) + np.abs(v).mean(ax, keepdims=True)) * rstd
    p, pm = xhat * gam + bet, xm * np.abs(gam) + np.abs(bet)
    flat = lambda a: np.broadcast_to(a, shape).reshape(x.shape)  # noqa: E731
    out = {"y": flat(swish(p) if swish_ else p), "mean": mean.reshape(samples, groups), "rstd": rstd.reshape(samples, groups)}
    scale = {"y": flat(1.1 * pm if swish_ else pm), "mean": np.abs(v).mean(ax), "rstd": (rstd * (1 + xm.max(ax, keepdims=True))).reshape(samples, groups)}
    if dy is None:
        return out, scale
    d = dy.reshape(shape)
    dv = d * swish_slope(p) if swish_ else d
    dvm = np.abs(d) * (1.1 + pm) if swish_ else np.abs(d)       # |swish''| <= 0.5, times the error of p
    dxh, dxm = dv * gam, dvm * np.abs(gam)
    out["x"] = flat(rstd * (dxh - dxh.mean(ax, keepdims=True) - xhat * (dxh * xhat).mean(ax, keepdims=True)))
    scale["x"] = flat(rstd * (dxm + dxm.mean(ax, keepdims=True) + xm * (dxm * xm).mean(ax, keepdims=True)))
    out["gamma"], scale["gamma"] = (dv * xhat).sum((0, 1)).reshape(-1), (dvm * xm).sum((0, 1)).reshape(-1)
    out["beta"], scale["beta"] = dv.sum((0, 1)).reshape(-1), dvm.sum((0, 1)).reshape(-1)
    return out, scale


def philox(n, seed, offset):
    """Words 0 .. n - 1: one at a time in Python's integers."""
    words = []
    for j in range((n + 3) // 4):
        x = [j & 0xFFFFFFFF, j >> 32, offset & 0xFFFFFFFF, offset >> 32 & 0xFFFFFFFF]
        k = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
        for _ in range(10):
            a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
            x = [(b >> 32) ^ x[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ x[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        words += x
    return np.array(words[:n], np.uint64)
