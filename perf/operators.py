"""Operators of a state space layer: what a program has them do, in plain torch and through the library.

  scan        the selective state space scan over packed sequences. "forward" answers a prompt (output and final state),
              "train" is forward and backward with every gradient
  conv        the short causal convolution in front of it, per channel, forward and backward
  step        one new token for each sequence of a batch: convolution and scan on the states that the last token left, the new
              states into buffers of their own
  group_norm  group norm, channels last, with the swish behind it where asked, forward and backward
  dropout     dropout by a counter-based generator with the residual added; "backward" is the gradient's way back

Tokens of all sequences are the rows of one matrix; a sequence may have no token at all. Where `own` is false, `run` computes
with elementary torch operations on the GPU.
"""
import math
import random

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f64": torch.float64}
SIZE = {"f32": 4, "f64": 8}
EPS = 1e-5


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # a few users of a small model, one new token each: the smallest call there is, launches are all of it
        {"name": "step-f32-4", "kind": "step", "dtype": "f32", "batch": 4, "dim": 256, "state": 16, "groups": 1, "width": 4},
        # a full batch of a large model, one new token each: the states are read and written once
        {"name": "step-f32-256", "kind": "step", "dtype": "f32", "batch": 256, "dim": 2048, "state": 16, "groups": 1, "width": 4},
        # one long prompt: few channels for the whole card, the token axis has to be divided
        {"name": "scan-f32-prompt", "kind": "scan", "dtype": "f32", "pass": "forward", "tokens": 16384, "sequences": 1, "dim": 1024,
         "state": 16, "groups": 1},
        # a training batch of packed texts of different lengths
        {"name": "scan-f32-train", "kind": "scan", "dtype": "f32", "pass": "train", "tokens": 16384, "sequences": 24, "dim": 1024,
         "state": 16, "groups": 1},
        # the double library, odd sizes, several groups of shared input and output rows
        {"name": "scan-f64-train", "kind": "scan", "dtype": "f64", "pass": "train", "tokens": 1501, "sequences": 7, "dim": 201,
         "state": 10, "groups": 3},
        # the convolution of a training batch
        {"name": "conv-f32-train", "kind": "conv", "dtype": "f32", "tokens": 16384, "sequences": 24, "dim": 2048, "width": 4},
        # the same in double with odd sizes and a narrow window
        {"name": "conv-f64-train", "kind": "conv", "dtype": "f64", "tokens": 2047, "sequences": 9, "dim": 333, "width": 3},
        # tokens of a windowed attention network: 64 images of 3136 tokens with 96 channels
        {"name": "norm-f32-images", "kind": "group_norm", "dtype": "f32", "samples": 64, "positions": 3136, "channels": 96,
         "groups": 8, "swish": True},
        # one norm per token, as behind the scan of a training batch
        {"name": "norm-f32-tokens", "kind": "group_norm", "dtype": "f32", "samples": 16384, "positions": 1, "channels": 2048,
         "groups": 16, "swish": False},
        # double, odd sizes
        {"name": "norm-f64-odd", "kind": "group_norm", "dtype": "f64", "samples": 5, "positions": 441, "channels": 60, "groups": 12,
         "swish": True},
        # a wide layer's activations: 65536 rows of 4096
        {"name": "drop-f32-65536", "kind": "dropout", "dtype": "f32", "rows": 65536, "cols": 4096, "pass": "forward", "p": 0.1},
        # the way back of an odd small matrix in double
        {"name": "drop-f64-small", "kind": "dropout", "dtype": "f64", "rows": 301, "cols": 77, "pass": "backward", "p": 0.5},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("step", "scan", "scan", "conv", "group_norm", "dropout"))
    dtype = rng.choice(("f32", "f32", "f64"))
    if kind == "step":
        groups = rng.choice((1, 1, 2, 4))
        return {"kind": kind, "dtype": dtype, "batch": _spread(rng, 1, 256), "dim": groups * _spread(rng, 8, 2048 // groups // 2),
                "state": rng.choice((8, 16, 16, rng.randint(1, 32))), "groups": groups, "width": rng.randint(2, 4)}
    if kind == "scan":
        groups = rng.choice((1, 1, 2, 3))
        state = rng.choice((8, 16, 16, rng.randint(1, 64)))
        dim = groups * _spread(rng, 4, 2048 // groups)
        most = (1 << 26) // (dim * state)
        tokens = _spread(rng, 1, max(1, min(16384, most)))
        return {"kind": kind, "dtype": dtype, "pass": rng.choice(("forward", "train")), "tokens": tokens,
                "sequences": _spread(rng, 1, 64), "dim": dim, "state": state, "groups": groups}
    if kind == "conv":
        return {"kind": kind, "dtype": dtype, "tokens": _spread(rng, 1, 16384), "sequences": _spread(rng, 1, 64),
                "dim": _spread(rng, 8, 2048), "width": rng.randint(2, 4)}
    if kind == "group_norm":
        groups = rng.choice((1, 4, 8, 16, 32))
        channels = groups * _spread(rng, 1, 2048 // groups)
        positions = rng.choice((1, _spread(rng, 2, 4096)))
        samples = _spread(rng, 1, max(1, min(16384, (1 << 25) // (channels * positions))))
        return {"kind": kind, "dtype": dtype, "samples": samples, "positions": positions, "channels": channels, "groups": groups,
                "swish": rng.choice((True, False))}
    return {"kind": kind, "dtype": dtype, "rows": _spread(rng, 1, 32768), "cols": _spread(rng, 1, 4096),
            "pass": rng.choice(("forward", "backward")), "p": rng.choice((0.05, 0.1, 0.25, 0.5))}


def work(case):
    s, kind = SIZE[case["dtype"]], case["kind"]
    if kind == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": (3 if case["pass"] == "forward" else 2) * n * s, "flops": 2 * n}
    if kind == "group_norm":
        n = case["samples"] * case["positions"] * case["channels"]
        return {"bytes": 4 * n * s + 4 * case["channels"] * s, "flops": 24 * n}
    if kind == "conv":
        n, w = case["tokens"] * case["dim"], case["width"]
        return {"bytes": 4 * n * s + (2 * w + 2 + 3 * (w - 1) * case["sequences"]) * case["dim"] * s, "flops": 6 * w * n}
    if kind == "step":
        n, st, w = case["batch"] * case["dim"], case["state"], case["width"]
        return {"bytes": s * (n * (2 * st + 2 * (w - 1) + 5) + 2 * case["batch"] * case["groups"] * st + case["dim"] * (st + w + 3)),
                "flops": n * (8 * st + 2 * w)}
    n, st = case["tokens"] * case["dim"], case["state"]
    rows, states = case["tokens"] * case["groups"] * st, case["dim"] * st
    if case["pass"] == "forward":
        return {"bytes": s * (4 * n + 2 * rows + states * (1 + 2 * case["sequences"])), "flops": n * (7 * st + 8)}
    return {"bytes": s * (8 * n + 4 * rows + states * (2 + 3 * case["sequences"])), "flops": n * (25 * st + 30)}


# ---------------------------------------------------------------- inputs
def _lengths(tokens, sequences, seed):
    """Lengths of packed sequences: they differ by up to a factor of about ten, and one in twelve has no token."""
    r = random.Random(seed)
    shares = [0.0 if sequences > 2 and r.random() < 1 / 12 else math.exp(r.uniform(0.0, 2.3)) for _ in range(sequences)]
    if not any(shares):
        shares[0] = 1.0
    total, at, marks = sum(shares), 0.0, [0]
    for share in shares:
        at += share
        marks.append(int(round(tokens * at / total)))
    marks[-1] = tokens
    return [b - a for a, b in zip(marks, marks[1:])]


class _Inputs:
    """Random tensors on the GPU from one seed."""

    def __init__(self, case, seed):
        self.dtype = TORCH[case["dtype"]]
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, scale=1.0):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=self.dtype) * scale

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.rand(shape, generator=self.g, device="cuda", dtype=self.dtype) * (hi - lo) + lo


def _scan_weights(r, dim, state):
    """Decay rates near -1 .. -state, and a bias whose softplus is a time step of 0.001 to 0.1, as such layers are set up."""
    A = -torch.arange(1, state + 1, device="cuda", dtype=r.dtype) * r.uniform(dim, state, lo=0.8, hi=1.2)
    step = torch.exp(r.uniform(dim, lo=math.log(1e-3), hi=math.log(1e-1)))
    return {"A": A, "D": r.normal(dim, scale=0.2) + 1.0, "bias": step + torch.log(-torch.expm1(-step))}


def prepare(case, seed):
    r, kind = _Inputs(case, seed), case["kind"]
    s = {"case": case}
    if kind in ("scan", "conv"):
        lengths = _lengths(case["tokens"], case["sequences"], seed)
        s["lengths"] = lengths
        s["offsets"] = torch.tensor([0] + list(np.cumsum(lengths)), device="cuda", dtype=torch.int32)
    if kind == "scan":
        T, d, n, q, S = case["tokens"], case["dim"], case["state"], case["groups"], case["sequences"]
        s.update(_scan_weights(r, d, n))
        s.update(u=r.normal(T, d), delta=r.normal(T, d, scale=0.5), z=r.normal(T, d), B=r.normal(T, q * n), C=r.normal(T, q * n),
                 h0=r.normal(S, d * n, scale=0.1), dy=r.normal(T, d))
    elif kind == "conv":
        T, d, w, S = case["tokens"], case["dim"], case["width"], case["sequences"]
        s.update(x=r.normal(T, d), w=r.normal(d, w, scale=w ** -0.5), bias=r.normal(d, scale=0.1),
                 state=r.normal(S, (w - 1) * d), dy=r.normal(T, d))
    elif kind == "step":
        b, d, n, q, w = case["batch"], case["dim"], case["state"], case["groups"], case["width"]
        s.update(_scan_weights(r, d, n))
        s.update(x=r.normal(b, d), w=r.normal(d, w, scale=w ** -0.5), conv_bias=r.normal(d, scale=0.1), delta=r.normal(b, d, scale=0.5),
                 z=r.normal(b, d), B=r.normal(b, q * n), C=r.normal(b, q * n), conv_state=r.normal(b, (w - 1) * d),
                 h=r.normal(b, d * n, scale=0.1))
    elif kind == "group_norm":
        shape = (case["samples"] * case["positions"], case["channels"])
        s.update(x=r.normal(*shape) + 0.5, gamma=r.normal(case["channels"], scale=0.1) + 1.0, beta=r.normal(case["channels"], scale=0.1),
                 dy=r.normal(*shape))
    else:
        s.update(x=r.normal(case["rows"], case["cols"]), residual=r.normal(case["rows"], case["cols"]), seed=(seed * 2654435761 + 17) % (1 << 64),
                 offset=seed + (1 << 33))
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ---------------------------------------------------------------- plain forms
def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x)))


def _where_rows(lengths):
    """Of each token: its sequence and its place in it."""
    n = torch.tensor(lengths, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), n)
    return seq, torch.arange(sum(lengths), device="cuda") - (torch.cumsum(n, 0) - n)[seq]


def _scan_rows(a, b, longest):
    """h_t = a_t h_(t-1) + b_t over dimension 0, in log2 steps: the step doubles the rows that each row has taken in."""
    k = 1
    while k < longest:
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _plain_scan(s):
    c = s["case"]
    T, d, n, q, lengths = c["tokens"], c["dim"], c["state"], c["groups"], s["lengths"]
    seq, place = _where_rows(lengths)
    first = (place == 0).view(T, 1, 1)
    A, u, h0 = s["A"], s["u"], s["h0"].view(-1, d, n)
    raw = s["delta"] + s["bias"]
    dt = _softplus(raw)
    a = torch.exp(dt[:, :, None] * A)
    Bd = s["B"].view(T, q, n).repeat_interleave(d // q, 1)
    Cd = s["C"].view(T, q, n).repeat_interleave(d // q, 1)
    kept = torch.where(first, 0.0, a)
    h = _scan_rows(kept, (dt * u)[:, :, None] * Bd + torch.where(first, a * h0[seq], 0.0), max(lengths))
    r = (h * Cd).sum(2) + s["D"] * u
    sz = _sigmoid(s["z"])
    y = r * (s["z"] * sz)
    ends = torch.cumsum(torch.tensor(lengths, device="cuda"), 0) - 1
    none = torch.tensor([m == 0 for m in lengths], device="cuda").view(-1, 1, 1)
    last = torch.where(none, h0, h[torch.clamp(ends, min=0)])
    out = {"y": y, "last": last.reshape(-1, d * n)}
    if c["pass"] == "forward":
        return out
    v = s["dy"] * (s["z"] * sz)
    after = torch.cat([kept[1:], torch.zeros_like(kept[:1])])       # the decay by which a token's state reaches the next token
    g = _scan_rows(after.flip(0), (v[:, :, None] * Cd).flip(0), max(lengths)).flip(0)
    del after, kept
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before = torch.where(first, h0[seq], before)
    gah = g * a * before
    gB = (g * Bd).sum(2)
    ddt = u * gB + (gah * A).sum(2)
    ddelta = ddt * _sigmoid(raw)
    dh0 = torch.zeros_like(h0)
    heads = torch.nonzero(place == 0).view(-1)
    dh0[seq[heads]] = (g * a)[heads]
    out.update(du=dt * gB + s["D"] * v, ddelta=ddelta, dz=s["dy"] * r * (sz * (1 + s["z"] * (1 - sz))),
               dA=(gah * dt[:, :, None]).sum(0), dB=(g * (dt * u)[:, :, None]).view(T, q, d // q, n).sum(2).view(T, q * n),
               dC=(h * v[:, :, None]).view(T, q, d // q, n).sum(2).view(T, q * n), dD=(v * u).sum(0), dbias=ddelta.sum(0),
               dh0=dh0.view(-1, d * n))
    return out


def _plain_conv(s):
    c = s["case"]
    T, d, w, S, lengths = c["tokens"], c["dim"], c["width"], c["sequences"], s["lengths"]
    seq, place = _where_rows(lengths)
    n = torch.tensor(lengths, device="cuda")
    start = torch.cumsum(n, 0) - n
    lag = torch.arange(w - 1, -1, -1, device="cuda")                # of column k of w
    rows = torch.cat([s["x"], s["state"].view(S * (w - 1), d)])

    def at(sequence, p):                                            # the row of place p of a sequence (before it: its state)
        return torch.where(p >= 0, start[sequence] + p, T + sequence * (w - 1) + p + w - 1)

    taken = at(seq[:, None], place[:, None] - lag)
    wt = s["w"].t()
    p = (rows[taken] * wt).sum(1) + s["bias"]
    sp = _sigmoid(p)
    ids = torch.arange(S, device="cuda")[:, None]
    last = rows[at(ids, n[:, None] - (w - 1) + torch.arange(w - 1, device="cuda"))].reshape(S, (w - 1) * d)
    g = s["dy"] * (sp * (1 + p * (1 - sp)))
    g0 = torch.cat([g, torch.zeros_like(g[:1])])                    # row T: no token

    def seen(sequence, p):                                          # the token at place p, T where there is none
        return torch.where((p >= 0) & (p < n[sequence]), start[sequence] + p, T)

    dx = (g0[seen(seq[:, None], place[:, None] + lag)] * wt).sum(1)
    past = torch.arange(-(w - 1), 0, device="cuda")
    dstate = (g0[seen(ids[:, :, None], past[None, :, None] + lag)] * wt).sum(2).reshape(S, (w - 1) * d)
    return {"y": p * sp, "last": last, "dx": dx, "dw": (g[:, None, :] * rows[taken]).sum(0).t().contiguous(), "dbias": g.sum(0),
            "dstate": dstate}


def _plain_step(s):
    c = s["case"]
    b, d, n, q, w = c["batch"], c["dim"], c["state"], c["groups"], c["width"]
    rows = torch.cat([s["conv_state"].view(b, w - 1, d), s["x"].view(b, 1, d)], 1)
    p = (rows * s["w"].t()).sum(1) + s["conv_bias"]
    u = p * _sigmoid(p)
    dt = _softplus(s["delta"] + s["bias"])
    Bd = s["B"].view(b, q, 1, n).expand(b, q, d // q, n).reshape(b, d, n)
    Cd = s["C"].view(b, q, 1, n).expand(b, q, d // q, n).reshape(b, d, n)
    h = torch.exp(dt[:, :, None] * s["A"]) * s["h"].view(b, d, n) + (dt * u)[:, :, None] * Bd
    r = (h * Cd).sum(2) + s["D"] * u
    return {"u": u, "y": r * (s["z"] * _sigmoid(s["z"])), "conv_state": rows[:, 1:].reshape(b, (w - 1) * d), "h": h.view(b, d * n)}


def _plain_group_norm(s):
    c = s["case"]
    S, P, G, C = c["samples"], c["positions"], c["groups"], c["channels"]
    x = s["x"].view(S, P, G, C // G)
    gamma, beta = s["gamma"].view(G, C // G), s["beta"].view(G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean((1, 3), keepdim=True) + EPS)
    xhat = (x - mean) * rstd
    v = xhat * gamma + beta
    dy = s["dy"].view(S, P, G, C // G)
    if c["swish"]:
        sv = _sigmoid(v)
        y, dv = v * sv, dy * (sv * (1 + v * (1 - sv)))
    else:
        y, dv = v, dy
    dxhat = dv * gamma
    dx = rstd * (dxhat - dxhat.mean((1, 3), keepdim=True) - xhat * (dxhat * xhat).mean((1, 3), keepdim=True))
    return {"y": y.reshape(S * P, C), "mean": mean.reshape(S, G), "rstd": rstd.reshape(S, G), "dx": dx.reshape(S * P, C),
            "dgamma": (dv * xhat).sum((0, 1)).reshape(C), "dbeta": dv.sum((0, 1)).reshape(C)}


_M32 = 0xFFFFFFFF


def _philox(n, seed, offset):
    """Words 0 .. n - 1 of Philox4x32-10 (Salmon and others, "Parallel random numbers: as easy as 1, 2, 3", 2011) with the key
    `seed`: block j has the counter (j, offset), each of 64 bits. In 64-bit integers, whose products wrap around."""
    j = torch.arange((n + 3) // 4, device="cuda")
    x = [j & _M32, j >> 32, torch.full_like(j, offset & _M32), torch.full_like(j, offset >> 32 & _M32)]
    key = [seed & _M32, seed >> 32 & _M32]
    for _ in range(10):
        a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [(b >> 32 & _M32) ^ x[1] ^ key[0], b & _M32, (a >> 32 & _M32) ^ x[3] ^ key[1], a & _M32]
        key = [key[0] + 0x9E3779B9 & _M32, key[1] + 0xBB67AE85 & _M32]
    return torch.stack(x, 1).view(-1)[:n]


def _plain_dropout(s):
    c, x = s["case"], s["x"]
    keep = _philox(x.numel(), s["seed"], s["offset"]).view_as(x) < int(round((1 - c["p"]) * 2 ** 32))
    y = torch.where(keep, x * (1 / (1 - c["p"])), 0.0)
    return y + s["residual"] if c["pass"] == "forward" else y


_PLAIN = {"scan": _plain_scan, "conv": _plain_conv, "step": _plain_step, "group_norm": _plain_group_norm, "dropout": _plain_dropout}


# ---------------------------------------------------------------- the library's calls
_eng = None
_NP = {torch.float32: np.dtype(np.float32), torch.float64: np.dtype(np.float64), torch.int32: np.dtype(np.int32)}
_LEGACY_STREAM = 1       # CUDA's handle of the stream that torch works on by default


def _engine():
    global _eng
    if _eng is None:
        from parallelreverseautodiff_b200 import engine as E

        _eng = E.Engine(0)
        _eng.use_stream(_LEGACY_STREAM)
    return _eng


def _m(t):
    from parallelreverseautodiff_b200.engine import DeviceMatrix

    return DeviceMatrix(_engine(), t.data_ptr(), t.shape, _NP[t.dtype], owned=False)


def _own_scan(s):
    e, c = _engine(), s["case"]
    new = torch.empty_like
    of = {k: _m(s[k]) for k in ("u", "delta", "A", "B", "C", "D", "z", "h0", "offsets")}
    of.update(delta_bias=_m(s["bias"]), groups=c["groups"], sequences=c["sequences"], delta_softplus=True)
    out = {"y": new(s["u"]), "last": new(s["h0"])}
    if c["pass"] == "forward":
        e.selective_scan_forward(**of, out=_m(out["y"]), h_last=_m(out["last"]))
        return out
    _, _, saved = e.selective_scan_forward(**of, out=_m(out["y"]), h_last=_m(out["last"]), save=True)
    out.update(du=new(s["u"]), ddelta=new(s["u"]), dz=new(s["u"]), dA=new(s["A"]), dB=new(s["B"]), dC=new(s["C"]), dD=new(s["D"]),
               dbias=new(s["bias"]), dh0=new(s["h0"]))
    e.selective_scan_backward(**of, saved=saved, dy=_m(s["dy"]), out={k: _m(out[v]) for k, v in (
        ("u", "du"), ("delta", "ddelta"), ("z", "dz"), ("A", "dA"), ("B", "dB"), ("C", "dC"), ("D", "dD"), ("delta_bias", "dbias"),
        ("h0", "dh0"))})
    return out


def _own_conv(s):
    e, c = _engine(), s["case"]
    new = torch.empty_like
    of = {k: _m(s[k]) for k in ("x", "w", "bias", "state", "offsets")}
    of.update(sequences=c["sequences"], swish=True)
    out = {"y": new(s["x"]), "last": new(s["state"]), "dx": new(s["x"]), "dw": new(s["w"]), "dbias": new(s["bias"]),
           "dstate": new(s["state"])}
    e.causal_conv_forward(**of, out=_m(out["y"]), state_out=_m(out["last"]))
    e.causal_conv_backward(**of, dy=_m(s["dy"]), out={k: _m(out["d" + k]) for k in ("x", "w", "bias", "state")})
    return out


def _own_step(s):
    e, c = _engine(), s["case"]
    new = torch.empty_like
    out = {"u": new(s["x"]), "y": new(s["x"]), "conv_state": new(s["conv_state"]), "h": new(s["h"])}
    u = _m(out["u"])
    e.causal_conv_step(_m(s["x"]), _m(s["w"]), _m(s["conv_state"]), bias=_m(s["conv_bias"]), swish=True, out=u,
                       state_out=_m(out["conv_state"]))
    e.selective_scan_step(u, _m(s["delta"]), _m(s["A"]), _m(s["B"]), _m(s["C"]), _m(s["h"]), D=_m(s["D"]), z=_m(s["z"]),
                          delta_bias=_m(s["bias"]), delta_softplus=True, groups=c["groups"], out=_m(out["y"]), h_out=_m(out["h"]))
    return out


def _own_group_norm(s):
    e, c = _engine(), s["case"]
    new = torch.empty_like
    stats = torch.empty((2, c["samples"], c["groups"]), device="cuda", dtype=s["x"].dtype)
    out = {"y": new(s["x"]), "mean": stats[0], "rstd": stats[1], "dx": new(s["x"]), "dgamma": new(s["gamma"]), "dbeta": new(s["beta"])}
    x, gamma, beta, mean, rstd = _m(s["x"]), _m(s["gamma"]), _m(s["beta"]), _m(stats[0]), _m(stats[1])
    e.group_norm_forward(x, c["groups"], gamma, beta, positions=c["positions"], eps=EPS, swish=c["swish"],
                         out=(_m(out["y"]), mean, rstd))
    e.group_norm_backward(x, mean, rstd, _m(s["dy"]), c["groups"], gamma, beta, positions=c["positions"], swish=c["swish"],
                          out=(_m(out["dx"]), _m(out["dgamma"]), _m(out["dbeta"])))
    return out


def _own_dropout(s):
    e, c = _engine(), s["case"]
    y = torch.empty_like(s["x"])
    e.dropout(_m(s["x"]), c["p"], s["seed"], s["offset"], residual=_m(s["residual"]) if c["pass"] == "forward" else None, out=_m(y))
    return y


_OWN = {"scan": _own_scan, "conv": _own_conv, "step": _own_step, "group_norm": _own_group_norm, "dropout": _own_dropout}


# ---------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    """Sequence by sequence and token by token in 64 bits; gradients by differentiating those steps."""
    kind = case["kind"]
    if kind == "dropout" and case["rows"] * case["cols"] > 1 << 23:
        return None
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in prepare(case, seed).items()}
    with torch.enable_grad():
        return {"scan": _exact_scan, "conv": _exact_conv, "step": _exact_step, "group_norm": _exact_group_norm,
                "dropout": _exact_dropout}[kind](s)


def _leaves(s, names):
    return [s[k].detach().clone().requires_grad_(True) for k in names]


def _gradients(y, dy, names, leaves):
    got = torch.autograd.grad(y, leaves, dy, allow_unused=True)
    return {"d" + k: torch.zeros_like(x) if g is None else g for k, x, g in zip(names, leaves, got)}


def _exact_scan(s):
    c, lengths = s["case"], s["lengths"]
    d, n, q, train = c["dim"], c["state"], c["groups"], c["pass"] == "train"
    names = ("u", "delta", "z", "A", "B", "C", "D", "bias", "h0")
    leaves = _leaves(s, names)
    with torch.set_grad_enabled(train):
        u, delta, z, A, B, C, D, bias, h0 = leaves
        dt = torch.nn.functional.softplus(delta + bias, threshold=700.0)
        order = sorted(range(len(lengths)), key=lambda i: -lengths[i])      # the longest first: the active ones stay in front
        starts = [sum(lengths[:i]) for i in order]
        sizes = [lengths[i] for i in order]
        h = h0.view(-1, d, n)[order]
        first = torch.tensor(starts, device="cuda")
        rows, parts, ended = [], [], []
        active = len(order)
        for t in range(max(lengths)):
            while sizes[active - 1] <= t:
                active -= 1
            if active < h.shape[0]:
                ended.append(h[active:])
                h = h[:active]
            at = first[:active] + t
            m = dt[at].unsqueeze(2)
            wide = lambda x: x[at].view(active, q, 1, n).expand(active, q, d // q, n).reshape(active, d, n)  # noqa: E731
            h = torch.exp(m * A) * h + m * u[at].unsqueeze(2) * wide(B)
            parts.append((h * wide(C)).sum(2))
            rows.append(at)
        back = torch.argsort(torch.cat(rows))
        r = torch.cat(parts)[back] + D * u
        y = r * torch.nn.functional.silu(z)
        final = torch.cat([h] + ended[::-1])[torch.argsort(torch.tensor(order, device="cuda"))]
    out = {"y": y.detach(), "last": final.detach().reshape(-1, d * n)}
    if train:
        out.update(_gradients(y, s["dy"], names, leaves))
    return out


def _exact_conv(s):
    c, lengths = s["case"], s["lengths"]
    d, w = c["dim"], c["width"]
    names = ("x", "w", "bias", "state")
    leaves = _leaves(s, names)
    x, wt, bias, state = leaves
    at, ys, lasts = 0, [], []
    for i, m in enumerate(lengths):
        whole = torch.cat([state[i].view(w - 1, d), x[at:at + m]])
        if m:
            ys.append(torch.nn.functional.conv1d(whole.t().unsqueeze(0), wt.unsqueeze(1), bias, groups=d)[0].t())
        lasts.append(whole[m:].reshape(-1))
        at += m
    y = torch.nn.functional.silu(torch.cat(ys))
    return {"y": y.detach(), "last": torch.stack(lasts).detach(), **_gradients(y, s["dy"], names, leaves)}


def _exact_step(s):
    c = s["case"]
    b, d, n, q, w = c["batch"], c["dim"], c["state"], c["groups"], c["width"]
    whole = torch.cat([s["conv_state"].view(b, w - 1, d), s["x"].unsqueeze(1)], 1)
    u = torch.nn.functional.silu(torch.einsum("bkd,dk->bd", whole, s["w"]) + s["conv_bias"])
    dt = torch.nn.functional.softplus(s["delta"] + s["bias"], threshold=700.0)
    decay = torch.exp(torch.einsum("bd,dn->bdn", dt, s["A"])).view(b, q, d // q, n)
    B, C = s["B"].view(b, q, n), s["C"].view(b, q, n)
    h = decay * s["h"].view(b, q, d // q, n) + torch.einsum("bqe,bqn->bqen", (dt * u).view(b, q, d // q), B)
    y = (torch.einsum("bqen,bqn->bqe", h, C).reshape(b, d) + s["D"] * u) * torch.nn.functional.silu(s["z"])
    return {"u": u, "y": y, "conv_state": whole[:, 1:].reshape(b, -1), "h": h.reshape(b, d * n)}


def _exact_group_norm(s):
    c = s["case"]
    S, P, G, C = c["samples"], c["positions"], c["groups"], c["channels"]
    names = ("x", "gamma", "beta")
    leaves = _leaves(s, names)
    x, gamma, beta = leaves
    rows = x.view(S, P, G, C // G).transpose(1, 2).reshape(S * G, P * (C // G))
    mean = rows.mean(1)
    rstd = (rows.var(1, unbiased=False) + EPS).rsqrt()
    xhat = ((rows - mean[:, None]) * rstd[:, None]).view(S, G, P, C // G).transpose(1, 2).reshape(S * P, C)
    y = xhat * gamma + beta
    if c["swish"]:
        y = torch.nn.functional.silu(y)
    return {"y": y.detach(), "mean": mean.detach().view(S, G), "rstd": rstd.detach().view(S, G), **_gradients(y, s["dy"], names, leaves)}


def _exact_dropout(s):
    """The generator in numpy's unsigned integers."""
    c, n = s["case"], s["case"]["rows"] * s["case"]["cols"]
    u32, u64, low = np.uint32, np.uint64, np.uint64(0xFFFFFFFF)
    j = np.arange((n + 3) // 4, dtype=u64)
    ctr = np.stack([j & low, j >> u64(32), np.full_like(j, s["offset"] & 0xFFFFFFFF), np.full_like(j, s["offset"] >> 32)]).astype(u32)
    k0, k1 = s["seed"] & 0xFFFFFFFF, s["seed"] >> 32 & 0xFFFFFFFF
    for _ in range(10):
        p0, p1 = ctr[0].astype(u64) * u64(0xD2511F53), ctr[2].astype(u64) * u64(0xCD9E8D57)
        ctr = np.stack([(p1 >> u64(32)).astype(u32) ^ ctr[1] ^ u32(k0), (p1 & low).astype(u32),
                        (p0 >> u64(32)).astype(u32) ^ ctr[3] ^ u32(k1), (p0 & low).astype(u32)])
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    keep = torch.from_numpy((ctr.T.reshape(-1)[:n].astype(np.float64) < round((1 - c["p"]) * 2 ** 32))).to(s["x"].device)
    y = s["x"] * keep.view_as(s["x"]) / (1 - c["p"])
    return y + s["residual"] if c["pass"] == "forward" else y
