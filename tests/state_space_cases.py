"""Scans whose results are compared with bounds that follow every rounding."""
import numpy as np

import state_space_bounds as bounds
import state_space_reference as R

# a result as a whole is off by no more than this many half steps of itself: each of its terms has fewer than 64 roundings along the
# longest way, as signs come; twice that for states, whose errors are those of as many tokens as they remember
WHOLE = 128
CASES = [dict(lengths=[700], d=20, n=8, groups=2), dict(lengths=[3, 700, 45, 0, 301], d=150, n=16, groups=1),
         dict(lengths=[129] * 5, d=33, n=5, groups=1), dict(lengths=[64, 0, 1, 200], d=66, n=32, groups=2),
         dict(lengths=[300, 90], d=20, n=128, groups=1), dict(lengths=[31, 2, 260], d=40, n=64, groups=1)]


def inputs(case, f):
    """Decays from slow to fast, as layers of this kind are set up: |A| of 1 to n, time steps about 0.001 to 0.2."""
    lengths, d, n, q = (case[k] for k in ("lengths", "d", "n", "groups"))
    T, r = sum(lengths), np.random.default_rng(sum(lengths) + d + n)
    x = dict(u=r.standard_normal((T, d)), delta=r.standard_normal((T, d)) * 0.5, A=-np.arange(1, n + 1) * r.uniform(0.8, 1.2, (d, n)),
             B=r.standard_normal((T, q * n)), C=r.standard_normal((T, q * n)), D=r.standard_normal(d), z=r.standard_normal((T, d)),
             delta_bias=np.log(np.expm1(np.exp(r.uniform(np.log(1e-3), np.log(1e-1), d)))), h0=r.standard_normal((len(lengths), d * n)))
    return {k: v.astype(f) for k, v in x.items()}, r.standard_normal((T, d)).astype(f)


def expected(case, f, e):
    x, dy = inputs(case, f)
    of = dict(x, lengths=case["lengths"], groups=case["groups"], dy=dy)
    return x, dy, R.scan(**of), bounds.scan_bounds(e, **of)


def worst(got, want, bound, e):
    """By result: the largest share of its bound, and the share of the bound of the whole."""
    shares = {}
    for k in want:
        g = np.asarray(got[k], np.float64).reshape(want[k].shape)
        off = np.abs(g - want[k])
        shares[k] = (float((off / np.maximum(bound[k].reshape(off.shape), 1e-300)).max()),
                     float(np.sqrt((off ** 2).sum()) / (WHOLE * e * np.sqrt((want[k] ** 2).sum()))))
    return shares
