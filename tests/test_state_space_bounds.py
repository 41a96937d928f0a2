"""The bounds that the scan kernels are held to reject what is a little wrong (mistakes planted in the reference)."""
import numpy as np
import pytest

import state_space_cases as S
import state_space_reference as R

E32 = 2.0 ** -24


@pytest.mark.parametrize("case", S.CASES, ids=lambda c: f"{c['d']}-{c['n']}")
def test_bounds_reject_what_is_wrong(case):
    x, dy, want, bound = S.expected(case, np.float32, E32)
    of = dict(lengths=case["lengths"], groups=case["groups"], dy=dy)

    def rejected(got, but=()):
        for k, (single, whole) in S.worst(got, want, bound, E32).items():
            assert k in but or max(single, whole) > 1.2, (k, single, whole)

    rejected({k: 0 * v for k, v in want.items()})
    rejected({k: v * (1 + 2e-5) for k, v in want.items()})
    rejected(R.scan(**{**x, "A": x["A"].astype(np.float64) * (1 + 1e-4)}, **of), but="D")
    rejected(R.scan(**{**x, "delta_bias": x["delta_bias"].astype(np.float64) - 1e-4}, **of), but="D")
    # and take what is right up to the last roundings
    rounded = {k: v.astype(np.float32) for k, v in want.items()}
    assert all(max(s) < 1 for s in S.worst(rounded, want, bound, E32).values())
