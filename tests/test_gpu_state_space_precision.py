"""Scans over long sequences and many channels against 64 bits, to bounds that follow every rounding."""
import numpy as np
import pytest

import state_space_cases as S
from test_gpu_state_space import F, STEP
from util import HEADROOM

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("case", S.CASES, ids=lambda c: f"{c['d']}-{c['n']}")
def test_scan_to_its_roundings(engine, dtype, case):
    """One by one and as a whole (S.WHOLE half steps), packed and, where they are equal, by their number."""
    e, f, step = engine, F[dtype], STEP[dtype]
    x, dy, want, bound = S.expected(case, f, step)
    lengths = case["lengths"]
    for packed in (True, False) if len(set(lengths)) == 1 else (True,):
        of = dict({k: e.upload(v) for k, v in x.items()}, sequences=len(lengths), groups=case["groups"])
        if packed:
            of["offsets"] = e.sequence_offsets(lengths)
        y, last, saved = e.selective_scan_forward(**of, h_last=True, save=True)
        grads = e.selective_scan_backward(**of, saved=saved, dy=e.upload(dy))
        got = {"y": y.numpy(), "last": last.numpy(), **{k: m.numpy() for k, m in grads.items()}}
        shares = S.worst(got, want, bound, step)
        for k, (single, whole) in shares.items():
            for name, share in ((f"scan {k} {dtype}, each", single), (f"scan {k} {dtype}, whole", whole)):
                HEADROOM[name] = max(HEADROOM.get(name, 0.0), share)
        assert set(shares) == {"y", "last", *x}
        assert all(max(s) <= 1 for s in shares.values()), shares
