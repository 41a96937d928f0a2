"""Shapes of device matrices, and what the operators that take pitches refuse before anything is launched."""
import numpy as np
import pytest

from parallelreverseautodiff_b200 import engine as E
from recording_library import recording_engine

F = np.dtype(np.float32)


@pytest.mark.parametrize("kind", [np.int32, np.int64, np.uint16, int])
def test_sizes_of_numpy_integers(kind):
    """65000 x 65000 values are more than 32 bits count."""
    e = recording_engine()
    n = kind(65000)
    for m in (E.DeviceMatrix(e, 0, (n, n), F, owned=False), E.DeviceMatrix(e, 0, [n, n], F, owned=False),
              E.DeviceMatrix(e, 0, (1,), F, owned=False).view((n, n)), e.empty((n, n), F), e.zeros((n, n), F)):
        assert m.size == 65000 ** 2 and m.nbytes == 4 * 65000 ** 2 and all(type(s) is int for s in m.shape)
    assert e.lib.live == {p: 4 * 65000 ** 2 for p in e.lib.live}
    assert e.lib.taken()[-1] == ("prad_zero", (1, m.ptr, 4 * 65000 ** 2))
