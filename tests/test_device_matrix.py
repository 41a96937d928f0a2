"""Shapes of device matrices, and what the operators that take pitches refuse before anything is launched."""
import numpy as np
import pytest

from parallelreverseautodiff_b200 import _lib
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


def _refused(e, call, status):
    e.lib.taken()
    with pytest.raises(_lib.PradError) as err:
        call()
    assert err.value.status == status and not [c for c in e.lib.taken() if not c[0].endswith("_bytes")]


T, D, N = 10, 8, 4


def _scan(e, f):
    m = lambda *s: e.empty(s, f)  # noqa: E731
    return dict(u=m(T, D), delta=m(T, D), A=m(D, N), B=m(T, N), C=m(T, N), z=m(T, D))


def _calls(e, f):
    """Calls whose result has a pitch: by name, the matrix and the pitch as their keywords."""
    m = lambda *s: e.empty(s, f)  # noqa: E731
    scan, one = _scan(e, f), m(T, D)
    saved = m(e.selective_scan_saved(T, D, N, f))
    return {
        "scan forward": lambda out, ld: e.selective_scan_forward(**scan, out=out, ld_y=ld),
        "scan step": lambda out, ld: e.selective_scan_step(**scan, h=m(T, D * N), out=out, ld_y=ld),
        "conv forward": lambda out, ld: e.causal_conv_forward(one, m(D, 4), out=out, ld_y=ld),
        "conv step": lambda out, ld: e.causal_conv_step(one, m(D, 4), m(T, 3 * D), out=out, ld_y=ld),
        "conv backward": lambda out, ld: e.causal_conv_backward(one, m(D, 4), one, out={"x": out.view((T, D))}, ld_dx=ld),
        "scan backward": lambda out, ld: e.selective_scan_backward(
            **scan, saved=saved, dy=one, out=dict(u=m(T, D), delta=out.view((T, D)), A=m(D, N), B=m(T, N), C=m(T, N), z=m(T, D)),
            gradient_pitches={"delta": ld}),
    }


@pytest.mark.parametrize("name", ["scan forward", "scan step", "conv forward", "conv step", "conv backward", "scan backward"])
def test_results_with_a_pitch_have_their_type_and_room(name):
    e = recording_engine()
    double = _calls(e, np.dtype(np.float64))[name]
    _refused(e, lambda: double(e.empty((T, 12), F), 12), _lib.ERR_INVALID)         # four bytes where eight are written
    call = _calls(e, F)[name]
    for ld in (9, 12):
        call(e.empty((T, ld), F), ld)
        call(e.empty((1, (T - 1) * ld + D), F), ld)                                # the last row needs no more than its columns
        call(e.empty((T, 2 * ld), F).view((T, ld), 5), 2 * ld)
        _refused(e, lambda: call(e.empty((1, (T - 1) * ld + D - 1), F), ld), _lib.ERR_SHAPE)
        _refused(e, lambda: call(e.empty((1, (T - 1) * ld + D + 4), F).view((1, T * D), 5), ld), _lib.ERR_SHAPE)
    call(E.DeviceMatrix(e, 1 << 30, (T, D), F, owned=False), 100)                  # memory of others: its owner knows


def test_inputs_with_a_pitch_have_room():
    e = recording_engine()
    m = lambda *s: e.empty(s, F)  # noqa: E731
    scan, saved, one, w, state = _scan(e, F), m(e.selective_scan_saved(T, D, N, F)), m(T, D), m(D, 4), m(T, 3 * D)
    for k in ("u", "delta", "z", "B", "C"):
        columns = scan[k].shape[1]
        wide = {**scan, k: m(T, 2 * columns).view((T, columns), columns)}
        for call in (lambda s, p: e.selective_scan_forward(**s, pitches=p), lambda s, p: e.selective_scan_step(**s, h=m(T, D * N), pitches=p),
                     lambda s, p: e.selective_scan_backward(**s, saved=saved, dy=one, pitches=p)):
            call(wide, {k: 2 * columns})
            _refused(e, lambda: call(wide, {k: 2 * columns + 1}), _lib.ERR_SHAPE)
            _refused(e, lambda: call(scan, {k: 2 * columns}), _lib.ERR_SHAPE)
    for call in (lambda: e.causal_conv_forward(one, w, ld_x=2 * D), lambda: e.causal_conv_step(one, w, state, ld_x=2 * D),
                 lambda: e.causal_conv_backward(one, w, one, ld_x=2 * D), lambda: e.causal_conv_backward(one, w, one, ld_dy=2 * D),
                 lambda: e.selective_scan_backward(**scan, saved=saved, dy=one, ld_dy=2 * D), lambda: e.causal_conv_forward(one, w, ld_y=2 * D),
                 lambda: e.selective_scan_backward(**scan, saved=saved, dy=one, gradient_pitches={"B": 2 * N})):
        _refused(e, call, _lib.ERR_SHAPE)
    nothing = m(0, D)
    e.causal_conv_forward(nothing, w, sequences=0, ld_x=2 * D, ld_y=2 * D)


def test_a_single_token_of_width_one_needs_no_state():
    e = recording_engine()
    x, w = e.empty((T, D), F), e.empty((D, 1), F)
    y = e.causal_conv_step(x, w, None)
    assert e.lib.taken()[-1] == ("prad_causal_conv_step", (1, E.F32, x.ptr, 0, w.ptr, None, None, y.ptr, 0, None, T, D, 1, 1))
