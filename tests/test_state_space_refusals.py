"""What the state space entry points refuse, before any device is looked at, and the reference that their tests compare with."""
import ctypes as C

import numpy as np
import pytest

import state_space_reference as R
from parallelreverseautodiff_b200 import _lib

P = C.c_void_p(1 << 20)        # never followed: every call here is refused
Q = C.c_void_p(1 << 21)


def _status(name, *args):
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.prad_last_error().decode()


def _scan(**over):
    s = dict(tokens=12, sequences=3, dim=8, state=4, groups=2, u=P, delta=P, A=P, B=P, C=P)
    s.update(over)
    return _lib.Scan(**s)


@pytest.mark.parametrize("over,status,text", [
    (dict(tokens=-1), _lib.ERR_SHAPE, "bad shape"),
    (dict(dim=0), _lib.ERR_SHAPE, "bad shape"),
    (dict(state=0), _lib.ERR_SHAPE, "bad shape"),
    (dict(groups=3), _lib.ERR_SHAPE, "do not divide into 3 groups"),
    (dict(state=129), _lib.ERR_UNSUPPORTED, "at most 128 states"),
    (dict(tokens=1 << 31), _lib.ERR_UNSUPPORTED, "tokens"),
    (dict(tokens=13), _lib.ERR_SHAPE, "13 tokens do not divide into 3 sequences"),
    (dict(sequences=0), _lib.ERR_SHAPE, "do not divide"),
    (dict(ld_u=7), _lib.ERR_SHAPE, "pitch"),
    (dict(ld_B=7), _lib.ERR_SHAPE, "pitch"),
    (dict(u=None), _lib.ERR_INVALID, "null pointer"),
    (dict(C=None), _lib.ERR_INVALID, "null pointer"),
    (dict(offsets=(1 << 20) + 2), _lib.ERR_INVALID, "unaligned offsets"),
])
def test_scan_refuses(over, status, text):
    s = C.byref(_scan(**over))
    for name, rest in (("prad_selective_scan_forward", (Q, 0, None, None)),
                       ("prad_selective_scan_backward", (Q, Q, 0, C.byref(_lib.ScanGradients(Q, Q, Q, Q, Q, Q))))):
        got, message = _status(name, None, 0, s, *rest)
        assert got == status and text in message, message


def test_scan_refuses_more():
    good, g = _scan(), _lib.ScanGradients(Q, Q, Q, Q, Q, Q)
    ref = C.byref(good)
    cases = [
        ("prad_selective_scan_forward", (5, ref, Q, 0, None, None), _lib.ERR_INVALID, "dtype"),
        ("prad_selective_scan_forward", (0, None, Q, 0, None, None), _lib.ERR_INVALID, "null scan"),
        ("prad_selective_scan_forward", (0, ref, None, 0, None, None), _lib.ERR_INVALID, "null pointer"),
        ("prad_selective_scan_forward", (0, ref, P, 0, None, None), _lib.ERR_INVALID, "y may not be an input"),
        ("prad_selective_scan_forward", (0, ref, Q, 7, None, None), _lib.ERR_SHAPE, "pitch"),
        ("prad_selective_scan_forward", (0, C.byref(_scan(h0=P)), Q, 0, P, None), _lib.ERR_INVALID, "h_last may not be h0"),
        ("prad_selective_scan_backward", (0, ref, None, Q, 0, C.byref(g)), _lib.ERR_INVALID, "null pointer"),
        ("prad_selective_scan_backward", (0, ref, Q, Q, 0, None), _lib.ERR_INVALID, "null gradients"),
        ("prad_selective_scan_backward", (0, C.byref(_scan(z=P)), Q, Q, 0, C.byref(_lib.ScanGradients(Q, Q, None, Q, Q, Q))),
         _lib.ERR_INVALID, "null pointer"),
        ("prad_selective_scan_backward", (0, ref, Q, Q, 0, C.byref(_lib.ScanGradients(Q, Q, Q, Q, Q, Q, None, None, Q))),
         _lib.ERR_INVALID, "dh0 without an h0"),
        ("prad_selective_scan_forward", (0, C.byref(_scan(delta=(1 << 20) + 2)), Q, 0, None, None), _lib.ERR_INVALID, "unaligned pointer"),
        ("prad_selective_scan_forward", (1, ref, C.c_void_p((1 << 21) + 4), 0, None, None), _lib.ERR_INVALID, "unaligned pointer"),
        ("prad_selective_scan_step", (0, ref, Q, 0, Q), _lib.ERR_SHAPE, "one token for each sequence"),
        ("prad_selective_scan_step", (0, C.byref(_scan(sequences=12)), Q, 0, Q), _lib.ERR_INVALID, "null pointer"),
        # a call that is right otherwise: there is no context
        ("prad_selective_scan_forward", (0, ref, Q, 0, None, None), _lib.ERR_NOT_INITIALIZED, "prad_init"),
        ("prad_selective_scan_backward", (0, ref, Q, Q, 0, C.byref(g)), _lib.ERR_NOT_INITIALIZED, "prad_init"),
    ]
    for name, args, status, text in cases:
        got, message = _status(name, None, *args)
        assert got == status and text in message, (name, message)
    n = C.c_size_t()
    assert _status("prad_selective_scan_saved_bytes", 0, ref, C.byref(n))[0] == 0 and n.value >= 8 * 4 * 4
    assert _status("prad_selective_scan_saved_bytes", 0, ref, None)[0] == _lib.ERR_INVALID
    assert _status("prad_selective_scan_saved_bytes", 0, C.byref(_lib.Scan(12, 3, 8, 4, 2)), C.byref(n))[0] == 0
    assert _status("prad_selective_scan_saved_bytes", 0, C.byref(_lib.Scan(12, 3, 8, 4, 3)), C.byref(n))[0] == _lib.ERR_SHAPE


def test_conv_refuses():
    def call(x=P, ld_x=0, w=P, bias=None, state=None, offsets=None, y=Q, ld_y=0, state_out=None, sequences=2, tokens=6, dim=5, width=4):
        return _status("prad_causal_conv_forward", None, 0, x, ld_x, w, bias, state, offsets, y, ld_y, state_out, sequences, tokens, dim,
                       width, 1)

    for over, status, text in [
        (dict(width=0), _lib.ERR_UNSUPPORTED, "widths"), (dict(width=9), _lib.ERR_UNSUPPORTED, "widths"),
        (dict(dim=0), _lib.ERR_SHAPE, "bad shape"), (dict(dim=(1 << 20) + 1), _lib.ERR_UNSUPPORTED, "channels"),
        (dict(tokens=7), _lib.ERR_SHAPE, "do not divide"), (dict(ld_x=4), _lib.ERR_SHAPE, "pitch"),
        (dict(w=None), _lib.ERR_INVALID, "null pointer"), (dict(y=P), _lib.ERR_INVALID, "y may not be x"),
        (dict(state=P, state_out=P), _lib.ERR_INVALID, "state_out may not be the state"),
        (dict(bias=C.c_void_p((1 << 20) + 1)), _lib.ERR_INVALID, "unaligned pointer"),
        (dict(), _lib.ERR_NOT_INITIALIZED, "prad_init"),
    ]:
        got, message = call(**over)
        assert got == status and text in message, (over, message)
    got, message = _status("prad_causal_conv_backward", None, 0, P, 0, P, None, None, None, Q, 0, P, 0, None, None, None, 2, 6, 5, 4, 1)
    assert got == _lib.ERR_INVALID and "dx may not be" in message
    got, message = _status("prad_causal_conv_step", None, 0, P, 0, P, None, None, Q, 0, None, 6, 5, 4, 1)
    assert got == _lib.ERR_INVALID and "null pointer" in message


def test_norm_and_dropout_refuse():
    def norm(samples=2, positions=3, channels=12, groups=4, eps=1e-5, x=P):
        return _status("prad_group_norm_forward", None, 0, x, None, None, Q, Q, Q, samples, positions, channels, groups, eps, 0)

    for over, status, text in [
        (dict(groups=5), _lib.ERR_SHAPE, "do not divide into 5 groups"), (dict(groups=0), _lib.ERR_SHAPE, "bad shape"),
        (dict(samples=-1), _lib.ERR_SHAPE, "bad shape"), (dict(eps=-1.0), _lib.ERR_INVALID, "eps"),
        (dict(eps=float("nan")), _lib.ERR_INVALID, "eps"), (dict(x=None), _lib.ERR_INVALID, "null pointer"),
        (dict(), _lib.ERR_NOT_INITIALIZED, "prad_init"),
    ]:
        got, message = norm(**over)
        assert got == status and text in message, (over, message)

    def drop(x=P, n=10, p=0.5):
        return _status("prad_dropout", None, 0, x, None, Q, n, p, 1, 2, None)

    for over, status, text in [
        (dict(p=-0.1), _lib.ERR_INVALID, "[0, 1]"), (dict(p=1.5), _lib.ERR_INVALID, "[0, 1]"), (dict(p=float("nan")), _lib.ERR_INVALID, "[0, 1]"),
        (dict(n=-1), _lib.ERR_SHAPE, "negative"), (dict(x=None), _lib.ERR_INVALID, "null pointer"),
        (dict(), _lib.ERR_NOT_INITIALIZED, "prad_init"),
    ]:
        got, message = drop(**over)
        assert got == status and text in message, (over, message)


def test_dropout_refuses_more_than_a_launch_holds():
    got, message = _status("prad_dropout", None, 0, P, None, Q, 1 << 62, 0.5, 1, 2, None)
    assert got == _lib.ERR_UNSUPPORTED and "too many" in message, message


def test_the_structs_are_the_headers():
    assert C.sizeof(_lib.Scan) == 8 + 24 + 10 * 8 + 5 * 8 and _lib.Scan.offsets.offset == 32
    assert C.sizeof(_lib.ScanGradients) == 14 * 8


# ---------------------------------------------------------------- the reference itself
def test_reference_generator_gives_the_published_vectors():
    # the known answers of the generator's authors
    assert [hex(w) for w in R.philox(4, 0, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    assert [hex(w) for w in R.philox(8, 0, 0)][:4] == [hex(w) for w in R.philox(4, 0, 0)]


def _difference(f, x, dx, h=1e-6):
    return (f(x + h * dx) - f(x - h * dx)) / (2 * h)


def test_reference_gradients_against_differences():
    """Central differences of a random functional of the outputs, one input at a time: truncation and cancellation are each
    below 1e-8 of the values here (h = 1e-6, third derivatives and values of order ten)."""
    r = np.random.default_rng(5)
    T, d, n, q, lengths = 11, 6, 3, 2, [4, 0, 6, 1]
    x = dict(u=r.standard_normal((T, d)), delta=r.standard_normal((T, d)), A=-r.uniform(0.2, 2, (d, n)), B=r.standard_normal((T, q * n)),
             C=r.standard_normal((T, q * n)), D=r.standard_normal(d), z=r.standard_normal((T, d)), delta_bias=r.standard_normal(d),
             h0=r.standard_normal((4, d * n)))
    dy = r.standard_normal((T, d))
    got = R.scan(**x, lengths=lengths, groups=q, dy=dy)
    for k in x:
        dx = r.standard_normal(x[k].shape)
        want = _difference(lambda v: (R.scan(**{**x, k: v}, lengths=lengths, groups=q)["y"] * dy).sum(), x[k], dx)
        assert abs((got[k] * dx).sum() - want) < 1e-6, k
    x = dict(x=r.standard_normal((T, d)), w=r.standard_normal((d, 3)), bias=r.standard_normal(d), state=r.standard_normal((4, 2 * d)))
    got = R.conv(**x, lengths=lengths, dy=dy)
    for k in x:
        dx = r.standard_normal(x[k].shape)
        want = _difference(lambda v: (R.conv(**{**x, k: v}, lengths=lengths)["y"] * dy).sum(), x[k], dx)
        assert abs((got[k] * dx).sum() - want) < 1e-6, k
    x = dict(x=r.standard_normal((12, 6)), gamma=r.standard_normal(6), beta=r.standard_normal(6))
    dy = r.standard_normal((12, 6))
    got = R.group_norm(**x, samples=3, positions=4, groups=2, swish_=True, dy=dy)[0]
    for k in x:
        dx = r.standard_normal(x[k].shape)
        want = _difference(lambda v: (R.group_norm(**{**x, k: v}, samples=3, positions=4, groups=2, swish_=True)[0]["y"] * dy).sum(), x[k], dx)
        assert abs((got[k] * dx).sum() - want) < 1e-6, k
