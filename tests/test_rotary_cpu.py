"""Tables of rotary angles against the formulas in high precision, and what the rotary store refuses; no GPU needed."""
import ctypes as C
from fractions import Fraction

import numpy as np
import pytest

from miinfer_b200._lib import Rotary, RotaryScaling, lib
from test_paged_cpu import DEVICE, INVALID, OK, RANGE, UNSUPPORTED, batch_of, no_gpu, view_of

PLAIN, LINEAR, BASE, BANDS, RAMP = range(5)


def turns(dims, theta, kind=None, factor=4.0, original=4096.0, low=1.0, high=32.0):
    out, magnitude = (C.c_uint64 * (dims // 2))(), C.c_float(-1)
    how = None if kind is None else C.byref(RotaryScaling(kind, factor, original, low, high))
    assert lib.b200kv_rotary_turns(dims, theta, how, out, C.byref(magnitude)) == OK
    return list(out), magnitude.value


def frequencies(dims, theta, kind, factor, original, low, high):
    """In 80 bits, from the definitions."""
    f = np.longdouble
    i = np.arange(dims // 2).astype(f)
    base = f(theta) * (f(factor) ** (f(dims) / f(dims - 2)) if kind == BASE else 1)
    x = base ** (-2 * i / dims)
    if kind == LINEAR:
        return x / factor
    if kind == BANDS:
        kept = np.clip((original * x / (2 * f(np.pi)) - low) / (f(high) - f(low)), 0, 1)
        return kept * x + (1 - kept) * x / factor
    if kind == RAMP:
        pair = lambda times: dims * np.log(original / (times * 2 * np.pi)) / (2 * np.log(theta))
        a, b = max(np.floor(pair(high)), 0), min(np.ceil(pair(low)), dims - 1)
        part = np.clip((i - a) / (b - a if b > a else 0.001), 0, 1)
        return part * x / factor + (1 - part) * x
    return x


@pytest.mark.parametrize("dims,theta", [(16, 10000.0), (64, 1e6), (96, 5e5), (128, 1e4), (256, 1e7)])
@pytest.mark.parametrize("kind,factor,original,low,high", [(PLAIN, 1, 0, 1, 2), (LINEAR, 4, 0, 1, 2), (BASE, 8, 0, 1, 2), (BANDS, 8, 8192, 1, 4), (RAMP, 4, 32768, 1, 32),
                                                           (RAMP, 2.5, 300, 0.5, 3), (RAMP, 0.5, 4096, 1, 32), (BANDS, 1, 64, 2, 2.5)])
def test_tables_are_the_frequencies_fractions_of_a_turn(dims, theta, kind, factor, original, low, high):
    got, magnitude = turns(dims, theta, kind, factor, float(original), low, high)
    want = frequencies(dims, theta, kind, factor, float(original), low, high)
    for t, f in zip(got, want):
        # numpy's pi has 53 bits: 2^-53 of a frequency; what is left of both sides is of 64 bits, of which the powers lose a few
        assert abs(t / 2.0 ** 64 - float(f / (2 * np.longdouble(np.pi))) % 1.0) <= 2.0 ** -51 * float(f) + 2.0 ** -58
    expected = 0.1 * np.log(factor) + 1 if kind == RAMP and factor > 1 else 1.0
    assert abs(magnitude - expected) <= 2.0 ** -23


def test_angles_of_far_positions():
    """pos * turns modulo 2^64 against rational arithmetic: the first pair turns by one radian a position."""
    (first, *_), _ = turns(128, 1e6)
    two_pi = Fraction(62831853071795864769252867665590057683943, 10 ** 40)
    for p in (1, 1000, 1 << 20, 2_000_000_011):
        exact = (Fraction(p) / two_pi) % 1
        got = Fraction(first * p % 2 ** 64, 2 ** 64)
        assert abs(got - exact) <= Fraction(p, 2 ** 63)


def test_frequencies_of_the_caller():
    f = np.array([0.0, 1.0, 2 * np.pi, -0.25, 100.0])
    out = (C.c_uint64 * 5)()
    assert lib.b200kv_rotary_turns_of(f.ctypes.data_as(C.POINTER(C.c_double)), 5, out) == OK
    assert out[0] == 0 and abs(out[1] / 2.0 ** 64 - 1 / (2 * np.pi)) < 2.0 ** -52
    assert min(out[2], 2 ** 64 - out[2]) < 2 ** 12                       # a double's two pi is a turn but for its rounding
    assert abs(out[3] / 2.0 ** 64 - (1 - 0.25 / (2 * np.pi))) < 2.0 ** -52 and abs(out[4] / 2.0 ** 64 - (100 / (2 * np.pi)) % 1) < 2.0 ** -48
    bad = np.array([1.0, np.nan])
    assert lib.b200kv_rotary_turns_of(bad.ctypes.data_as(C.POINTER(C.c_double)), 2, out) == INVALID
    assert lib.b200kv_rotary_turns_of(None, 2, out) == INVALID


@pytest.mark.parametrize("dims,theta,how", [(0, 1e4, None), (24, 1e4, None), (272, 1e4, None), (64, 1.0, None), (64, float("nan"), None), (64, float("inf"), None),
                                            (64, 1e4, RotaryScaling(5, 2, 0, 1, 2)), (64, 1e4, RotaryScaling(-1, 2, 0, 1, 2)), (64, 1e4, RotaryScaling(LINEAR, 0, 0, 1, 2)),
                                            (64, 1e4, RotaryScaling(BASE, float("nan"), 0, 1, 2)), (64, 1e4, RotaryScaling(BANDS, 2, 0, 1, 2)),
                                            (64, 1e4, RotaryScaling(BANDS, 2, 64, 2, 2)), (64, 1e4, RotaryScaling(RAMP, 2, 64, 0, 2)), (64, 1e4, RotaryScaling(RAMP, 2, float("inf"), 1, 2))])
def test_tables_that_are_refused(dims, theta, how):
    out = (C.c_uint64 * 256)()
    assert lib.b200kv_rotary_turns(dims, theta, None if how is None else C.byref(how), out, None) == INVALID
    assert lib.b200kv_rotary_turns(64, 1e4, None, None, None) == INVALID


def rotate(v, b, r=None, q=1 << 20, q_stride=8 * 128, key=1 << 21, key_stride=256, value=1 << 22, value_stride=256, dtype=0, q_norm=None, k_norm=None, epsilon=1e-6, positions=None,
           query_heads=8, q_out=1 << 23, out_dtype=0, gate=None, **rotary):
    r = Rotary(**{**dict(turns=4096, dims=128, layout=0, magnitude=1.0), **rotary})
    return lib.b200kv_paged_rotary(C.byref(v), C.byref(b), C.byref(r), q, q_stride, key, key_stride, value, value_stride, dtype, q_norm, k_norm, epsilon, positions, query_heads, q_out,
                                   out_dtype, gate, None)


@no_gpu
@pytest.mark.parametrize("change", [{}, dict(key=None, value=None), dict(q=None, q_out=None, query_heads=0), dict(dims=0, turns=None), dict(dims=16, layout=1), dict(q_stride=1600, key_stride=1600, value_stride=1600),
                                    dict(gate=1 << 24, q_stride=2048), dict(q_out=1 << 20), dict(q_out=(1 << 20) + 9 * 2048), dict(dtype=1, out_dtype=1)])
def test_calls_that_are_right_end_at_the_missing_device(change):
    assert rotate(view_of(), batch_of(), **change) == DEVICE


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(q=None)), (INVALID, dict(q_out=None)), (INVALID, dict(key=None)), (INVALID, dict(value=None)), (INVALID, dict(q=None, q_out=None, key=None, value=None)),
    (INVALID, dict(dtype=2)), (INVALID, dict(dtype=-1)), (INVALID, dict(out_dtype=3)), (INVALID, dict(epsilon=float("nan"))), (INVALID, dict(epsilon=-1e-6)),
    (UNSUPPORTED, dict(dims=144)), (UNSUPPORTED, dict(dims=24)), (INVALID, dict(layout=2)), (INVALID, dict(turns=None)), (INVALID, dict(turns=4100)), (INVALID, dict(magnitude=float("inf"))),
    (INVALID, dict(q=(1 << 20) + 8)), (INVALID, dict(key=(1 << 21) + 2)), (INVALID, dict(value=(1 << 22) + 4)), (INVALID, dict(q_out=(1 << 23) + 8)), (INVALID, dict(gate=(1 << 24) + 4, q_stride=2048)),
    (INVALID, dict(q_stride=1016)), (INVALID, dict(q_stride=1028)), (INVALID, dict(key_stride=248)), (INVALID, dict(value_stride=260)), (INVALID, dict(gate=1 << 24)),
    (INVALID, dict(query_heads=0)), (INVALID, dict(q_stride=1 << 32)), (INVALID, dict(gate=1 << 24, q=None, q_out=None)), (INVALID, dict(q_norm=2)), (INVALID, dict(positions=1)),
    (INVALID, dict(q_out=(1 << 20) + 2048)), (INVALID, dict(q_out=1 << 20, out_dtype=1)), (INVALID, dict(q_out=1 << 20, q_stride=1032)), (INVALID, dict(q_out=1 << 20, gate=1 << 24, q_stride=2048)),
    (INVALID, dict(gate=1 << 20, q_stride=2048)), (INVALID, dict(gate=(1 << 23) + 16, q_stride=2048)), (INVALID, dict(q_out=1 << 21)), (INVALID, dict(q_out=(1 << 22) - 16)),
])
def test_arguments_that_are_refused(status, change):
    assert rotate(view_of(), batch_of(), **change) == status


@pytest.mark.parametrize("status,view,batch", [(UNSUPPORTED, dict(head_dim=96), {}), (INVALID, dict(key_q8=None), {}), (RANGE, {}, dict(max_length=161)), (INVALID, {}, dict(lengths=None)),
                                               (OK, {}, dict(total_tokens=0, max_tokens=0)), (OK, {}, dict(sequences=0))])
def test_views_and_batches(status, view, batch):
    assert rotate(view_of(**view), batch_of(**batch)) == status
    assert lib.b200kv_paged_rotary(C.byref(view_of()), C.byref(batch_of()), None, 16, 1024, 16, 256, 16, 256, 0, None, None, 1e-6, None, 8, 16, 0, None, None) == INVALID
