"""CPU: sizes and refusals of the 4-bit entry points (nothing here reaches a kernel), and the host's own
description of the formats."""
import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest

import fp4_reference as ref

INVALID, UNSUPPORTED = 1, 3


def status(call):
    import importlib
    tb = importlib.import_module("tetris_b200")
    with pytest.raises(tb.TetrisError) as e:
        call()
    return e.value.status


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("rows,cols", [(0, 1), (1, 1), (1, 32), (5, 33), (128, 64), (129, 65), (1000, 4095), (1 << 30, 1 << 20)])
def test_sizes(tb, fmt, rows, cols):
    codes, scales = tb.fp4_sizes(rows, cols, fmt)
    assert codes == rows * ref.pitch(cols)
    assert scales == -(-rows // 128) * ref.tiles(cols, fmt) * 512
    assert (codes, scales) == tb._fp4_storage(rows, cols, fmt)


def test_bad_sizes_and_formats_are_refused(tb):
    assert status(lambda: tb.fp4_sizes(1, 0, tb.FP4_MX)) == INVALID
    assert status(lambda: tb.fp4_sizes(-1, 1, tb.FP4_MX)) == INVALID
    assert status(lambda: tb.fp4_sizes(1, 1, 2)) == INVALID
    assert status(lambda: tb.fp4_sizes(1 << 31, 1, tb.FP4_MX)) == UNSUPPORTED
    assert status(lambda: tb.fp4_sizes(1, (1 << 24) + 1, tb.FP4_MX)) == UNSUPPORTED


def test_quantize_refuses_bad_arguments(tb):
    """(the addresses are never looked at: each call fails before)"""
    q = lambda **k: tb.fp4_quantize(**{**dict(input=4096, codes=4096, scales=4096, rows=4, cols=32, format=tb.FP4_NV), **k})
    assert status(lambda: q(format=7)) == INVALID
    assert status(lambda: q(format=tb.FP4_MX, exponent=1)) == INVALID
    assert status(lambda: q(exponent=101)) == INVALID
    assert status(lambda: q(exponent=-101)) == INVALID
    assert status(lambda: q(rows=-1)) == INVALID
    assert status(lambda: q(cols=0)) == INVALID
    assert status(lambda: q(ld=31)) == INVALID
    assert status(lambda: q(dtype=3)) == INVALID
    assert status(lambda: q(input=4098)) == INVALID
    assert status(lambda: q(input=4097, dtype=tb.BF16)) == INVALID
    assert status(lambda: tb.fp4_dequantize(4096, 4096, 4096, 4, 32, tb.FP4_NV, ld=8)) == INVALID
    assert status(lambda: tb.fp4_dequantize(4096, 4096, 4096, 4, 32, tb.FP4_MX, exponent=-3)) == INVALID
    tb.fp4_quantize(0, 0, 0, 0, 32, tb.FP4_MX)  # no rows: nothing to do
    tb.fp4_dequantize(0, 0, 0, 0, 32, tb.FP4_MX)


def test_filters_refuse_bad_arguments(tb):
    w = np.zeros((8, 32), np.float32)
    assert status(lambda: tb.Fp4Filter(w, 32, 8, format=5)) == INVALID
    assert status(lambda: tb.Fp4Filter(w, 32, 8, exponent=3)) == INVALID
    assert status(lambda: tb.Fp4Filter(w, 32, 8, format=tb.FP4_NV, exponent=200)) == INVALID
    assert status(lambda: tb.Fp4Filter(np.zeros((8, 32, 3, 3), np.float32), 32, 8, 3)) == UNSUPPORTED
    with pytest.raises(ValueError):
        tb.Fp4Filter(w, 32, 9)
    lib, out = tb.lib(), ctypes.c_void_p()
    assert lib.tetris_fp4_filter_create(None, 0, 32, 8, 1, 0, 0, 0, None, ctypes.byref(out)) == INVALID
    assert lib.tetris_fp4_filter_create(w.ctypes.data, 0, 0, 8, 1, 0, 0, 0, None, ctypes.byref(out)) == INVALID
    assert lib.tetris_fp4_filter_create(w.ctypes.data, 0, 32, 0, 1, 0, 0, 0, None, ctypes.byref(out)) == INVALID
    lib.tetris_fp4_filter_destroy(None)


def test_products_refuse_a_missing_filter(tb):
    lib, n = tb.lib(), ctypes.c_int64(0)
    assert lib.tetris_fp4_product(None, 4096, 4096, 1, 0, None, 4096, 0, 0, 0, None) == INVALID
    assert lib.tetris_fp4_linear(None, 4096, 0, 1, 0, 0, None, 4096, 0, 0, 0, None, 0, None) == INVALID
    assert lib.tetris_fp4_conv2d(None, 4096, 4096, 1, 1, 1, 1, 0, 0, None, 0, None, 0, None) == INVALID
    assert lib.tetris_fp4_workspace(None, 1, ctypes.byref(n)) == INVALID
    assert lib.tetris_fp4_filter_check(None) == INVALID
    assert lib.tetris_fp4_filter_info(None, None) == INVALID
    assert lib.tetris_fp4_filter_download(None, None, None) == INVALID


def test_host_tensors_are_checked_before_the_call(tb):
    """Types, strides and sizes of tensors, by the Python layer."""
    import torch
    x, buf = torch.zeros(4, 64), torch.zeros(4096, dtype=torch.uint8)
    with pytest.raises(ValueError):
        tb.fp4_quantize(x.double(), buf, buf, 4, 64, tb.FP4_MX)
    with pytest.raises(ValueError):
        tb.fp4_quantize(x.t(), buf, buf, 64, 4, tb.FP4_MX)          # columns apart
    with pytest.raises(ValueError):
        tb.fp4_quantize(x[:, ::2], buf, buf, 4, 32, tb.FP4_MX)
    with pytest.raises(ValueError):
        tb.fp4_quantize(x, buf[:127], buf, 4, 64, tb.FP4_MX)        # codes one byte short
    with pytest.raises(ValueError):
        tb.fp4_quantize(x, buf, buf[:511], 4, 64, tb.FP4_MX)        # scales one byte short
    with pytest.raises(ValueError):
        tb.fp4_quantize(x[:1].expand(4, 64), buf, buf, 4, 64, tb.FP4_MX)
    with pytest.raises(ValueError):
        tb.fp4_quantize(x, buf, buf, 5, 64, tb.FP4_MX)              # more rows than the tensor has
    with pytest.raises(ValueError):
        tb.fp4_quantize(x, buf, buf, 4, 64, tb.FP4_MX, dtype=tb.BF16)


def test_numbers_that_do_not_fit_the_calls_integers(tb):
    """A number of 33 bits would reach the library as another one, a stride of 2^32 + 1 as one that writes every pixel."""
    import types
    import torch
    wide, f = (1 << 32) + 1, types.SimpleNamespace(in_channel_=32, out_channel_=8, format_=tb.FP4_NV, handle=None, _handle=None)
    x, y, buf = torch.zeros(4, 32), torch.zeros(4, 8), torch.zeros(4096, dtype=torch.uint8)
    calls = [lambda: tb.fp4_sizes(1, wide, tb.FP4_MX),
             lambda: tb.fp4_quantize(4096, 4096, 4096, 1, wide, tb.FP4_MX),
             lambda: tb.fp4_dequantize(4096, 4096, 4096, 1, wide, tb.FP4_MX),
             lambda: tb.fp4_quantize(x, buf, buf, 4, 32, tb.FP4_NV, exponent=wide),
             lambda: tb.fp4_dequantize(buf, buf, x, 4, 32, tb.FP4_NV, exponent=-wide),
             lambda: tb.fp4_product(f, buf, buf, y, 4, exponent=wide),
             lambda: tb.fp4_linear(f, x, y, 4, exponent=wide),
             lambda: tb.fp4_conv2d(f, x, y, 1, 2, 2, wide, 0),
             lambda: tb.fp4_conv2d(f, x, y, 1, 2, 2, 1, wide - 1),
             lambda: tb.fp4_conv2d(f, 4096, 4096, wide, 2, 2, 1, 0),
             lambda: tb.fp4_conv2d(f, x, y, 1, 2, 2, 1, 0, exponent=wide),
             lambda: tb.Fp4Filter(np.zeros((8, 32), np.float32), 32, 8, format=tb.FP4_NV, exponent=wide)]
    for call in calls:
        with pytest.raises(ValueError):
            call()


def test_numbers_that_do_not_fit_64_bits(tb):
    """Rows and row distances of 65 bits would arrive as other ones, a type of 33 bits as FP32."""
    import types
    import torch
    wide, f = 1 << 64, types.SimpleNamespace(in_channel_=32, out_channel_=8, format_=tb.FP4_MX, handle=None, _handle=None)
    few, buf = torch.zeros(10), torch.zeros(4096, dtype=torch.uint8)
    calls = [lambda: tb.fp4_sizes(wide, 32, tb.FP4_MX),
             lambda: tb.fp4_workspace(f, wide + 1),
             lambda: tb.fp4_quantize(4096, 4096, 4096, wide, 32, tb.FP4_MX),
             lambda: tb.fp4_quantize(4096, 4096, 4096, 0, 32, tb.FP4_MX, ld=wide),
             lambda: tb.fp4_dequantize(4096, 4096, 4096, -wide, 32, tb.FP4_MX),
             lambda: tb.fp4_dequantize(4096, 4096, 4096, 0, 32, tb.FP4_MX, ld=-wide),
             lambda: tb.fp4_quantize(few, buf, buf, 4 - wide, 32, tb.FP4_MX),
             lambda: tb.fp4_quantize(few, buf, buf, 4, 32, tb.FP4_MX, ld=-wide),
             lambda: tb.fp4_product(f, 4096, 4096, 4096, wide),
             lambda: tb.fp4_product(f, 4096, 4096, 4096, 0, ld=wide),
             lambda: tb.fp4_linear(f, 4096, 4096, wide),
             lambda: tb.fp4_linear(f, 4096, 4096, 0, ld_input=wide),
             lambda: tb.fp4_linear(f, 4096, 4096, 0, ld_output=wide),
             lambda: tb.fp4_quantize(4096, 4096, 4096, 0, 32, tb.FP4_MX, dtype=1 << 32),
             lambda: tb.fp4_dequantize(4096, 4096, 4096, 0, 32, tb.FP4_MX, dtype=1 << 32)]
    for call in calls:
        with pytest.raises(ValueError):
            call()


def test_reference_rounds_to_even_and_saturates():
    v = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.25, -5.0] + [0] * 22])
    code, byte = ref.quantize(v, ref.MX)
    assert byte[0, 0] == 127 and list(code[0, :10]) == [0, 2, 2, 4, 4, 6, 6, 7, 0, 14]
    assert ref.E4M3[0x7E] == 448 and ref.E4M3[1] == 2.0 ** -9 and np.isnan(ref.E4M3[0x7F])


def _to_24_bits(x):
    """A Fraction rounded to 24 significant bits, ties to even."""
    if x == 0:
        return x
    e = math.frexp(float(abs(x)))[1] - 24
    unit = Fraction(2) ** e
    n = x / unit
    n = n.numerator // n.denominator + (1 if (n % 1, n.numerator // n.denominator % 2) > (Fraction(1, 2), 0) else 0)
    return n * unit


def _neighbours(x):
    """x of at most 24 bits with the numbers of 24 bits before and behind it."""
    up = Fraction(2) ** (math.frexp(float(x))[1] - 24)
    down = up / 2 if math.frexp(float(x))[0] == 0.5 else up
    return (x - down, -1), (x, 0), (x + up, 1)


@pytest.mark.parametrize("m", range(8, 16))
def test_quotient_of_two_operations_on_and_beside_the_borders(m):
    """The codes' quotient x / s as x r + x r', r' = r (1 - r s), all in 24 bits, in exact arithmetic: on a border
    between codes and one last place beside it, it lies where the real quotient does, whichever reciprocal within two
    last places r is.  It never falls where x grows (x r grows by 2^-24 |x r| a place at least, x r' and its rounding
    change by less than 2^-42 |x r|), so these values decide for all others.  Exponents only shift it."""
    s = Fraction(m, 8)
    nearest = _to_24_bits(1 / s)
    for places in range(-2, 3):
        r = nearest + places * Fraction(2) ** (math.frexp(float(nearest))[1] - 24)
        rest = _to_24_bits(_to_24_bits(1 - r * s) * r)
        for border in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
            b = Fraction(border)
            for x, side in _neighbours(b * s):
                q = _to_24_bits(x * r + _to_24_bits(x * rest))
                assert (q > b) - (q < b) == side, (m, places, border, side)


def test_sixth_of_two_operations_on_and_beside_the_borders():
    """The same for the block scale of the NV form, largest / 6 as largest * RN(1 / 6) + largest * (what that rounding
    left): on every border between E4M3 numbers and one last place beside it."""
    sixth = _to_24_bits(Fraction(1, 6))
    rest = _to_24_bits(Fraction(1, 6) - sixth)
    for lo, hi in zip(ref.E4M3[0:126], ref.E4M3[1:127]):
        b = (Fraction(lo) + Fraction(hi)) / 2
        for x, side in _neighbours(6 * b):
            q = _to_24_bits(x * sixth + _to_24_bits(x * rest))
            assert (q > b) - (q < b) == side, (lo, side)
