"""GPU: 4-bit quantisation and products against the formats' definition in 64 bits.

Tolerances.  Codes and scale bytes: equal.  Dequantised values: FP32 and BF16 hold them exactly inside their
range, FP16 rounds by at most eps / 2.  A product's sum of K terms is formed in steps of at least 16 terms;
every step may truncate, at most one last place (2^-23 of what the sum of the absolute terms can reach)
when the terms are aligned and one when they are added: |error| <= (K / 16 + 4) 2^-22 sum |a w|.  The result's
type adds half a step, eps / 2 relative.
"""
import numpy as np
import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu
FORMATS = [ref.MX, ref.NV]


def dtypes(torch):
    return {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def activations(torch, rows, cols, seed, spread=3.0, dtype="fp32"):
    """Rows of different magnitude, a fifth of the values zero."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp2(spread * torch.randn(rows, 1, device="cuda", generator=g))
    x *= torch.rand(rows, cols, device="cuda", generator=g) >= 0.2
    return x.to(dtypes(torch)[dtype])


def f64(t):
    return t.double().cpu().numpy()


def buffers(tb, torch, rows, cols, fmt, fill=0xAB, extra=64):
    """(codes, scales) with `extra` bytes behind each, all of them `fill`."""
    return [torch.full((n + extra,), fill, dtype=torch.uint8, device="cuda") for n in tb.fp4_sizes(rows, cols, fmt)]


def quantized(tb, torch, x, fmt, exponent=0):
    rows, cols = x.shape
    codes, scales = buffers(tb, torch, rows, cols, fmt)
    tb.fp4_quantize(x, codes, scales, rows, cols, fmt, exponent)
    return codes, scales


def stored(tb, codes, scales, rows, cols, fmt):
    """(codes [rows, cols] with +0 for a zero, scale bytes [rows, blocks]) out of the buffers."""
    n = tb.fp4_sizes(rows, cols, fmt)
    c = ref.unpack_codes(codes.cpu().numpy()[:n[0]].reshape(rows, -1), cols)
    b = scales.cpu().numpy()[ref.scale_offsets(rows, cols, fmt)]
    return np.where(c == 8, 0, c), b


def check_quantized(tb, torch, x, fmt, exponent=0):
    rows, cols = x.shape
    codes, scales = quantized(tb, torch, x, fmt, exponent)
    want_c, want_b = ref.quantize(f64(x), fmt, exponent)
    got_c, got_b = stored(tb, codes, scales, rows, cols, fmt)
    assert np.array_equal(got_b[:, :want_b.shape[1]], want_b)
    assert np.array_equal(got_c, want_c)
    # zeros behind the last column and block; rows past the last one and what lies behind: as they were
    n = tb.fp4_sizes(rows, cols, fmt)
    packed = codes.cpu().numpy()
    assert not ref.unpack_codes(packed[:n[0]].reshape(rows, -1), 2 * ref.pitch(cols))[:, cols:].any()
    assert not got_b[:, want_b.shape[1]:].any()
    assert (packed[n[0]:] == 0xAB).all()
    s = scales.cpu().numpy()
    touched = np.zeros(s.size, bool)
    touched[ref.scale_offsets(rows, cols, fmt)] = True
    assert (s[~touched] == 0xAB).all()


SHAPES = [(1, 1), (1, 16), (3, 17), (5, 31), (7, 33), (2, 63), (33, 64), (129, 65), (130, 100), (33, 255), (2, 4095), (64, 128), (257, 200),
          (3, 129), (1000, 72)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_is_bit_exact(tb, torch_cuda, fmt, dtype, rows, cols):
    x = activations(torch_cuda, rows, cols, rows * 1000 + cols, dtype=dtype, spread=1.0 if dtype == "fp16" else 3.0)
    check_quantized(tb, torch_cuda, x, fmt, -3 if fmt == ref.NV else 0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_on_and_beside_every_border(tb, torch_cuda, fmt):
    """Values on the borders between codes and between scales, and one last place beside them."""
    torch = torch_cuda
    block = ref.BLOCK[fmt]
    rows = []
    scales = ref.E4M3[1:127] if fmt == ref.NV else 2.0 ** np.arange(-20.0, 20.0)
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    for s in scales:
        for step in (-1, 0, 1):
            v = (borders * s).astype(np.float32)
            v = (v.view(np.int32) + step).view(np.float32)
            row = np.zeros(block, np.float32)
            row[0] = 6 * s  # the block's scale is s
            row[1:8], row[8:15] = v, -v
            rows.append(row)
    if fmt == ref.NV:  # largest values on the borders between scales
        for lo, hi in zip(ref.E4M3[0:126], ref.E4M3[1:127]):
            for step in (-1, 0, 1):
                row = np.zeros(block, np.float32)
                row[3] = (np.float32(3 * (lo + hi)).view(np.int32) + step).view(np.float32)
                row[5] = row[3] / 7
                rows.append(row)
    x = torch.from_numpy(np.stack(rows)).cuda()
    check_quantized(tb, torch, x, fmt)
    if fmt == ref.NV:
        for exponent in (-90, -7, 5, 90):
            check_quantized(tb, torch, (x.double() * 2.0 ** exponent).float(), fmt, exponent)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_over_the_whole_range_of_fp32(tb, torch_cuda, fmt):
    """Random bit patterns (no infinities or NaN): values at both ends of FP32, denormals."""
    torch = torch_cuda
    rng = np.random.default_rng(5)
    bits = rng.integers(0, 0x7F800000, (300, 96), dtype=np.uint32)
    lead = rng.integers(0, 255, (300, 3), dtype=np.uint32).repeat(32, 1)  # blocks whose values are of one magnitude
    bits[:150] = (bits[:150] & 0x7FFFFF) | (np.maximum(lead[:150].astype(np.int64) - rng.integers(0, 4, (150, 96)), 0).astype(np.uint32) << 23)
    x = bits.view(np.float32) * np.where(rng.random(bits.shape) < 0.5, -1, 1).astype(np.float32)
    for exponent in ([0] if fmt == ref.MX else [0, -100, 100, -30, 64]):
        check_quantized(tb, torch, torch.from_numpy(x).cuda(), fmt, exponent)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_blocks_with_infinities_and_nan(tb, torch_cuda, fmt, bad, dtype):
    torch = torch_cuda
    x = activations(torch, 5, 100, 3, dtype=dtype, spread=1.0)
    x[1, 40] = bad
    x[3, 99] = bad
    check_quantized(tb, torch, x, fmt)
    codes, scales = quantized(tb, torch, x, fmt)
    y = torch.empty(5, 100, device="cuda")
    tb.fp4_dequantize(codes, scales, y, 5, 100, fmt)
    block = ref.BLOCK[fmt]
    want = torch.zeros(5, 100, dtype=torch.bool)
    want[1, 40 // block * block:(40 // block + 1) * block] = True
    want[3, 99 // block * block:] = True
    assert torch.equal(y.isnan().cpu(), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_quantize_rows_apart_and_off_the_vector_path(tb, torch_cuda, fmt, dtype):
    torch = torch_cuda
    base = activations(torch, 20, 300, 9, dtype=dtype, spread=1.0)
    for view in (base[:, :200], base[:, 1:201], base[::2, 3:64], base[5:6, 7:8]):
        check_quantized(tb, torch, view, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_dequantize_every_code_under_every_scale(tb, torch_cuda, fmt, dtype):
    torch = torch_cuda
    block = ref.BLOCK[fmt]
    code = np.tile(np.arange(16, dtype=np.uint8), (256, block // 16))[:, :block]
    byte = np.arange(256, dtype=np.uint8)[:, None]
    if fmt == ref.NV:
        byte = byte & 0x7F  # scales carry no sign
    codes = torch.from_numpy(ref.pack_codes(code)).cuda()
    scales = torch.from_numpy(ref.pack_scales(byte, block, fmt)).cuda()
    for exponent in ([0] if fmt == ref.MX else [0, -20, 13]):
        y = torch.empty(256, block, dtype=dtypes(torch)[dtype], device="cuda")
        tb.fp4_dequantize(codes, scales, y, 256, block, fmt, exponent)
        want = torch.from_numpy(ref.values(code, byte, fmt, exponent)).to(dtypes(torch)[dtype]).double().numpy()
        assert np.array_equal(f64(y), want, equal_nan=True)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_dequantize_shapes_rows_apart(tb, torch_cuda, fmt, rows, cols):
    torch = torch_cuda
    x = activations(torch, rows, cols, 77, spread=1.0)
    codes, scales = quantized(tb, torch, x, fmt, -4 if fmt == ref.NV else 0)
    want = ref.values(*ref.quantize(f64(x), fmt, -4 if fmt == ref.NV else 0), fmt, -4 if fmt == ref.NV else 0)
    for off in (0, 1):
        out = torch.full((rows, cols + 7), -7.0, device="cuda")
        tb.fp4_dequantize(codes, scales, out[:, off:off + cols], rows, cols, fmt, -4 if fmt == ref.NV else 0)
        assert np.array_equal(f64(out[:, off:off + cols]), want)
        out[:, off:off + cols] = -7.0
        assert bool((out == -7.0).all())


# ---- products -----------------------------------------------------------------------------------
def reference_product(x, w, fmt, ex, ew):
    """(a w^T, sum |a w|) in 64 bits from the quantised values of x and w."""
    a = ref.values(*ref.quantize(f64(x), fmt, ex), fmt, ex)
    b = ref.values(*ref.quantize(f64(w), fmt, ew), fmt, ew)
    return a @ b.T, np.abs(a) @ np.abs(b).T


def check_product(got, want, terms, k, torch):
    eps = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}[got.dtype]
    d = np.abs(f64(got) - want)
    allowed = (k / 16 + 4) * 2.0 ** -22 * terms + eps / 2 * np.abs(want) + 2.0 ** -25
    assert np.isfinite(f64(got)).all()
    assert (d <= allowed).all(), "%d of %d outside, worst %g times what is allowed" % ((d > allowed).sum(), d.size, (d / allowed).max())


def filter_and_weights(tb, torch, n, k, fmt, seed, exponent=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(n, k, device="cuda", generator=g) * 0.05
    w *= torch.rand(n, k, device="cuda", generator=g) >= 0.5
    f = tb.Fp4Filter(w, k, n, format=fmt) if exponent is None else tb.Fp4Filter(w, k, n, format=fmt, exponent=exponent)
    return f, w


PRODUCTS = [  # rows, K, N
    (1, 1, 1), (1, 64, 128), (1, 4096, 300), (2, 31, 3), (3, 100, 129), (5, 15, 130), (8, 256, 128), (9, 257, 64), (15, 33, 31), (16, 512, 256), (17, 128, 96),
    (31, 63, 127), (32, 1024, 255), (33, 255, 1), (48, 2048, 200), (63, 65, 128), (64, 640, 384), (65, 129, 130), (100, 333, 77), (127, 191, 256), (128, 256, 128),
    (129, 511, 129), (160, 96, 640), (192, 1000, 100), (255, 320, 60), (256, 768, 512), (257, 64, 257), (300, 1537, 300), (511, 48, 1000), (640, 16, 16), (1000, 2048, 1000),
    (2049, 128, 130), (5000, 64, 256), (333, 8192, 260),
    (1100, 4096, 2000), (2400, 700, 2300), (4000, 2048, 700)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,k,n", PRODUCTS)
def test_product(tb, torch_cuda, fmt, rows, k, n):
    torch = torch_cuda
    ex = -2 if fmt == ref.NV else 0
    x = activations(torch, rows, k, rows + k + n, spread=1.0)
    f, w = filter_and_weights(tb, torch, n, k, fmt, rows + 7 * k)
    want, terms = reference_product(x, w, fmt, ex, f.exponent_)
    codes, scales = quantized(tb, torch, x, fmt, ex)
    y = torch.full((rows + 1, n), float("nan"), device="cuda")
    tb.fp4_product(f, codes, scales, y[:rows], rows, ex)
    f.check()
    check_product(y[:rows], want, terms, k, torch)
    assert bool(y[rows].isnan().all())  # rows behind the last one stay as they were
    for dtype in (torch.bfloat16, torch.float16):
        z = torch.empty(rows, n, dtype=dtype, device="cuda")
        tb.fp4_product(f, codes, scales, z, rows, ex)
        assert torch.equal(z, y[:rows].to(dtype))  # the same sums, rounded once
    bias = torch.randn(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    z = torch.empty(rows, n, device="cuda")
    tb.fp4_product(f, codes, scales, z, rows, ex, bias=bias, relu=True)
    assert torch.equal(z, torch.relu(y[:rows] + bias))
    again = torch.empty(rows, n, device="cuda")
    for _ in range(3):
        tb.fp4_product(f, codes, scales, again, rows, ex)
        assert torch.equal(again, y[:rows])
    # the same from floating point in one call
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    for dtype in ("fp32", "bf16", "fp16"):
        xt = x.to(dtypes(torch)[dtype])
        codes, scales = quantized(tb, torch, xt, fmt, ex)
        tb.fp4_product(f, codes, scales, again, rows, ex)
        z = torch.full((rows + 1, n), float("nan"), device="cuda")
        tb.fp4_linear(f, xt, z, rows, work, ex)
        assert torch.equal(z[:rows], again) and bool(z[rows].isnan().all())
    f.check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [1, 20, 150, 700])
def test_rows_apart_in_and_out(tb, torch_cuda, fmt, rows):
    torch = torch_cuda
    k, n = 200, 150
    f, w = filter_and_weights(tb, torch, n, k, fmt, 5)
    base = activations(torch, rows, k + 9, 6, spread=1.0)
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    for off in (0, 1, 4):
        x = base[:, off:off + k]
        want = torch.empty(rows, n, device="cuda")
        tb.fp4_linear(f, x.contiguous(), want, rows, work)
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            out = torch.full((rows, n + 5), -3.0, dtype=dtype, device="cuda")
            tb.fp4_linear(f, x, out[:, off:off + n], rows, work)
            assert torch.equal(out[:, off:off + n], want.to(dtype))
            out[:, off:off + n] = -3.0
            assert bool((out == -3.0).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,k,n,ld", [(19, 1, 2, 8), (5, 64, 7, 16), (300, 64, 30, 40), (300, 64, 27, 32), (700, 300, 130, 136), (2000, 512, 250, 264),
                                         (2000, 512, 255, 256), (3000, 256, 513, 520)])
def test_aligned_rows_apart_whose_ends_are_not(tb, torch_cuda, fmt, dtype, rows, k, n, ld):
    """Rows of an output that begin on 16 bytes and end inside of them: what lies between the rows, and behind the last
    one of a buffer that ends with it, stays as it was."""
    torch = torch_cuda
    f, w = filter_and_weights(tb, torch, n, k, fmt, 51)
    x = activations(torch, rows, k, 52, spread=1.0)
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    want = torch.empty(rows, n, device="cuda")
    tb.fp4_linear(f, x, want, rows, work)
    check_product(want, *reference_product(x, w, fmt, 0, f.exponent_), k, torch)
    need = (rows - 1) * ld + n
    whole = torch.full((need + 64,), -3.0, dtype=dtypes(torch)[dtype], device="cuda")
    tb.fp4_linear(f, x, whole[:need], rows, work, ld_output=ld)
    f.check()
    assert bool((whole[need:] == -3.0).all())
    out = torch.cat([whole[:need], whole[need:need + ld - n]]).view(rows, ld)
    assert torch.equal(out[:, :n], want.to(out.dtype))
    assert bool((out[:, n:] == -3.0).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [3, 40, 300])
def test_nan_stays_in_its_row_and_channel(tb, torch_cuda, fmt, rows):
    torch = torch_cuda
    k, n = 300, 140
    x = activations(torch, rows, k, 8, spread=1.0)
    g = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randn(n, k, device="cuda", generator=g)
    x[1, 37] = float("nan")
    w[130, 299] = float("inf")
    w[7] = 0
    f = tb.Fp4Filter(w, k, n, format=fmt)
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    for relu in (False, True):
        y = torch.empty(rows, n, device="cuda")
        tb.fp4_linear(f, x, y, rows, work, relu=relu)
        want = torch.zeros(rows, n, dtype=torch.bool)
        want[1], want[:, 130] = True, True
        assert torch.equal(y.isnan().cpu(), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows", [1, 20, 129, 300])
def test_scales_of_rows_that_are_not_there_do_not_matter(tb, torch_cuda, fmt, rows):
    torch = torch_cuda
    k, n = 320, 128
    f, _ = filter_and_weights(tb, torch, n, k, fmt, 3)
    x = activations(torch, rows, k, 4, spread=1.0)
    got = []
    for fill in (0x00, 0xFF, 0x7F):
        codes, scales = buffers(tb, torch, rows, k, fmt, fill=fill)
        tb.fp4_quantize(x, codes, scales, rows, k, fmt)
        y = torch.empty(rows, n, device="cuda")
        tb.fp4_product(f, codes, scales, y, rows)
        got.append(y)
    assert bool(got[0].isfinite().all()) and torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("fmt", FORMATS)
def test_many_rows_equal_their_slices(tb, torch_cuda, fmt):
    """Rows in one call and in several: every variant that a number of rows selects gives the same sums up to
    their order."""
    torch = torch_cuda
    rows, k, n = 700, 1100, 260
    f, w = filter_and_weights(tb, torch, n, k, fmt, 11)
    x = activations(torch, rows, k, 12, spread=1.0)
    want, terms = reference_product(x, w, fmt, 0, f.exponent_)
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    at = 0
    for count in (1, 2, 7, 16, 17, 32, 33, 64, 100, 128, 129, 171):
        y = torch.empty(count, n, device="cuda")
        tb.fp4_linear(f, x[at:at + count], y, count, work)
        check_product(y, want[at:at + count], terms[at:at + count], k, torch)
        at += count
    assert at == rows


@pytest.mark.parametrize("rows,k,n", [(3, 100, 70), (2, 2000, 40), (40, 2048, 200), (300, 200, 150), (2000, 64, 96)])
@pytest.mark.parametrize("ex,ew", [(100, 35), (30, 100), (-60, -70), (100, -100), (-100, 100)])
def test_exponents_whose_sum_leaves_fp32(tb, torch_cuda, rows, k, n, ex, ew):
    """2^(ex + ew) need not be an FP32 number: the results are those at exponents 0, shifted.  Beyond FP32's largest
    number (sums of 2000 terms of 1e-4 have a deviation of 0.0045, times 2^135 2e38 of 3.4e38) they are infinite, below
    its smallest normal one (all of (-60, -70)) they may be zero."""
    torch = torch_cuda
    x = activations(torch, rows, k, 91, spread=0.0) * 0.01
    w = torch.randn(n, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(92)) * 0.01
    shift = lambda t, e: (t.double() * 2.0 ** e).float()
    f0 = tb.Fp4Filter(w, k, n, format=ref.NV, exponent=0)
    f = tb.Fp4Filter(shift(w, ew), k, n, format=ref.NV, exponent=ew)
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    want, y = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, device="cuda")
    tb.fp4_linear(f0, x, want, rows, work)
    tb.fp4_linear(f, shift(x, ex), y, rows, work, ex)
    want = (want.double() * 2.0 ** (ex + ew)).float()
    assert bool(((y == want) | ((want.abs() < 2.0 ** -126) & (y == 0))).all())


@pytest.mark.parametrize("rows,k,n", [(1, 2048, 1000), (3, 300, 140), (40, 2048, 200), (300, 512, 255), (2000, 64, 256)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_bias_and_relu_are_rounded_once(tb, torch_cuda, rows, k, n, dtype):
    torch = torch_cuda
    f, _ = filter_and_weights(tb, torch, n, k, ref.MX, 61)
    x = activations(torch, rows, k, 62, spread=1.0)
    bias = torch.randn(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(63))
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    plain, y = torch.empty(rows, n, device="cuda"), torch.empty(rows, n, dtype=dtypes(torch)[dtype], device="cuda")
    tb.fp4_linear(f, x, plain, rows, work)
    tb.fp4_linear(f, x, y, rows, work, bias=bias)
    assert torch.equal(y, (plain + bias).to(y.dtype))
    tb.fp4_linear(f, x, y, rows, work, bias=bias, relu=True)
    assert torch.equal(y, torch.relu(plain + bias).to(y.dtype))
    tb.fp4_linear(f, x, y, rows, work, relu=True)
    assert torch.equal(y, torch.relu(plain).to(y.dtype))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,k,n", [(1, (1 << 20) + 33, 40), (5, (1 << 20) - 1, 130), (300, 300001, 40), (2, 1 << 24, 9), (200, 1 << 18, 3000)])
def test_long_sums_of_whole_numbers_are_exact(tb, torch_cuda, fmt, rows, k, n):
    """Values 0, 1 and -1: every partial sum is a whole number below 2^24, whatever the order.  The NV form holds 1 as
    6 E4M3(1 / 6) = 33/32: there a sum is 33^2 / 2^10 times a whole number, which stays below 2^24 / 33^2 = 15406 (sums
    of 2^24 terms have a deviation of 2730)."""
    torch = torch_cuda
    g = torch.Generator(device="cuda").manual_seed(k)
    signs = lambda r: torch.randint(-1, 2, (r, k), device="cuda", generator=g, dtype=torch.int8).to(torch.bfloat16)
    x, w = signs(rows), signs(n)
    f = tb.Fp4Filter(w, k, n, format=fmt, exponent=0)
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    y = torch.empty(rows, n, device="cuda")
    tb.fp4_linear(f, x, y, rows, work)
    f.check()
    want = torch.zeros(rows, n, dtype=torch.float64, device="cuda")
    for c in range(0, k, 1 << 18):
        want += x[:, c:c + (1 << 18)].double() @ w[:, c:c + (1 << 18)].double().t()
    assert torch.equal(y.double(), want * (1 if fmt == ref.MX else (33 / 32) ** 2))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k,n", [(100, 2048), (128, 512), (64, 16), (300, 300), (2048, 1000)])
def test_a_workspace_for_some_rows_is_enough_for_fewer(tb, torch_cuda, fmt, k, n):
    """A program that serves changing numbers of rows takes one workspace, for the most."""
    torch = torch_cuda
    f, w = filter_and_weights(tb, torch, n, k, fmt, 41)
    most = 2500
    sizes = [tb.fp4_workspace(f, r) for r in range(1, most + 1)]
    assert sizes == sorted(sizes)
    x = activations(torch, most, k, 42, spread=1.0)
    want, terms = reference_product(x, w, fmt, 0, f.exponent_)
    for rows in (513, 1793, 2305, 2500):
        work = torch.empty(sizes[rows - 1], dtype=torch.uint8, device="cuda")
        for fewer in (1, 17, 509, 1789, 2301):
            if fewer <= rows:
                y = torch.empty(fewer, n, device="cuda")
                tb.fp4_linear(f, x[:fewer], y, fewer, work)
                check_product(y, want[:fewer], terms[:fewer], k, torch)
    f.check()


# ---- layers -------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n,h,w,ic,oc,stride", [(1, 1, 1, 8, 8, 1), (2, 7, 5, 64, 40, 1), (3, 9, 8, 33, 130, 2), (1, 14, 14, 256, 128, 2),
                                                (2, 13, 11, 20, 255, 3), (4, 28, 28, 128, 64, 1), (1, 5, 5, 16, 16, 9)])
def test_layer(tb, torch_cuda, fmt, n, h, w, ic, oc, stride):
    torch = torch_cuda
    ex = -5 if fmt == ref.NV else 0
    g = torch.Generator(device="cuda").manual_seed(h * ic)
    x = torch.rand(n, h, w, ic, device="cuda", generator=g)
    x *= torch.rand(x.shape, device="cuda", generator=g) >= 0.5
    f, wt = filter_and_weights(tb, torch, oc, ic, fmt, oc)
    picked = x[:, ::stride, ::stride].reshape(-1, ic)
    rows = picked.shape[0]
    want, terms = reference_product(picked, wt, fmt, ex, f.exponent_)
    bias = torch.randn(oc, device="cuda", generator=g)
    y = torch.full((n, -(-h // stride), -(-w // stride), oc), float("nan"), device="cuda")
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    tb.fp4_conv2d(f, x, y, n, h, w, stride, 0, work, ex)
    check_product(y.reshape(rows, oc), want, terms, ic, torch)
    z = torch.empty_like(y)
    tb.fp4_conv2d(f, x, z, n, h, w, stride, 0, work, ex, bias=bias, relu=True)
    assert torch.equal(z, torch.relu(y + bias))
    f.check()


def test_four_bit_layers_between_sparse_ones(tb, torch_cuda):
    """A bottleneck block as a network runs it, on one stream and as a captured graph: a 4-bit 1x1 layer, a
    sparse 3x3 layer, a strided 4-bit 1x1 layer, a 4-bit classifier on the pooled pixels."""
    torch = torch_cuda
    rng = np.random.default_rng(3)
    n, h, w = 2, 12, 12
    a_w, c_w, d_w = (rng.normal(0, 0.1, s).astype(np.float32) for s in ((64, 96), (160, 48), (100, 160)))
    b_w = rng.normal(0, 0.05, (48, 64, 3, 3)).astype(np.float32)
    b_w[rng.random(b_w.shape) < 0.8] = 0
    a, c, d = tb.Fp4Filter(a_w, 96, 64), tb.Fp4Filter(c_w, 48, 160, format=tb.FP4_NV), tb.Fp4Filter(d_w, 160, 100)
    b = tb.SparseFilter(b_w, 64, 48, 3)
    x = torch.rand(n, h, w, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    y1, y2, y3 = (torch.empty(n, e, e, k, device="cuda") for e, k in ((12, 64), (12, 48), (6, 160)))
    y4 = torch.empty(n, 100, device="cuda", dtype=torch.bfloat16)
    work = torch.empty(max(tb.fp4_workspace(f, n * h * w) for f in (a, c, d)), dtype=torch.uint8, device="cuda")

    def step(stream=None):
        tb.fp4_conv2d(a, x, y1, n, h, w, 1, 0, work, relu=True, cuda_stream=stream)
        tb.sparse_conv2d_fused(b, y1, y2, n, h, w, 1, 1, stream)
        tb.fp4_conv2d(c, y2, y3, n, h, w, 2, 0, work, -8, cuda_stream=stream)
        tb.fp4_linear(d, y3.view(n, 36 * 160)[:, :160], y4, n, work, cuda_stream=stream)
        return y4

    step()
    torch.cuda.synchronize()
    got = [t.clone() for t in (y1, y2, y3, y4)]
    # layer by layer in 64 bits, from what the layer before really gave
    v = lambda t, f, e: ref.values(*ref.quantize(f64(t.reshape(-1, t.shape[-1])), f, e), f, e)
    q = lambda m, f, e: ref.values(*ref.quantize(m, f, e), f, e)
    for t, src, m, fmt, ex, ew, k in ((got[0], x, a_w, ref.MX, 0, 0, 96), (got[2], got[1][:, ::2, ::2], c_w, ref.NV, -8, c.exponent_, 48),
                                      (got[3], got[2].reshape(n, -1)[:, :160], d_w, ref.MX, 0, 0, 160)):
        av, wv = v(src, fmt, ex), q(m, fmt, ew)
        want, terms = av @ wv.T, np.abs(av) @ np.abs(wv).T
        if t is got[0]:
            want = np.maximum(want, 0)
        check_product(t.reshape(-1, t.shape[-1]), want, terms, k, torch)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(stream)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(stream)
    first = x.clone()
    for k in range(3):
        x.copy_(first * (k + 1) / 2)
        for t in (y1, y2, y3, y4):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = y4.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(replayed, y4)
        if k == 1:
            assert torch.equal(y4, got[3])
    for f in (a, c, d):
        f.check()


def test_calls_on_two_streams_at_once(tb, torch_cuda):
    torch = torch_cuda
    f, _ = filter_and_weights(tb, torch, 384, 512, ref.NV, 1)
    x = [activations(torch, r, 512, r, spread=1.0) for r in (300, 5)]
    work = [torch.empty(tb.fp4_workspace(f, t.shape[0]), dtype=torch.uint8, device="cuda") for t in x]
    want = [torch.empty(t.shape[0], 384, device="cuda") for t in x]
    for t, w, y in zip(x, work, want):
        tb.fp4_linear(f, t, y, t.shape[0], w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in x]
    got = [torch.empty_like(y) for y in want]
    for _ in range(20):
        for t, w, y, s in zip(x, work, got, streams):
            tb.fp4_linear(f, t, y, t.shape[0], w, cuda_stream=s)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- filters, refusals --------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
def test_filters_from_host_and_device_arrays(tb, torch_cuda, fmt):
    torch = torch_cuda
    w = activations(torch, 130, 100, 21, spread=2.0)
    for source in (w, w.cpu(), w.cpu().numpy(), w.bfloat16(), w.half().cpu()):
        f = tb.Fp4Filter(source, 100, 130, format=fmt)
        dense = source.astype(np.float64) if isinstance(source, np.ndarray) else source.double().cpu().numpy()
        if fmt == ref.NV:
            assert 2688 * 2.0 ** f.exponent_ >= np.abs(dense).max() > 2688 * 2.0 ** (f.exponent_ - 1)
        code, byte = ref.quantize(dense, fmt, f.exponent_)
        got, scales = f.download()
        got = ref.unpack_codes(got, 2 * ref.pitch(100))
        assert np.array_equal(np.where(got == 8, 0, got)[:, :100], code) and not got[:, 100:].any()
        assert np.array_equal(scales, ref.pack_scales(byte, 100, fmt))
        info = f.info()
        assert (info.in_channel, info.out_channel, info.format, info.device, info.pitch) == (100, 130, fmt, 0, ref.pitch(100))
        f.close()
        with pytest.raises(RuntimeError):
            f.check()
    zero = tb.Fp4Filter(np.zeros((3, 5), np.float32), 5, 3, format=fmt)
    assert zero.exponent_ == 0
    y = torch.full((4, 3), 9.0, device="cuda")
    tb.fp4_linear(zero, activations(torch, 4, 5, 1), y, 4, torch.empty(tb.fp4_workspace(zero, 4), dtype=torch.uint8, device="cuda"))
    assert not y.any()


def test_refusals_on_the_device(tb, torch_cuda):
    torch = torch_cuda
    f, _ = filter_and_weights(tb, torch, 4096, 4096, ref.MX, 1)
    x = activations(torch, 300, 4096, 2)
    y = torch.full((300, 4096), 5.0, device="cuda")
    codes, scales = quantized(tb, torch, x, ref.MX)
    need = tb.fp4_workspace(f, 300)
    assert need  # (products of fewer values quantise them on their own)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()

    def refused(call, status=1):
        with pytest.raises(tb.TetrisError) as e:
            call()
        assert e.value.status == status, str(e.value)

    refused(lambda: tb.fp4_linear(f, x, y, 300, work[:need - 1]))
    refused(lambda: tb.fp4_linear(f, x, y, 300))
    refused(lambda: tb.fp4_linear(f, x.cpu(), y, 300, work))
    refused(lambda: tb.fp4_linear(f, x, y.cpu(), 300, work))
    refused(lambda: tb.fp4_linear(f, x, y, 300, work.cpu()))
    refused(lambda: tb.fp4_linear(f, x, y, 300, work, exponent=2))
    refused(lambda: tb.fp4_linear(f, x, y, 300, work, bias=torch.zeros(4096)))
    refused(lambda: tb.fp4_product(f, codes.cpu(), scales, y, 300))
    refused(lambda: tb.fp4_product(f, codes, scales.cpu(), y, 300))
    refused(lambda: tb.fp4_product(f, codes[1:], scales, y, 300))
    refused(lambda: tb.fp4_product(f, codes, scales, y, -1))
    refused(lambda: tb.fp4_product(f, codes.data_ptr(), scales, y.data_ptr(), 300, ld=4095))
    refused(lambda: tb.fp4_product(f, codes.data_ptr(), scales.data_ptr(), y.data_ptr(), 300, dtype=9))
    refused(lambda: tb.fp4_quantize(x.cpu(), codes, scales, 300, 4096, ref.MX))
    refused(lambda: tb.fp4_dequantize(codes, scales, x.cpu(), 300, 4096, ref.MX))
    refused(lambda: tb.fp4_conv2d(f, x, y, 3, 10, 10, 1, 1, work), 3)
    refused(lambda: tb.fp4_conv2d(f, x, y, 3, 10, 10, 0, 0, work))
    lib = tb.lib()
    assert lib.tetris_fp4_linear(f.handle, x.data_ptr(), 0, 300, 0, 0, None, y.data_ptr(), 0, 0, 2, work.data_ptr(), need, None) == 1
    assert lib.tetris_fp4_linear(f.handle, None, 0, 300, 0, 0, None, y.data_ptr(), 0, 0, 0, work.data_ptr(), need, None) == 1
    assert lib.tetris_fp4_linear(f.handle, x.data_ptr(), 0, 300, 0, 0, None, None, 0, 0, 0, work.data_ptr(), need, None) == 1
    for call in (lambda: tb.fp4_linear(f, x, y, 301, work), lambda: tb.fp4_linear(f, x[:, :100], y, 300, work),
                 lambda: tb.fp4_linear(f, x.double(), y, 300, work), lambda: tb.fp4_product(f, codes, scales, y[:299], 300),
                 lambda: tb.fp4_linear(f, x, y, 300, work, bias=torch.zeros(4095, device="cuda")),
                 lambda: tb.fp4_conv2d(f, x, y, 4, 10, 10, 1, 0, work), lambda: tb.fp4_conv2d(f, x.half(), y, 3, 10, 10, 1, 0, work)):
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()
    assert bool((y == 5.0).all())
    tb.fp4_linear(f, x[:0], y[:0], 0, work)
    tb.fp4_product(f, codes, scales, y[:0], 0)
    tb.fp4_conv2d(f, x[:0], y[:0], 0, 10, 10, 1, 0, work)
    torch.cuda.synchronize()
    assert bool((y == 5.0).all())


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_bounded_wait_gives_up_and_the_next_product_passes(tb, torch_cuda, rows):
    """Every CTA leaves out its first activations: the waits run out, the launch returns, the status is read, and
    the next product of the same filter is right."""
    torch = torch_cuda
    k, n = 600, 200
    f, w = filter_and_weights(tb, torch, n, k, ref.NV, 31)
    x = activations(torch, rows, k, 32, spread=1.0)
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    y = torch.empty(rows, n, device="cuda")
    torch.cuda.synchronize()
    tb.test_inject(1, 2000)
    try:
        tb.fp4_linear(f, x, y, rows, work)
        with pytest.raises(tb.TetrisError) as e:
            f.check()
        assert e.value.status == 2 and "gave up" in str(e.value)
    finally:
        tb.test_inject(0)
    f.check()
    tb.fp4_linear(f, x, y, rows, work)
    f.check()
    want, terms = reference_product(x, w, ref.NV, 0, f.exponent_)
    check_product(y, want, terms, k, torch)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,k,n", [(3000, 4096, 4096), (300, 8192, 200), (40, 16384, 300), (1, 16384, 200), (1, 8192, 20000), (2, 8192, 9000)])
def test_give_up_where_stages_are_used_again(tb, torch_cuda, fmt, rows, k, n):
    """More K steps than the ring has stages: after a wait that gave up nothing may be sent for into a stage whose
    last load is still owed, and the product that follows at once, placed while the first one ends, is right.
    Many tiles of a CTA, clusters, rows quantised by the product itself."""
    torch = torch_cuda
    x = activations(torch, rows, k, 33, spread=1.0, dtype="bf16")
    f, w = filter_and_weights(tb, torch, n, k, fmt, 34)
    work = torch.empty(tb.fp4_workspace(f, rows), dtype=torch.uint8, device="cuda")
    want, y, z = (torch.empty(rows, n, device="cuda") for _ in range(3))
    tb.fp4_linear(f, x, want, rows, work)
    f.check()
    for _ in range(3):
        z.fill_(float("nan"))
        torch.cuda.synchronize()
        tb.test_inject(1, 500)
        try:
            tb.fp4_linear(f, x, y, rows, work)
        finally:
            tb.test_inject(0)
        tb.fp4_linear(f, x, z, rows, work)
        with pytest.raises(tb.TetrisError) as e:
            f.check()
        assert e.value.status == 2 and "gave up" in str(e.value)
        assert torch.equal(z, want)
    f.check()


def test_offsets_past_32_bits(tb, torch_cuda):
    """17 GB of activations, 4.3 GB of codes: the last rows come out as they do on their own."""
    torch = torch_cuda
    cols, rows, n, part = 16384, 530000, 48, 1000
    base = activations(torch, part, cols, 5, spread=1.0, dtype="bf16")
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x.view(rows // part, part, cols)[:] = base
    f, w = filter_and_weights(tb, torch, n, cols, ref.MX, 6)
    want_codes, want_scales = quantized(tb, torch, base, ref.MX)
    codes, scales = [torch.empty(s, dtype=torch.uint8, device="cuda") for s in tb.fp4_sizes(rows, cols, ref.MX)]
    tb.fp4_quantize(x, codes, scales, rows, cols, ref.MX)
    pitch = ref.pitch(cols)
    assert torch.equal(codes[-part * pitch:], want_codes[:part * pitch])
    y = torch.empty(rows, n, device="cuda")
    tb.fp4_product(f, codes, scales, y, rows)
    f.check()
    check_product(y[-part:], *reference_product(base, w, ref.MX, 0, 0), cols, torch)
    assert torch.equal(y[-part:], y[:part])
    x.zero_()
    tb.fp4_dequantize(codes, scales, x, rows, cols, ref.MX)
    back = torch.empty_like(base)
    tb.fp4_dequantize(want_codes, want_scales, back, part, cols, ref.MX)
    assert torch.equal(x[-part:], back)


def test_first_call_inside_a_capture(torch_cuda):
    """A process whose first product is captured: nothing on the launch path needs an earlier call."""
    import os
    import subprocess
    import sys
    code = """
import sys
sys.path.insert(0, %r)
from conftest import load_package
import torch
tb = load_package()
w = torch.randn(300, 512, device='cuda')
f = tb.Fp4Filter(w, 512, 300)
x, y = torch.randn(700, 512, device='cuda'), torch.zeros(700, 300, device='cuda')
z = torch.zeros(2, 300, device='cuda')
room = torch.empty(tb.fp4_workspace(f, 700), dtype=torch.uint8, device='cuda')
torch.cuda.synchronize()
s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    tb.fp4_linear(f, x, y, 700, room, cuda_stream=s)
    tb.fp4_linear(f, x[:2], z, 2, cuda_stream=s)
g.replay()
torch.cuda.synchronize()
f.check()
a = torch.empty_like(y)
tb.fp4_linear(f, x, a, 700, room)
assert torch.equal(a, y) and bool(y.abs().sum() > 0)
tb.fp4_linear(f, x[:2], a, 2)
assert torch.equal(a[:2], z)
print('captured')
""" % os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
