"""The 4-bit floating-point operators as a list of cases that a timing program can run.

A case is a dict of plain values; `prepare` builds what a program holds before the call, `run` is one
pass: in elementary torch operations where `own` is false, through the engine's public entry points
where it is true.  The kinds:

  quantize  rows of activations into 4-bit codes and block scales, and those back into values
  product   quantised activations times a 4-bit filter: Y = A W^T (+ bias, ReLU)
  linear    floating-point activations times a 4-bit filter, quantised on the way
  conv      a 1x1 layer on NHWC activations with a 4-bit filter: the same on an image's pixels

Formats.  Codes are E2M1: a sign and a magnitude out of {0, 0.5, 1, 1.5, 2, 3, 4, 6}, two to a byte,
the even column in the low half, a row's bytes padded with zeros to a multiple of 16.
  mx  blocks of 32 columns; scale 2^e (E8M0: e + 127), e = floor(log2(largest |x|)) - 2, at least -127
  nv  blocks of 16 columns of u = x 2^-exponent; scale E4M3 of (largest |u|) / 6, at most 448
A code is x (or u) over its block's scale, rounded to nearest, ties to the even code, at most 6.
Scales lie in tiles of 128 rows x 4 blocks: byte (r % 32) * 16 + (r / 32) * 4 + j of a tile is block j
of row r, tiles in the order of the blocks, then of the rows.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_PKG = "tetris-artifact-evalution_b200"
_BLOCK = {"mx": 32, "nv": 16}
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _package():
    if "tetris_b200" not in sys.modules:
        here = os.path.join(os.getcwd(), _PKG)
        spec = importlib.util.spec_from_file_location(
            "tetris_b200", os.path.join(here, "__init__.py"), submodule_search_locations=[here])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["tetris_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["tetris_b200"]


# ---- cases --------------------------------------------------------------------------------------
def _quantize(fmt, rows, k, x, y):
    return {"kind": "quantize", "fmt": fmt, "rows": rows, "k": k, "x": x, "y": y}


def _product(fmt, rows, k, n, y, relu=False, bias=False):
    return {"kind": "product", "fmt": fmt, "rows": rows, "k": k, "n": n, "y": y, "relu": relu, "bias": bias}


def _linear(fmt, rows, k, n, x, y, relu=False, bias=False):
    return {"kind": "linear", "fmt": fmt, "rows": rows, "k": k, "n": n, "x": x, "y": y, "relu": relu, "bias": bias}


def _conv(fmt, batch, h, w, k, n, stride=1, relu=False, sparsity=0.8):
    return {"kind": "conv", "fmt": fmt, "batch": batch, "h": h, "w": w, "k": k, "n": n, "stride": stride,
            "relu": relu, "sparsity": sparsity}


def listed():
    return [
        # the activations of ResNet-50's first stage (256 channels at 56x56, 16 images)
        dict(_quantize("mx", 50176, 256, "fp32", "fp32"), name="quantize mx 50176x256 fp32"),
        # a long batch of wide rows in 16 bits
        dict(_quantize("nv", 4096, 8192, "bf16", "bf16"), name="quantize nv 4096x8192 bf16"),
        # few rows of odd length: the smallest call, where latency counts
        dict(_quantize("nv", 7, 4095, "fp32", "fp32"), name="quantize nv 7x4095 fp32"),
        # one quantised row against a square filter: serving one input
        dict(_product("mx", 1, 4096, 4096, "fp32"), name="product mx 1x4096x4096"),
        # the largest: where the tensor cores' rate counts
        dict(_product("nv", 8192, 4096, 8192, "bf16"), name="product nv 8192x4096x8192"),
        # nothing a multiple of a tile: 333 rows of a 2048 -> 1000 classifier
        dict(_product("nv", 333, 2048, 1000, "fp32", bias=True), name="product nv 333x2048x1000"),
        # the classifier of ResNet-50 on one image: the smallest product
        dict(_linear("mx", 1, 2048, 1000, "fp32", "fp32", bias=True), name="linear mx 1x2048x1000 fp32"),
        # a serving batch against a wide filter: bound by the reading of the filter
        dict(_linear("nv", 16, 8192, 8192, "bf16", "bf16"), name="linear nv 16x8192x8192 bf16"),
        # a long batch in 16 bits through a widening layer
        dict(_linear("mx", 4096, 4096, 16384, "bf16", "bf16", relu=True, bias=True), name="linear mx 4096x4096x16384"),
        # ResNet-50's 64 -> 256 at 56x56, 16 images: bound by the writing of the activations
        dict(_conv("mx", 16, 56, 56, 64, 256, relu=True), name="conv mx 56x56 64-256 b16"),
        # the last layer of YOLOv3's first detection head: 255 channels on 13x13 images
        dict(_conv("nv", 8, 13, 13, 1024, 255, sparsity=0.875), name="conv nv 13x13 1024-255 b8"),
        # a downsampling projection of ResNet-50: every second pixel of 56x56 images
        dict(_conv("nv", 16, 56, 56, 256, 512, stride=2), name="conv nv 56x56 s2 256-512 b16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _columns(rng, lo, hi):
    """Widths: mostly multiples of 64 or 16, odd ones among them."""
    c = _log_int(rng, lo, hi)
    step = rng.choice([64, 64, 64, 16, 16, 1])
    return max(lo, min(hi, (c + step - 1) // step * step))


def draw(rng):
    kind = rng.choice(["quantize", "quantize", "product", "product", "product", "linear", "linear", "linear", "conv", "conv"])
    fmt = rng.choice(["mx", "nv"])
    x, y = rng.choice(["fp32", "bf16", "fp16"]), rng.choice(["fp32", "fp32", "bf16", "fp16"])
    while True:
        if kind == "conv":
            h = _log_int(rng, 7, 112)
            case = _conv(fmt, _log_int(rng, 1, 16), h, h if rng.random() < 0.7 else _log_int(rng, 7, 112),
                         _columns(rng, 16, 2048), _columns(rng, 16, 2048), rng.choice([1, 1, 2]), rng.random() < 0.5,
                         round(rng.uniform(0.0, 0.95), 3))
        elif kind == "quantize":
            case = _quantize(fmt, _log_int(rng, 1, 65536), _columns(rng, 16, 16384), x, y)
        else:
            rows = _log_int(rng, 1, 64) if rng.random() < 0.5 else _log_int(rng, 32, 65536)
            k, n = _columns(rng, 16, 16384), _columns(rng, 16, 16384)
            relu, bias = rng.random() < 0.3, rng.random() < 0.5
            case = _product(fmt, rows, k, n, y, relu, bias) if kind == "product" else _linear(fmt, rows, k, n, x, y, relu, bias)
        w = work(case)
        if w["flops"] <= 2.0 * 8192 * 4096 * 8192 and w["bytes"] <= 120e6:
            return case


def _extent(size, stride):
    return (size - 1) // stride + 1


def _rows(case):
    if case["kind"] == "conv":
        return case["batch"] * _extent(case["h"], case["stride"]) * _extent(case["w"], case["stride"])
    return case["rows"]


def work(case):
    """One reading of what goes in and one writing of what comes out; 2 operations a product."""
    rows, k, block = _rows(case), case["k"], _BLOCK[case["fmt"]]
    quantised = -(-k // 2) + -(-k // block)  # bytes of a row's codes and scales
    if case["kind"] == "quantize":
        return {"bytes": float(rows * (k * _BYTES[case["x"]] + 2 * quantised + k * _BYTES[case["y"]])), "flops": 4.0 * rows * k}
    n = case["n"]
    out = rows * n * _BYTES[case.get("y", "fp32")] + (4 * n if case.get("bias") else 0)
    into = rows * (quantised if case["kind"] == "product" else k * _BYTES[case.get("x", "fp32")])
    return {"bytes": float(into + n * quantised + out), "flops": 2.0 * rows * n * k}


# ---- the operators in elementary operations -----------------------------------------------------
def _pow2(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e)


def _floor_log2(v):
    """Exponent of v > 0, exactly."""
    return torch.frexp(v).exponent.to(torch.int64) - 1


def _blocks(x, block):
    """[rows, k] as [rows, blocks, block] with zeros behind the last column."""
    rows, k = x.shape
    wide = torch.zeros(rows, -(-k // block) * block, dtype=x.dtype, device=x.device)
    wide[:, :k] = x
    return wide.view(rows, -1, block)


def _e4m3(v):
    """v >= 0 rounded to E4M3: steps of 2^-3 of its binade, of 2^-9 below 2^-6; at most 448."""
    step = _pow2(torch.clamp(_floor_log2(torch.clamp(v, min=2.0 ** -40)), min=-6) - 3)
    return torch.clamp(torch.round(v / step) * step, max=448.0)


def _scales(top, fmt):
    """Block scales, float64, from the largest magnitudes of the blocks."""
    if fmt == "nv":
        return _e4m3(top / 6)
    return _pow2(torch.clamp(_floor_log2(torch.clamp(top, min=2.0 ** -149)) - 2, min=-127))


def _magnitudes(q):
    """0 <= q rounded to the magnitudes of E2M1."""
    step = torch.where(q < 2, 0.5, torch.where(q < 4, 1.0, 2.0))
    return torch.clamp(torch.round(q / step) * step, max=6.0)


def _quantised(x, fmt, exponent):
    """(signed E2M1 values [rows, blocks, block], scales [rows, blocks]), float64 with borders in 64 bits."""
    u = _blocks(x.double() * 2.0 ** -exponent, _BLOCK[fmt])
    s = _scales(u.abs().amax(2), fmt)
    m = _magnitudes(u.abs() / torch.where(s > 0, s, 1.0)[..., None])
    return torch.where(s[..., None] > 0, torch.copysign(m, u), torch.zeros_like(m)), s


def _values(x, fmt, exponent):
    """x as its quantised form stands for it, float32."""
    m, s = _quantised(x, fmt, exponent)
    return (m * s[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]].mul(2.0 ** exponent).float()


# ---- packed form --------------------------------------------------------------------------------
def _pitch(k):
    return -(-k // 32) * 16


def _tile_counts(rows, k, fmt):
    return -(-rows // 128), -(-k // (4 * _BLOCK[fmt]))


def _pack(x, fmt, exponent):
    """(codes uint8 [rows, pitch], scales uint8 in tiles) of the quantised form of x."""
    rows, k = x.shape
    m, s = _quantised(x, fmt, exponent)
    a = m.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(m).to(torch.uint8) << 3)
    code = code.reshape(rows, -1)
    wide = torch.zeros(rows, 2 * _pitch(k), dtype=torch.uint8, device=x.device)
    wide[:, :min(code.shape[1], wide.shape[1])] = code[:, :wide.shape[1]]
    wide[:, k:] = 0
    codes = wide[:, 0::2] | (wide[:, 1::2] << 4)
    byte = s.float().to(torch.float8_e4m3fn).view(torch.uint8) if fmt == "nv" else (_floor_log2(s) + 127).to(torch.uint8)
    tr, tk = _tile_counts(rows, k, fmt)
    full = torch.zeros(tr * 128, tk * 4, dtype=torch.uint8, device=x.device)
    full[:rows, :byte.shape[1]] = byte
    return codes.contiguous(), full.view(tr, 4, 32, tk, 4).permute(0, 3, 2, 1, 4).contiguous()


def _unpack(codes, scales, rows, k, fmt, exponent):
    """float32 values of the packed form."""
    nibble = torch.stack((codes & 15, codes >> 4), 2).reshape(rows, -1)
    a = (nibble & 7).float()
    a = torch.where(a < 4, a * 0.5, torch.where(a < 6, a - 2, a * 2 - 8))
    v = torch.where(nibble >= 8, -a, a)
    byte = scales.permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[:rows]
    s = byte.view(torch.float8_e4m3fn).float() if fmt == "nv" else torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte.int() - 127)
    s = s.repeat_interleave(_BLOCK[fmt], 1)
    return v[:, :k] * s[:, :k] * 2.0 ** exponent


# ---- a pass -------------------------------------------------------------------------------------
def _inputs(case, seed):
    """(activations, weights or None, bias or None) of the case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rows, k = _rows(case), case["k"]
    if case["kind"] == "conv":  # what a ReLU leaves, and a pruned filter
        x = torch.rand(case["batch"], case["h"], case["w"], k, device="cuda", generator=g)
        x *= torch.rand(x.shape, device="cuda", generator=g) >= 0.5
    else:  # rows of different magnitude, a few wide columns
        x = torch.randn(rows, k, device="cuda", generator=g)
        x *= torch.exp2(torch.randn(rows, 1, device="cuda", generator=g))
        x *= 1 + 7 * (torch.rand(1, k, device="cuda", generator=g) < 0.01)
    x = x.to(_TYPES[case.get("x", "fp32")])
    w = b = None
    if case["kind"] != "quantize":
        w = torch.randn(case["n"], k, device="cuda", generator=g) * 0.05
        if case["kind"] == "conv":
            w *= torch.rand(w.shape, device="cuda", generator=g) >= case["sparsity"]
        if case.get("bias"):
            b = torch.randn(case["n"], device="cuda", generator=g)
    return x, w, b


def _exponents(case):
    """Exponents of the whole tensors (activations, weights): the nv form holds up to 2688 * 2^exponent, here
    1.3 for what a ReLU leaves of an image, 1344 for wide rows, 0.33 for weights; the mx form needs none."""
    if case["fmt"] == "mx":
        return 0, 0
    return (-11 if case["kind"] == "conv" else -1), -13


def prepare(case, seed):
    x, w, b = _inputs(case, seed)
    ex, ew = _exponents(case)
    state = {"case": case, "bias": b, "ex": ex}
    if case["kind"] == "product":
        state["codes"], state["scales"] = _pack(x, case["fmt"], ex)
    else:
        state["x"] = x
    if own:
        tb = state["tb"] = _package()
        fmt = state["fmt"] = tb.FP4_MX if case["fmt"] == "mx" else tb.FP4_NV
        rows, k, dev = _rows(case), case["k"], x.device
        if w is not None:  # the filter as the engine keeps it, room for the result
            state["filter"] = tb.Fp4Filter(w, k, case["n"], format=fmt, exponent=ew)
            state["y"] = torch.empty(rows, case["n"], dtype=_TYPES[case.get("y", "fp32")], device=dev)
        if case["kind"] == "quantize":
            sizes = tb.fp4_sizes(rows, k, fmt)
            state["codes"], state["scales"] = (torch.empty(s, dtype=torch.uint8, device=dev) for s in sizes)
            state["y"] = torch.empty(rows, k, dtype=_TYPES[case["y"]], device=dev)
        elif case["kind"] != "product":
            state["workspace"] = torch.empty(tb.fp4_workspace(state["filter"], rows), dtype=torch.uint8, device=dev)
    elif w is not None:  # the values that the 4-bit filter stands for
        state["w"] = _values(w, case["fmt"], ew)
    return state


def _run_own(s):
    c, tb = s["case"], s["tb"]
    if c["kind"] == "quantize":
        tb.fp4_quantize(s["x"], s["codes"], s["scales"], c["rows"], c["k"], s["fmt"], s["ex"])
        tb.fp4_dequantize(s["codes"], s["scales"], s["y"], c["rows"], c["k"], s["fmt"], s["ex"])
    elif c["kind"] == "product":
        tb.fp4_product(s["filter"], s["codes"], s["scales"], s["y"], c["rows"], s["ex"], bias=s["bias"], relu=c["relu"])
    elif c["kind"] == "linear":
        tb.fp4_linear(s["filter"], s["x"], s["y"], c["rows"], s["workspace"], s["ex"], bias=s["bias"], relu=c["relu"])
    else:
        tb.fp4_conv2d(s["filter"], s["x"], s["y"], c["batch"], c["h"], c["w"], c["stride"], 0, s["workspace"], s["ex"], relu=c["relu"])
    return s["y"]


def run(state):
    if own:
        return _run_own(state)
    c, ex = state["case"], state["ex"]
    if c["kind"] == "quantize":
        codes, scales = _pack(state["x"], c["fmt"], ex)
        return _unpack(codes, scales, c["rows"], c["k"], c["fmt"], ex).to(_TYPES[c["y"]])
    if c["kind"] == "product":
        a = _unpack(state["codes"], state["scales"], c["rows"], c["k"], c["fmt"], ex)
    else:
        x = state["x"]
        a = _values(x[:, ::c["stride"], ::c["stride"]].reshape(-1, c["k"]) if c["kind"] == "conv" else x, c["fmt"], ex)
    y = a @ state["w"].t()
    if state["bias"] is not None:
        y = y + state["bias"]
    if c["relu"]:
        y = torch.clamp(y, min=0)
    return y.to(_TYPES[c.get("y", "fp32")])


# ---- the operators from their definition, in 64 bits ---------------------------------------------
_CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest(v, table):
    """The entry of an ascending table nearest to v >= 0; halfway between two, the one of even index."""
    t = torch.tensor(table, dtype=torch.float64, device=v.device)
    half = (t[:-1] + t[1:]) / 2
    at = torch.searchsorted(half, v.contiguous())           # a border goes down ...
    up = torch.searchsorted(half, v.contiguous(), right=True)  # ... or up
    return t[torch.where((at != up) & (at % 2 == 1), up, at)]


def _stands_for(x, fmt, exponent):
    """float64 values of the quantised form of x, from tables of what 4 and 8 bits can hold."""
    block, (rows, k) = _BLOCK[fmt], x.shape
    u = torch.nn.functional.pad(x.double() / 2.0 ** exponent, (0, -k % block)).reshape(rows, -1, block)
    top = u.abs().max(dim=2, keepdim=True).values
    if fmt == "nv":
        table = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 9) for e in range(16) for m in range(8)]
        s = _nearest(top / 6, table[:127])
    else:
        powers = torch.tensor([2.0 ** e for e in range(-125, 128)], dtype=torch.float64, device=x.device)
        s = torch.cat((powers[:1], powers))[torch.searchsorted(powers, top, right=True)] / 4
    v = _nearest(u.abs() / torch.where(s == 0, torch.ones_like(s), s), _CODES) * s
    return (v * torch.sign(u)).reshape(rows, -1)[:, :k] * 2.0 ** exponent


def exact(case, seed):
    x, w, b = _inputs(case, seed)
    ex, ew = _exponents(case)
    if case["kind"] == "conv":
        x = x[:, ::case["stride"], ::case["stride"]].reshape(-1, case["k"])
    a = _stands_for(x, case["fmt"], ex)
    if case["kind"] == "quantize":
        return a
    y = torch.matmul(a, _stands_for(w, case["fmt"], ew).t())
    if b is not None:
        y += b.double()
    return torch.relu(y) if case["relu"] else y
