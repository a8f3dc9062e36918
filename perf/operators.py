"""The operators of microscaled products, as a serving program calls them: rows and weights in blocks of 32 numbers that share
a power of two, held in 4 bits (e2m1) or 8 (e4m3).

A block's scale is the smallest power of two with which no number of the block is past the type's largest (6, or 448); a number
is its nearest element times the scale, ties to the even element.  Weights are held in 4 bits, the rows that meet them in 8 or
in 4, sums are 32 bits wide.

Kinds of case:

* "quantise": rows of bfloat16 to blocks: the attention's output in front of the output projection, and a weight at load time.
* "norm": the residual's addition (of a bfloat16 result, or of the float32 parts that a product with a split K leaves), the
  root-mean-square norm, and its rows as blocks.
* "product": rows in blocks times a weight in blocks.
* "gate_up": the product of a gated feed-forward's first half, silu(gate) * up, and its rows as blocks for the second half.

Sizes: one token, a few decoding requests, prompt portions; the widths of the Qwen3-4B, 8B and 32B shapes that the framework's
product tables name, and odd ones.  Rows are normal with a few channels that are far larger than the others, as a decoder's
are; weights are N(0, 0.02).
"""
from __future__ import annotations

import math
import random

import torch

own = False

BLOCK = 32
LARGEST = {"mxfp8": 448.0, "mxfp4": 6.0}
EPS = 1e-6
QWEN3_WIDTHS = (2560, 4096, 5120)
QWEN3_PRODUCTS = ((6144, 2560), (2560, 4096), (2560, 9728), (6144, 4096), (4096, 12288), (10240, 5120))       # (N, K)
QWEN3_GATED = ((9728, 2560), (12288, 4096))                                                                   # (feed-forward width, K)


def listed() -> list:
    return [
        # the attention's output of eight decoding requests, in front of the output projection
        dict(name="quantise-8x4096-8bit", kind="quantise", rows=8, width=4096, form="mxfp8"),
        # a gate|up weight as it is loaded, and the values that its elements stand for
        dict(name="quantise-19456x2560-4bit", kind="quantise", rows=19456, width=2560, form="mxfp4"),
        # one decoding request: the residual's addition of an output projection that left four parts
        dict(name="norm-1x2560-parts4", kind="norm", rows=1, width=2560, parts=4, form="mxfp8"),
        # an odd batch of an odd width
        dict(name="norm-37x1530", kind="norm", rows=37, width=1530, parts=0, form="mxfp8"),
        # a prompt portion
        dict(name="norm-4096x4096", kind="norm", rows=4096, width=4096, parts=0, form="mxfp8"),
        # one decoding request's second half of the feed-forward
        dict(name="product-1x2560x9728", kind="product", rows=1, n=2560, k=9728, form="mxfp8"),
        # q, k and v of eight decoding requests
        dict(name="product-8x6144x2560", kind="product", rows=8, n=6144, k=2560, form="mxfp8"),
        # a ragged step: a hundred rows, nothing a multiple of anything
        dict(name="product-100x1531x2610", kind="product", rows=100, n=1531, k=2610, form="mxfp8"),
        # a prompt portion's second half of the feed-forward
        dict(name="product-2048x2560x9728", kind="product", rows=2048, n=2560, k=9728, form="mxfp8"),
        # a prompt portion whose rows are held in 4 bits too
        dict(name="product-4096x6144x4096-4bit", kind="product", rows=4096, n=6144, k=4096, form="mxfp4"),
        # the first half of the feed-forward: eight decoding requests, and a prompt portion
        dict(name="gate_up-8x9728x2560", kind="gate_up", rows=8, ff=9728, k=2560, form="mxfp8"),
        dict(name="gate_up-4096x12288x4096", kind="gate_up", rows=4096, ff=12288, k=4096, form="mxfp8"),
    ]


def _between(rng: random.Random, low: int, high: int) -> int:
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("quantise", "norm", "product", "product", "gate_up"))
    rows = rng.choice((_between(rng, 1, 64), _between(rng, 1, 4096)))
    form = rng.choice(("mxfp8", "mxfp8", "mxfp4"))
    if kind == "quantise":
        return dict(kind=kind, rows=rows, width=rng.choice((rng.choice(QWEN3_WIDTHS), _between(rng, 33, 12288))), form=form)
    if kind == "norm":
        width = rng.choice((rng.choice(QWEN3_WIDTHS), _between(rng, 33, 8192)))
        return dict(kind=kind, rows=rows, width=width, parts=rng.choice((0, 1, 2, 4, 7)) if rows <= 64 else 0, form="mxfp8")
    if kind == "product":
        n, k = rng.choice((rng.choice(QWEN3_PRODUCTS), (_between(rng, 16, 10240), _between(rng, 33, 12288))))
        return dict(kind=kind, rows=rows, n=n, k=k, form=form)
    ff, k = rng.choice((rng.choice(QWEN3_GATED), (32 * _between(rng, 1, 384), _between(rng, 33, 4096))))
    return dict(kind=kind, rows=rows, ff=ff, k=k, form="mxfp8")


# ---------------------------------------------------------------- inputs


def _numbers(seed: int, *shape, std: float = 1.0) -> torch.Tensor:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda") * std


def _activations(seed: int, rows: int, width: int) -> torch.Tensor:
    """Normal rows, every 97th channel or so a dozen times larger."""
    x = _numbers(seed, rows, width)
    x[:, seed % 61::97] *= 12.0
    return x


def _weight(seed: int, n: int, k: int, step: int = 4096) -> tuple:
    """(elements as codes of 4 bits [n, blocks * 32], scales as codes of 8 bits [n, blocks]) of an N(0, 0.02) weight."""
    parts = [_codes(_numbers(seed + 7 * i, min(step, n - i), k, std=0.02), "mxfp4") for i in range(0, n, step)]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def prepare(case: dict, seed: int) -> dict:
    kind, rows = case["kind"], case["rows"]
    state = {"case": dict(case)}
    if kind == "quantise":
        x = _activations(seed, rows, case["width"]) if case["form"] == "mxfp8" or rows <= 4096 else _numbers(seed, rows, case["width"], std=0.02)
        state["x"] = x.bfloat16()
        return state
    if kind == "norm":
        width, parts = case["width"], case["parts"]
        state["residual"] = _activations(seed, rows, width)
        state["delta"] = _numbers(seed + 1, parts, rows, width, std=0.1) if parts else _numbers(seed + 1, rows, width, std=0.2).bfloat16()
        state["weight"] = (1.0 + _numbers(seed + 2, width, std=0.1)).bfloat16()
        return state
    x = _codes(_activations(seed, rows, case["k"]), case["form"])
    w = _weight(seed + 1, 2 * case["ff"] if kind == "gate_up" else case["n"], case["k"])
    if own:     # a serving program holds its rows as the operators in front left them, and its weights laid out once
        from arle_amd.kernels import mx

        state["x"] = mx.rows_from_codes(*x, case["k"], case["form"])
        state["w"] = mx.lay_weight(mx.rows_from_codes(*w, case["k"], "mxfp4"), gated=kind == "gate_up")
    else:
        state["x"], state["w"] = x, w
    return state


# ---------------------------------------------------------------- plain forms


def _codes(x: torch.Tensor, form: str) -> tuple:
    """(elements as codes uint8 [rows, blocks * 32], scales as codes uint8 [rows, blocks]) of float32 rows: a scale of code c is
    2^(c - 127); codes of e2m1 are sign, two bits of exponent, one of mantissa, a byte each.  Past the width: zeros."""
    rows, width = x.shape
    blocks = -(-width // BLOCK)
    v = torch.nn.functional.pad(x, (0, blocks * BLOCK - width)).view(rows, blocks, BLOCK)
    bits = v.abs().amax(-1).view(torch.int32)
    exponent, fraction = bits >> 23, bits & 0x7FFFFF
    of_largest = {"mxfp8": (8, 0x600000), "mxfp4": (2, 0x400000)}[form]        # 448 = 1.75 * 2^8, 6 = 1.5 * 2^2
    scale = (exponent - of_largest[0] + (fraction > of_largest[1])).clamp(min=0)
    v = torch.ldexp(v, (127 - scale).float().unsqueeze(-1))
    if form == "mxfp8":
        codes = v.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = v.abs()
        codes = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)) | (v.signbit().byte() << 3)
    return codes.view(rows, blocks * BLOCK), scale.to(torch.uint8)


def _values(codes: torch.Tensor, scales: torch.Tensor, width: int, form: str) -> torch.Tensor:
    """float32 [rows, width]: what the elements stand for."""
    if form == "mxfp8":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)[codes.int()]
    v = torch.ldexp(v.view(*scales.shape, BLOCK), (scales.float() - 127).unsqueeze(-1))
    return v.reshape(scales.shape[0], -1)[:, :width]


def _eight_bits(codes: torch.Tensor, scales: torch.Tensor, width: int) -> list:
    return [codes[:, :width].view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)]


def _plain(state: dict):
    case = state["case"]
    if case["kind"] == "quantise":
        codes, scales = _codes(state["x"].float(), case["form"])
        if case["form"] == "mxfp8":
            return _eight_bits(codes, scales, case["width"])
        return [_values(codes, scales, case["width"], "mxfp4").bfloat16()]
    if case["kind"] == "norm":
        delta, residual = state["delta"].float(), state["residual"]
        residual += delta.sum(0) if case["parts"] else delta
        y = residual * torch.rsqrt((residual * residual).mean(-1, keepdim=True) + EPS) * state["weight"].float()
        return [residual, *_eight_bits(*_codes(y, "mxfp8"), case["width"])]
    y = _values(*state["x"], case["k"], case["form"]) @ _values(*state["w"], case["k"], "mxfp4").T
    if case["kind"] == "product":
        return [y.bfloat16()]
    gate, up = y[:, :case["ff"]], y[:, case["ff"]:]
    return _eight_bits(*_codes(gate / (1.0 + torch.exp(-gate)) * up, "mxfp8"), case["ff"])


# ---------------------------------------------------------------- the framework's operators


def _own(state: dict):
    from arle_amd.kernels import mx

    case = state["case"]
    if case["kind"] == "quantise":
        rows = mx.quantize(state["x"], case["form"])
        return [rows.elements_e4m3(), rows.scales_e8m0()] if case["form"] == "mxfp8" else [mx.values(rows, torch.bfloat16)]
    if case["kind"] == "norm":
        rows = mx.add_rmsnorm(state["residual"], state["delta"], state["weight"], EPS, "mxfp8")
        return [state["residual"], rows.elements_e4m3(), rows.scales_e8m0()]
    if case["kind"] == "product":
        return [mx.gemm(state["x"], state["w"], torch.bfloat16)]
    rows = mx.gate_up_act(state["x"], state["w"], "mxfp8")
    return [rows.elements_e4m3(), rows.scales_e8m0()]


def run(state: dict):
    return _own(state) if own else _plain(state)


def work(case: dict) -> dict:
    rows = case["rows"]
    held = lambda width, form: width * (1.0 if form == "mxfp8" else 0.5) + math.ceil(width / BLOCK)     # bytes of a row in blocks
    if case["kind"] == "quantise":
        width = case["width"]
        return {"bytes": rows * (2 * width + (held(width, "mxfp8") if case["form"] == "mxfp8" else 2 * width)), "flops": 3 * rows * width}
    if case["kind"] == "norm":
        width = case["width"]
        delta = 4 * case["parts"] if case["parts"] else 2
        return {"bytes": rows * ((8 + delta) * width + held(width, "mxfp8")) + 2 * width, "flops": rows * width * (8 + case["parts"])}
    n = 2 * case["ff"] if case["kind"] == "gate_up" else case["n"]
    out = rows * (held(case["ff"], "mxfp8") if case["kind"] == "gate_up" else 2 * n)
    return {"bytes": (rows * held(case["k"], case["form"]) + n * held(case["k"], "mxfp4") + out), "flops": 2 * rows * n * case["k"]}


# ---------------------------------------------------------------- in 64 bits


def _exact_blocks(x: torch.Tensor, form: str) -> tuple:
    """(elements, scales) as the numbers that they are, float64 [rows, blocks, 32] and [rows, blocks], by search over powers of two
    and over the type's own numbers."""
    rows, width = x.shape
    x = torch.cat([x, x.new_zeros(rows, -width % BLOCK)], 1).reshape(rows, -1, BLOCK)
    most = x.abs().max(-1).values / LARGEST[form]
    power = torch.where(most > 0, torch.log2(most), torch.full_like(most, -127.0)).ceil()
    power = torch.where(torch.exp2(power - 1) >= most, power - 1, power)
    power = torch.where(torch.exp2(power) < most, power + 1, power).clamp(min=-127)
    scale = torch.exp2(power)
    if form == "mxfp8":
        grid = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    else:
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    a = x / scale.unsqueeze(-1)
    high = torch.searchsorted(grid, a.abs().contiguous()).clamp(max=grid.numel() - 1)
    low = (high - 1).clamp(min=0)
    to_low, to_high = a.abs() - grid[low], grid[high] - a.abs()
    at = torch.where((to_low < to_high) | ((to_low == to_high) & (low % 2 == 0)), low, high)
    return torch.copysign(grid[at], a), scale


def _exact_values(codes: torch.Tensor, scales: torch.Tensor, width: int, form: str) -> torch.Tensor:
    c = codes.long()
    e, m, bias = ((c >> 3) & 15, c & 7, 7) if form == "mxfp8" else ((c >> 1) & 3, c & 1, 1)
    steps = 8 if form == "mxfp8" else 2
    a = torch.where(e > 0, (1 + m / steps) * torch.exp2((e - bias).double()), m.double() / steps * 2.0 ** (1 - bias))
    a = torch.where((c >> (7 if form == "mxfp8" else 3)) & 1 > 0, -a, a)
    return (a * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, 1))[:, :width]


def exact(case: dict, seed: int):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    flat = lambda blocks, width: [blocks[0].flatten(1)[:, :width].contiguous(), blocks[1]]
    if case["kind"] == "quantise":
        width = case["width"]
        elements, scales = _exact_blocks(state["x"].double(), case["form"])
        if case["form"] == "mxfp8":
            return flat((elements, scales), width)
        return [(elements * scales.unsqueeze(-1)).flatten(1)[:, :width].contiguous()]
    if case["kind"] == "norm":
        h = state["residual"].double() + (state["delta"].double().sum(0) if case["parts"] else state["delta"].double())
        y = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * state["weight"].double()
        return [h, *flat(_exact_blocks(y, "mxfp8"), case["width"])]
    x = _exact_values(*state["x"], case["k"], case["form"])
    w = _exact_values(*state["w"], case["k"], "mxfp4")
    if case["kind"] == "product":
        return [x @ w.T]
    y = x @ w.T
    z = y[:, :case["ff"]]
    return flat(_exact_blocks(z * torch.sigmoid(z) * y[:, case["ff"]:], "mxfp8"), case["ff"])
