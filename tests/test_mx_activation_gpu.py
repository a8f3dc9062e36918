"""silu(gate) * up of the gated product to the last bits of 32: sums that are exact, results beside the borders between two elements."""
import pytest
import torch

import plain_mx as plain
from arle_amd.kernels import mx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OFF = 2.0**-20      # of a result: t = -gate log2(e) with its rounding taken along, an exponential, a reciprocal, two sums and four products of 32 bits


def gated_operands(rows, ff, form, seed, coarse):
    """Codes and scales of x [rows, 128] and w [2 ff, 128].  A row's gates lie around coarse[row] (a multiple of four, made by its first block), their
    finer bits, and the ups, come from three blocks of one number in every eight: multiples of 2^-16 up to 100, which 32 bits hold."""
    g = torch.Generator().manual_seed(seed)
    code = {v: c for c, v in enumerate([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])}
    to_form = (lambda c: c) if form == "mxfp4" else (lambda c: torch.tensor([0, 0x30, 0x38, 0x3C, 0x40, 0x44, 0x48, 0x4C], dtype=torch.uint8)[(c & 7).long()] | (c & 8) << 4)
    xe, we = torch.zeros(rows, 128, dtype=torch.uint8), torch.zeros(2 * ff, 128, dtype=torch.uint8)
    xs, ws = torch.zeros(rows, 4, dtype=torch.uint8), torch.zeros(2 * ff, 4, dtype=torch.uint8)
    for r, c in enumerate(coarse):      # |c| / 8 as up to three of the type's numbers
        left = abs(c) / 8
        for k in (0, 8, 16):
            take = max(v for v in code if v <= left)
            xe[r, k] = code[take] | (8 if c < 0 else 0)
            left -= take
        assert left == 0
    xs[:, 0], ws[:, 0] = 127 + 3, 127
    we[:ff, 0:24:8] = code[1.0]
    xe[:, 32::8], we[:, 32::8] = (torch.randint(0, 16, (n, 12), generator=g, dtype=torch.uint8) for n in (rows, 2 * ff))
    for block, power in ((1, -5), (2, -9), (3, -14)):
        xs[:, block], ws[:, block] = 127 + power, 127
    return (to_form(xe), xs), (we, ws)


def borders(want, form="mxfp8", off=OFF):
    """The codes of what is `off` under and above `want`, and where their blocks have one scale."""
    lo, hi = plain.quantize(want * (1 - off), form), plain.quantize(want * (1 + off), form)
    return lo, hi, (lo[1] == hi[1]).repeat_interleave(32, 1)[:, :want.shape[1]]


COARSE = [-84, -80, -76, -72, -68, -64, -84, -80, -76, -72, -60, -48, -40, -24, -8, 4]


@pytest.mark.parametrize("form", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("variant", [mx.GATED_ROWS, 3, 4, 5, 6])
def test_activation_between_two_elements(variant, form):
    M, ff = (16, 65536) if variant == mx.GATED_ROWS else (128, 8192)
    x, w = gated_operands(M, ff, form, 5, [COARSE[r % len(COARSE)] for r in range(M)])
    y = plain.dequantize(*x, form) @ plain.dequantize(*w, "mxfp4").T
    assert torch.equal(y, y.float().double()) and y.abs().max() < 100
    want = plain.gated(plain.dequantize(*x, form), plain.dequantize(*w, "mxfp4"))
    rows, weight = mx.rows_from_codes(*(t.to(DEV) for t in x), 128, form), mx.lay_weight(mx.rows_from_codes(*(t.to(DEV) for t in w), 128, "mxfp4"), gated=True)
    e, s = plain.unpack(mx.gate_up_act(rows, weight, "mxfp8", variant=variant))
    lo, hi, one = borders(want)
    assert ((s == lo[1]) | (s == hi[1])).all() and one.float().mean() > 0.99
    values = lambda c: plain.element_values(c, "mxfp8")[one]
    low, high, got = values(lo[0]), values(hi[0]), values(e)
    assert ((got >= torch.minimum(low, high)) & (got <= torch.maximum(low, high))).all()


@pytest.mark.parametrize("variant", [mx.GATED_ROWS, 3])
def test_gates_whose_exponential_is_near_the_largest_float(variant):
    """Between -87.3 and -88.7 the results are the smallest that a block can hold, and no zeros; under -88.73, where exp(-gate) is past the floats,
    they are zeros, and what is large comes back whole."""
    x, w = gated_operands(16, 512, "mxfp4", 7, [-88] * 16)
    x[1][:, 1:] -= 1          # gates from -89.5 to -86.5
    y = plain.dequantize(*x, "mxfp4") @ plain.dequantize(*w, "mxfp4").T
    gate, up = y.chunk(2, dim=1)
    want = plain.gated(plain.dequantize(*x, "mxfp4"), plain.dequantize(*w, "mxfp4"))
    rows, weight = mx.rows_from_codes(*(t.to(DEV) for t in x), 128, "mxfp4"), mx.lay_weight(mx.rows_from_codes(*(t.to(DEV) for t in w), 128, "mxfp4"), gated=True)
    e, s = plain.unpack(mx.gate_up_act(rows, weight, "mxfp8", variant=variant))
    got = plain.dequantize(e, s, "mxfp8")
    near, past = (gate > -88.7) & (gate < -87.3), gate < -88.73
    assert near.sum() > 1000 and past.sum() > 100 and (got[past] == 0).all()
    # half a step of the element, or of the smallest one, behind the arithmetic of 32 bits, whose own smallest step is 2^-149
    least = 2.0**-10 * plain.scale_values(s).repeat_interleave(32, 1)
    assert ((got - want).abs() <= torch.maximum(2.0**-4 * want.abs(), least) * (1 + 2 * OFF) + OFF * want.abs() + 2.0**-148)[near].all()
    huge = torch.zeros(1, 32, device=DEV)
    huge[0, 0] = 2.0**120
    wide = torch.zeros(64, 32)
    wide[:, 0] = torch.tensor([1.0, 64.0])[torch.arange(64) % 2] * torch.where(torch.arange(64) < 32, 1.0, 2.0**-126)
    v = mx.values(mx.gate_up_act(mx.quantize(huge, "mxfp4"), mx.lay_weight(mx.quantize(wide.to(DEV), "mxfp4"), gated=True), variant=variant)).cpu()
    assert torch.equal(v[0], torch.tensor([2.0**114, 2.0**126])[torch.arange(32) % 2])


@pytest.mark.parametrize("variant", [mx.GATED_ROWS, 3])
def test_gates_that_are_far_below_zero(variant):
    """Exponentials past the floats give zeros, whatever is left of -gate behind t ln 2 in 32 bits: at these gates it is -1, by which an infinity would be
    multiplied as by zero."""
    gates = [85764464, 132280784, 178797104, 202055264, 434636864, 481153184, 527669504, 3 * 2**24, 2**29]
    blocks = 15
    xe, xs = torch.zeros(len(gates), 32 * blocks, dtype=torch.uint8), torch.zeros(len(gates), blocks, dtype=torch.uint8)
    for r, gate in enumerate(gates):
        for b in range(blocks):                       # a digit to the base four a block
            xe[r, 32 * b], xs[r, b] = (0, 10, 12, 13)[gate >> 2 * b & 3], 127 + 2 * b
    w = torch.zeros(128, 32 * blocks)
    w[:, ::32] = 1.0
    w[64:, ::32] = 2.0**-10
    rows = mx.rows_from_codes(xe.to(DEV), xs.to(DEV), 32 * blocks, "mxfp4")
    plainly = mx.gemm(rows, mx.lay_weight(mx.quantize(w.to(DEV), "mxfp4")), torch.float32)
    assert torch.equal(plainly[:, 0].cpu(), -torch.tensor(gates).float())
    v = mx.values(mx.gate_up_act(rows, mx.lay_weight(mx.quantize(w.to(DEV), "mxfp4"), gated=True), variant=variant))
    assert (v == 0).all()
