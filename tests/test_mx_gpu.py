"""The microscaled kernels against plain forms in 64 bits."""
import pytest
import torch

import plain_mx as plain
from arle_amd.kernels import mx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FORMS = ["mxfp8", "mxfp4"]


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _same(a, b):
    return all(torch.equal(p, q) for p, q in zip(plain.unpack(a), plain.unpack(b)))


def _wild(T, W, seed):
    """Rows whose blocks span the type's range: zeros, tiny and huge ones, ties, a maximum right at a border of two scales."""
    x = torch.randn(T, W, generator=_g(seed)) * torch.exp2(torch.randint(-100, 100, (T, W), generator=_g(seed + 1)).float() * (torch.rand(T, 1, generator=_g(seed + 2)) < 0.3))
    x[:, ::7] = 0
    if W >= 64:
        x[0, :32] = 0
        x[-1, 32:64] = torch.tensor([1.75, 1.5] * 16) * torch.exp2(torch.arange(32).float() - 16)
        x[0, 32:64] = torch.tensor([448.0, 6.0, 2.5, 5.0, 0.25, -0.25, 3.5, -1.25] * 4)      # ties of e2m1 at a scale of 1 under 6
        if T > 2:
            x[1, :32] = torch.tensor([6.0, 2.5, 5.0, 0.25, -0.25, 3.5, -1.25, 0.75] * 4)
            x[1, 32:64] = 2.0**-140 * torch.arange(32)
    return x


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,W", [(1, 1), (1, 31), (3, 32), (5, 33), (4, 255), (8, 256), (7, 264), (2, 1530), (1030, 72), (3, 4104), (1, 9000)])
def test_quantize_is_the_definition(form, dtype, T, W):
    x = _wild(T, W, T + W).to(dtype)
    rows = mx.quantize(x.to(DEV), form)
    e, s = plain.unpack(rows)
    want_e, want_s = plain.quantize(x.double(), form)
    assert torch.equal(s[:, :want_s.shape[1]], want_s) and not s[:, want_s.shape[1]:].any()
    assert torch.equal(plain.element_values(e[:, :W], form), plain.element_values(want_e, form)) and not e[:, W:].any()
    want = plain.dequantize(want_e, want_s, form)
    assert torch.equal(mx.values(rows).cpu().double(), want)
    big = want.abs() >= 2.0**-126          # bfloat16 holds these numbers as they are
    assert torch.equal(mx.values(rows, torch.bfloat16).cpu().double()[big], want[big])
    # no number is off by more than half a step of its element, or half of the smallest step
    half = {"mxfp8": 2.0**-4, "mxfp4": 2.0**-2}[form]
    scale = plain.scale_values(want_s).repeat_interleave(32, 1)[:, :W]
    least = {"mxfp8": 2.0**-10, "mxfp4": 2.0**-2}[form]
    assert ((want - x.double()).abs() <= torch.maximum(half * x.double().abs(), least * scale)).all()


@pytest.mark.parametrize("form", FORMS)
def test_quantize_of_views(form):
    """Rows apart, columns of a wider buffer, starts off any alignment."""
    buf = torch.randn(9, 700, generator=_g(1)).bfloat16().to(DEV)
    for view in (buf[:, :256], buf[:, 8:264], buf[:, 3:260], buf[::2, 5:6], buf[1:4, 13:], buf[:, 4:260]):
        got, want = mx.quantize(view, form), mx.quantize(view.contiguous(), form)
        assert _same(got, want)


@pytest.mark.parametrize("form", FORMS)
def test_not_a_number_stays_in_its_block(form):
    x = torch.randn(4, 128, generator=_g(2))
    x[0, 5], x[1, 40], x[2, 127] = float("nan"), float("inf"), -float("inf")
    rows = mx.quantize(x.to(DEV), form)
    v = mx.values(rows).cpu()
    bad = torch.zeros(4, 128, dtype=torch.bool)
    bad[0, :32] = bad[1, 32:64] = bad[2, 96:] = True
    assert torch.equal(v.isnan(), bad)
    w = mx.lay_weight(mx.quantize(torch.randn(40, 128, generator=_g(3)).to(DEV), "mxfp4"))
    for variant in sorted(VARIANT_ROWS):
        y = mx.gemm(rows, w, torch.float32, variant=variant).cpu()
        assert y[:3].isnan().all() and y[3].isfinite().all()


def _delta(kind, T, W, seed):
    if kind == "none":
        return None
    if kind == "bf16":
        return (torch.randn(T, W, generator=_g(seed)) * 0.3).bfloat16()
    return torch.randn(kind, T, W, generator=_g(seed)) * 0.3


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["none", "bf16", 1, 2, 4, 5, 9])
@pytest.mark.parametrize("T,W", [(1, 1), (2, 30), (3, 255), (5, 1028), (2, 1530), (3, 2560), (2, 4100), (1, 8196), (2, 16384)])
def test_add_rmsnorm(form, kind, T, W):
    eps = 1e-6
    res = torch.randn(T, W, generator=_g(T)) * 2
    res[-1] *= 1e-5        # eps counts
    weight = 1 + 0.1 * torch.randn(W, generator=_g(5))
    weight = weight.bfloat16() if W % 3 else weight
    delta = _delta(kind, T, W, 6)
    h, y = plain.norm(res, delta, weight, eps)
    r = res.to(DEV)
    rows = mx.add_rmsnorm(r, None if delta is None else delta.to(DEV), weight.to(DEV), eps, form)
    # a sum of parts + 1 numbers of 32 bits: at most a half step a addition of the largest partial sum
    parts = 0 if delta is None else delta.shape[0] if delta.dim() == 3 else 1
    size = res.double().abs() + (0 if delta is None else delta.double().abs().sum(0) if delta.dim() == 3 else delta.double().abs())
    assert ((r.cpu().double() - h).abs() <= parts * 2.0**-24 * size).all()
    e, s = plain.unpack(rows)
    assert not e[:, W:].any() and not s[:, -(-W // 32):].any()
    got = plain.dequantize(e[:, :W], s[:, :-(-W // 32)], form)
    # half a step of the element, or of the smallest one, and the 32-bit arithmetic: the sums of squares are added in a tree of at
    # most 16 + 10 levels, root, quotient and two products, which is less than 2^-18 of the number
    half, least = {"mxfp8": (2.0**-4, 2.0**-10), "mxfp4": (2.0**-2, 2.0**-2)}[form]
    scale = plain.scale_values(s).repeat_interleave(32, 1)[:, :W]
    slack = 2.0**-18 * y.abs() + parts * 2.0**-23 * size * (y.abs() / h.abs().clamp_min(1e-300))
    assert ((got - y).abs() <= torch.maximum(half * y.abs(), least * scale) * (1 + 2.0**-10) + slack).all()
    # and the scale is the smallest: twice the block's largest number is past the element's largest
    most = torch.nn.functional.pad(y.abs(), (0, -W % 32)).view(T, -1, 32).amax(-1)
    sc = plain.scale_values(s[:, :most.shape[1]])
    largest = plain.GRID[form][-1]
    assert (most <= largest * sc * (1 + 2.0**-18)).all() and ((2 * most >= largest * sc * (1 - 2.0**-18)) | (s[:, :most.shape[1]] == 0)).all()


def test_add_rmsnorm_of_picked_rows():
    """Rows by index, the same one twice; the residual stays as it was."""
    res = torch.randn(6, 300, generator=_g(1)).to(DEV)
    delta = torch.randn(3, 6, 300, generator=_g(2)).to(DEV)
    w = torch.ones(300, device=DEV)
    pick = torch.tensor([5, 0, 0, 3], dtype=torch.int32, device=DEV)
    before = res.clone()
    got = mx.add_rmsnorm(res, delta, w, 1e-6, "mxfp8", rows=pick)
    assert torch.equal(res, before)
    whole = mx.add_rmsnorm(res, delta, w, 1e-6, "mxfp8")
    assert all(torch.equal(a, b[pick.long().cpu()]) for a, b in zip(plain.unpack(got), plain.unpack(whole)))


# What a sum may be off by.  With an e4m3 operand the instruction aligns the products of 8 neighbouring k to the largest of them and drops what
# is under 2^-13 of that one's power of two (measured with two products, 1 and 1.875 * 2^-d: at d = 11, 12, 13 what came back of the second was
# 0.933, 0.8 and 0.533, its bits down to 2^-13, at 14 nothing; products in different eights, and the eights' sums, met in 32 bits): up to seven
# products are cut by up to 2^-13 of the largest each, so an eight by less than 7 * 2^-13 of the sum of its magnitudes.  Products of e2m1 with e2m1 differ by
# less than 2^8 and lose nothing.  Then half a step of 32 bits for every addition behind.
def _sum_error(form, K):
    return {"mxfp8": 7 * 2.0**-13, "mxfp4": 2.0**-22}[form] + (K / 8 + 16) * 2.0**-24


def _operands(M, N, K, form, seed, spread=8):
    """Codes over their whole range but NaN, scales over 2^spread."""
    top = 16 if form == "mxfp4" else 127
    xe = torch.randint(0, top, (M, K), generator=_g(seed), dtype=torch.uint8)
    if form == "mxfp8":
        xe |= torch.randint(0, 2, (M, K), generator=_g(seed + 1), dtype=torch.uint8) << 7
    xs = torch.randint(127 - spread // 2, 128 + spread // 2, (M, -(-K // 32)), generator=_g(seed + 2), dtype=torch.uint8)
    we = torch.randint(0, 16, (N, K), generator=_g(seed + 3), dtype=torch.uint8)
    ws = torch.randint(127 - spread // 2, 128 + spread // 2, (N, -(-K // 32)), generator=_g(seed + 4), dtype=torch.uint8)
    return (xe, xs), (we, ws), plain.dequantize(xe, xs, form), plain.dequantize(we, ws, "mxfp4")


VARIANT_ROWS = {0: (1, 9, 16), 1: (1, 8, 16), 2: (3, 33, 70), 3: (1, 64, 130), 4: (1, 127, 300), 5: (5, 128, 200), 6: (2, 255, 520), 7: (1, 128, 300), 8: (3, 250, 520)}
GATED = (3, 4, 5, 6)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("N,K", [(1, 1), (15, 33), (16, 128), (40, 256), (131, 700), (264, 1290), (600, 2610)])
@pytest.mark.parametrize("variant", sorted(VARIANT_ROWS))
def test_gemm(form, variant, N, K):
    for M in VARIANT_ROWS[variant]:
        x, w, xv, wv = _operands(M, N, K, form, M + N)
        rows, weight = mx.rows_from_codes(*(t.to(DEV) for t in x), K, form), mx.lay_weight(mx.rows_from_codes(*(t.to(DEV) for t in w), K, "mxfp4"))
        want, size = xv @ wv.T, xv.abs() @ wv.abs().T
        off = _sum_error(form, K) * size
        got = mx.gemm(rows, weight, torch.float32, variant=variant).cpu().double()
        assert ((got - want).abs() <= off).all(), (M, N, K)
        got16 = mx.gemm(rows, weight, torch.bfloat16, variant=variant).cpu().double()
        assert ((got16 - want).abs() <= off + 2.0**-8 * (want.abs() + off)).all(), (M, N, K)
        steps = rows.padded // (128 if variant in mx.ROW_VARIANTS else 512)
        for splits in (2, 3):
            if (splits - 1) * -(-steps // splits) < steps:
                parts = mx.gemm(rows, weight, torch.float32, partials_ok=True, variant=variant, splits=splits)
                assert parts.shape == (splits, M, N)
                assert ((parts.cpu().double().sum(0) - want).abs() <= off).all(), (M, N, K, splits)
                whole = mx.gemm(rows, weight, torch.bfloat16, variant=variant, splits=splits).cpu().double()
                assert ((whole - want).abs() <= off + 2.0**-8 * (want.abs() + off)).all(), (M, N, K, splits)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("N,K", [(15, 33), (40, 300), (131, 1290), (600, 520)])
@pytest.mark.parametrize("variant", sorted(VARIANT_ROWS))
def test_gemm_of_whole_numbers_is_exact(form, variant, N, K):
    """Numbers up to 3 times numbers up to 6, scales from 1/4 to 4: multiples of 1/32, sums under 2^19, so no bit may be lost."""
    for M in VARIANT_ROWS[variant][1:]:
        few = torch.tensor([0, 2, 4, 5, 8, 10, 12, 13] if form == "mxfp4" else [0, 0x38, 0x40, 0x44, 0x80, 0xB8, 0xC0, 0xC4], dtype=torch.uint8)
        xe = few[torch.randint(0, 8, (M, K), generator=_g(M))]
        we = torch.randint(0, 16, (N, K), generator=_g(N), dtype=torch.uint8)
        xs, ws = (torch.randint(125, 130, (rows, -(-K // 32)), generator=_g(rows + 1), dtype=torch.uint8) for rows in (M, N))
        got = mx.gemm(mx.rows_from_codes(xe.to(DEV), xs.to(DEV), K, form), mx.lay_weight(mx.rows_from_codes(we.to(DEV), ws.to(DEV), K, "mxfp4")),
                      torch.float32, variant=variant)
        assert torch.equal(got.cpu().double(), plain.dequantize(xe, xs, form) @ plain.dequantize(we, ws, "mxfp4").T), (M, N, K)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("out", FORMS)
@pytest.mark.parametrize("ff,K", [(1, 40), (32, 256), (100, 300), (256, 130), (300, 1100)])
@pytest.mark.parametrize("variant", GATED)
def test_gate_up_act(form, out, variant, ff, K):
    for M in VARIANT_ROWS[variant][1:]:
        x, w, xv, wv = _operands(M, 2 * ff, K, form, M + ff, spread=4)
        xs = x[1] - (12 if form == "mxfp8" else 4)      # gates of a size where the activation is neither 0 nor the identity
        xv = plain.dequantize(x[0], xs, form)
        rows = mx.rows_from_codes(x[0].to(DEV), xs.to(DEV), K, form)
        weight = mx.lay_weight(mx.rows_from_codes(*(t.to(DEV) for t in w), K, "mxfp4"), gated=True)
        got = mx.gate_up_act(rows, weight, out, variant=variant)
        e, s = plain.unpack(got)
        assert not e[:, ff:].any() and not s[:, -(-ff // 32):].any()
        want = plain.gated(xv, wv)
        gate, up = (xv @ wv.T).chunk(2, dim=1)
        gate_off, up_off = (_sum_error(form, K) * (xv.abs() @ wv.abs().T)).chunk(2, dim=1)
        # |silu'| <= 1.1; the 32-bit arithmetic of exponential, quotient and product stays under 2^-20 (for gates under -80 under 2^-100)
        slack = 1.1 * gate_off * (up.abs() + up_off) + (gate.abs() + gate_off) * up_off + 2.0**-20 * want.abs() + 2.0**-100
        half, least = {"mxfp8": (2.0**-4, 2.0**-10), "mxfp4": (2.0**-2, 2.0**-2)}[out]
        scale = plain.scale_values(s).repeat_interleave(32, 1)[:, :ff]
        v = plain.dequantize(e[:, :ff], s[:, :-(-ff // 32)], out)
        assert ((v - want).abs() <= torch.maximum(half * (want.abs() + slack), least * scale) + slack).all(), (M, ff, K)
        most = torch.nn.functional.pad(want.abs(), (0, -ff % 32)).view(M, -1, 32).amax(-1)
        slack_most = torch.nn.functional.pad(slack, (0, -ff % 32)).view(M, -1, 32).amax(-1)
        sc, largest = plain.scale_values(s[:, :most.shape[1]]), plain.GRID[out][-1]
        assert (most <= largest * sc + slack_most).all() and ((2 * (most + slack_most) >= largest * sc) | (s[:, :most.shape[1]] == 0)).all()


def test_strided_rows_and_slices():
    """A slice of rows, and rows apart in a wider buffer."""
    x = mx.quantize(torch.randn(40, 512, generator=_g(1)).to(DEV))
    w = mx.lay_weight(mx.quantize(torch.randn(70, 512, generator=_g(2)).to(DEV), "mxfp4"))
    whole = mx.gemm(x, w, torch.float32, variant=2)
    assert torch.equal(mx.gemm(x.part(7, 29), w, torch.float32, variant=2), whole[7:29])
    wide_e, wide_s = torch.zeros(40, 1024, dtype=torch.uint8, device=DEV), torch.zeros(40, 64, dtype=torch.uint8, device=DEV)
    wide_e[:, 256:768], wide_s[:, 16:32] = x.elements.view(torch.uint8), x.scales.view(torch.uint8)
    apart = mx.MXRows(wide_e[:, 256:768].view(torch.float8_e4m3fn), wide_s[:, 16:32].view(torch.float8_e8m0fnu), 512, "mxfp8")
    assert torch.equal(mx.gemm(apart, w, torch.float32, variant=2), whole)
    assert torch.equal(mx.values(apart), mx.values(x))


@pytest.mark.parametrize("variant", sorted(VARIANT_ROWS))
@pytest.mark.parametrize("K", [200, 1100])
def test_the_first_rows_of_a_weight(variant, K):
    """Tiles of a larger weight: a step's tiles lie further apart than there are."""
    x = mx.quantize(torch.randn(13, K, generator=_g(1)).to(DEV))
    w = mx.lay_weight(mx.quantize(torch.randn(600, K, generator=_g(2)).to(DEV), "mxfp4"))
    whole = mx.gemm(x, w, torch.float32, variant=variant)
    for n in (16, 48, 400):
        assert torch.equal(mx.gemm(x, w.first(n), torch.float32, variant=variant), whole[:, :n])


def test_every_kernel_of_few_or_many_rows_gives_the_same_row_whatever_stands_beside_it():
    x = mx.quantize(torch.randn(300, 700, generator=_g(1)).to(DEV))
    w = mx.lay_weight(mx.quantize(torch.randn(90, 700, generator=_g(2)).to(DEV), "mxfp4"))
    for variant, rows in ((0, 16), (1, 16), (2, 64), (3, 300), (4, 300), (5, 300), (6, 300), (7, 300), (8, 300)):
        whole = mx.gemm(x.part(0, rows), w, torch.float32, variant=variant)
        assert torch.equal(mx.gemm(x.part(rows - 1, rows), w, torch.float32, variant=variant)[0], whole[-1])


@pytest.mark.parametrize("M,N,K", [(1, 2560, 4096), (8, 48, 9728), (16, 6144, 2560), (17, 2560, 2560), (40, 6144, 2610), (100, 1531, 2610), (600, 2560, 4096)])
@pytest.mark.parametrize("form", FORMS)
def test_chosen_variants(form, M, N, K):
    """Whatever the sizes choose: whole sums, a stack where it may be one, and the two alike."""
    x, w, xv, wv = _operands(M, N, K, form, M)
    rows, weight = mx.rows_from_codes(*(t.to(DEV) for t in x), K, form), mx.lay_weight(mx.rows_from_codes(*(t.to(DEV) for t in w), K, "mxfp4"))
    want, off = xv @ wv.T, _sum_error(form, K) * (xv.abs() @ wv.abs().T)
    got = mx.gemm(rows, weight).cpu().double()
    assert ((got - want).abs() <= off + 2.0**-8 * (want.abs() + off)).all()
    stack = mx.gemm(rows, weight, torch.float32, partials_ok=True)
    total = stack.cpu().double().sum(0) if stack.dim() == 3 else stack.cpu().double()
    assert ((total - want).abs() <= off).all()
