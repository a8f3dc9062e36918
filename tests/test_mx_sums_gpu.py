"""How wide the sums of microscaled products are: rows in 4 bits lose nothing but the steps of 32 bits, rows in 8 bits up to 7 * 2^-13 of the largest
product of every eight neighbouring k."""
import pytest
import torch

import plain_mx as plain
from arle_amd.kernels import mx
from test_mx_gpu import VARIANT_ROWS, _operands

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("form", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("N,K", [(40, 256), (131, 700)])
@pytest.mark.parametrize("variant", sorted(VARIANT_ROWS))
def test_what_an_eight_loses(form, variant, N, K):
    M = VARIANT_ROWS[variant][1]
    x, w, xv, wv = _operands(M, N, K, form, M + N)
    rows, weight = mx.rows_from_codes(*(t.to(DEV) for t in x), K, form), mx.lay_weight(mx.rows_from_codes(*(t.to(DEV) for t in w), K, "mxfp4"))
    got = mx.gemm(rows, weight, torch.float32, variant=variant).cpu().double()
    products = torch.nn.functional.pad(xv[:, None] * wv[None], (0, -K % 8)).view(M, N, -1, 8)
    # eights that are added one behind the other: half a step of 32 bits each, of no more than all magnitudes; and a few sums of waves' parts
    steps = (products.shape[2] + 16) * 2.0**-24 * products.abs().sum((2, 3))
    lost = 7 * 2.0**-13 * products.abs().amax(3).sum(2) if form == "mxfp8" else 0.0
    assert ((got - products.sum((2, 3))).abs() <= lost + steps).all()


@pytest.mark.parametrize("variant", sorted(VARIANT_ROWS))
def test_a_large_product_hides_its_seven_neighbours_and_no_other(variant):
    """2^-4 and 2^-9 beside 2^4 in an eight lose nothing (2^-8 and 2^-13 of it), 2^-9 beside 2^6 may be lost; in the eight behind nothing ever is."""
    M, K = VARIANT_ROWS[variant][1], 64
    e = torch.zeros(M, K, dtype=torch.uint8)
    s = torch.full((M, 2), 127, dtype=torch.uint8)
    e[:, 0] = 0x58                            # e4m3: 2^4
    e[:, 1:8] = 0x18                          # 2^-4, 2^-8 of it
    e[:, 8:16] = 0x01                         # 2^-9
    w = torch.zeros(48, K)
    w[:, :16] = 1.0
    weight = mx.lay_weight(mx.quantize(w.to(DEV), "mxfp4"))
    got = mx.gemm(mx.rows_from_codes(e.to(DEV), s.to(DEV), K, "mxfp8"), weight, torch.float32, variant=variant).cpu()
    assert torch.equal(got, torch.full_like(got, 16.0 + 7 / 16 + 8 / 512))
    e[:, 1:8] = 0x01                          # 2^-9 beside 2^4: at the instruction's last bit
    got = mx.gemm(mx.rows_from_codes(e.to(DEV), s.to(DEV), K, "mxfp8"), weight, torch.float32, variant=variant).cpu()
    assert torch.equal(got, torch.full_like(got, 16.0 + 7 / 512 + 8 / 512))
    e[:, 0] = 0x68                            # 2^6: its neighbours are under 2^-13 of it, the next eight is whole
    got = mx.gemm(mx.rows_from_codes(e.to(DEV), s.to(DEV), K, "mxfp8"), weight, torch.float32, variant=variant).cpu()
    assert ((got >= 64.0 + 8 / 512) & (got <= 64.0 + 15 / 512)).all()


@pytest.mark.parametrize("form,most", [("mxfp8", 5.2e15), ("mxfp4", 10.5e15)])
def test_the_ceiling_of_scaled_products_is_plausible(form, most):
    """Above half of what the products behind it reach, under the published peak and a bit."""
    from arle_amd.kernels import ceilings

    for random_operands in (True, False):
        rate = ceilings.mfma_scaled_rate(DEV, form=form, iters=2000, repeats=2, random_operands=random_operands)
        assert 1e15 < rate < most
