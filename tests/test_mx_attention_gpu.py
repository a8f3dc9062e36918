"""Attention whose results may leave in blocks: which kernel takes them is the launcher's answer, whatever it was told to run."""
import pytest
import torch

import plain_mx as plain
from arle_amd.kernels import lib, mx, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _portion(T, nq, nkv, P, D=128):
    g = torch.Generator().manual_seed(T + P)
    pages = -(-T // P)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    q = torch.randn(T, nq * D, generator=g).bfloat16().to(DEV)
    k, v = (torch.randn(pages, nkv, *shape, generator=g).bfloat16().to(DEV) for shape in ((P, D), (D, P)))

    def run(**kw):
        out = torch.zeros(T, nq * D, dtype=torch.bfloat16, device=DEV)
        return ops.attn_paged_mfma(q, out, k, v, i32([list(range(pages))]), i32([0, T]), i32([0]), i32([0]), max_qlen=T, min_qlen=T, max_kv_len=T,
                                   num_q_heads=nq, num_kv_heads=nkv, head_dim=D, page_size=P, scale=D**-0.5, portion_splits=1, **kw)
    return run


@pytest.mark.parametrize("form", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("P", [4, 16])      # the kernel that leaves blocks takes pages of eight slots and more
@pytest.mark.parametrize("variant", [0, 1, -1])
def test_blocks_whichever_kernel_runs(variant, P, form):
    run = _portion(200, 8, 2, P)
    lib.function("arle_attn_prefill_variant")(variant)
    try:
        want, blocks = run(), mx.empty_rows(200, 8 * 128, form)
        got = run(blocks=blocks)
    finally:
        lib.function("arle_attn_prefill_variant")(-1)
    assert (got is blocks) == (variant != 0 and P == 16)
    if got is not blocks:
        assert torch.equal(got, want)
        got = mx.quantize(got, form)
    assert all(torch.equal(a, b) for a, b in zip(plain.unpack(got), plain.unpack(mx.quantize(want, form))))
