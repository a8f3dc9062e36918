"""More rows than one launch has threads for."""
import pytest
import torch

import plain_mx as plain
from arle_amd.kernels import mx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _column(rows):
    return (torch.arange(rows, dtype=torch.int32, device=DEV) % 7 - 3).float().view(rows, 1)


@pytest.mark.parametrize("picked", [False, True])
def test_norms_of_more_than_2_to_the_24_rows(picked):
    """A workgroup of 256 a row: 2^24 of them are 2^32 threads.  Rows of one number: itself by its magnitude, the sign but for zeros."""
    T = 2**24 + 5
    residual = _column(T)
    delta = torch.ones(T, 1, device=DEV)
    h = residual + delta
    pick = torch.arange(T - 1, -1, -1, dtype=torch.int32, device=DEV) if picked else None
    rows = mx.add_rmsnorm(residual, delta, torch.ones(1, device=DEV), 1e-12, "mxfp4", rows=pick)
    assert torch.equal(residual, _column(T) if picked else h)
    got = mx.values(rows)
    assert torch.equal(got, (h.flip(0) if picked else h).sign())


def test_quantisation_and_values_of_more_than_2_to_the_27_rows():
    """Workgroups of 64, two rows each: 2^27 rows are 2^32 threads, for values 2^26."""
    T = 2**27 + 10
    x = _column(T).bfloat16()
    q = mx.quantize(x, "mxfp4")
    assert torch.equal(mx.values(q, torch.bfloat16), x)
    last = q.part(T - 3, T)
    assert all(torch.equal(a, b) for a, b in zip(plain.unpack(last), plain.unpack(mx.quantize(x[-3:], "mxfp4"))))
