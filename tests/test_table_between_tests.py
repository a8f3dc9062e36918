"""A test that takes measured products in leaves the table of the tests behind it alone."""
import pytest

from arle_amd.kernels import ops

WIDTHS = (1000, 1096, False, True)


@pytest.mark.parametrize("turn", [0, 1])
def test_a_table_ends_with_its_test(turn):
    assert WIDTHS not in ops._PRODUCT_TABLE and ops._PRODUCT_TABLE, turn
    ops.load_product_table({"1000,1096,0,1": [[16, "rows", [2], 2]]})
    assert ops.choose_product(9, 1000, 1096, 1096, tiled=True, fused=False, partials_ok=True) == ops.ProductChoice("rows", (2,), 2)
    del ops._PRODUCT_TABLE[next(iter(ops._PRODUCT_TABLE))]
