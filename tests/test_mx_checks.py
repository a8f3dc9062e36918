"""What the microscaled entry points check of rows and weights that were taken apart and put together again, and of the choices a caller makes."""
import pytest
import torch
from torch.utils import _pytree as pytree

import plain_mx as plain
from arle_amd.kernels import mx, ops
from test_mx import _rows, no_gpu  # noqa: F401  (a fixture)


def test_exchanged_fields_reach_no_kernel(no_gpu):
    """A tuple with an exchanged field is one that nothing has checked: products, values and weights refuse it."""
    rows, w = _rows(3, 300)[2], mx.lay_weight(_rows(40, 300, "mxfp4")[2])
    wg, four = mx.lay_weight(_rows(40, 300, "mxfp4")[2], gated=True), _rows(32, 300, "mxfp4")[2]
    bad_rows = [rows._replace(rows=300), rows._replace(elements=rows.elements[:1]), rows._replace(scales=rows.scales[:, :1]), mx.MXRows._make(rows)]
    bad_weights = [w._replace(n=4000), w._replace(tiles=w.tiles[:, :1]), w._replace(pitch=1), mx.MXWeight._make(w)]
    calls = [lambda x=x: mx.gemm(x, w) for x in bad_rows] + [lambda x=x: mx.values(x) for x in bad_rows]
    calls += [lambda x=x: mx.gate_up_act(x, wg) for x in bad_rows] + [lambda v=v: mx.gemm(rows, v) for v in bad_weights]
    calls += [lambda: mx.gate_up_act(rows, wg._replace(n=4000)), lambda: mx.lay_weight(four._replace(rows=300))]
    for i, call in enumerate(calls):
        with pytest.raises(ops.ShapeError):
            call()
            pytest.fail(f"call {i} passed")


def test_rows_and_weights_are_put_together_from_their_fields(no_gpu):
    """As a program that maps a function over the tensors of a structure does; fields that do not fit the tensors are refused."""
    rows, w = _rows(3, 600)[2], mx.lay_weight(_rows(34, 600, "mxfp4")[2], gated=True)
    for held in (rows, w):
        again = pytree.tree_map_only(torch.Tensor, torch.clone, held)
        assert type(again) is type(held) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(held[:2], again[:2]))
        assert again[2:] == held[2:] and again[0].data_ptr() != held[0].data_ptr()
    for make in (lambda: mx.MXRows(*rows[:4], 4, *rows[5:]), lambda: mx.MXRows(*rows[:6], 4, rows[7]), lambda: mx.MXRows(*rows[:4], 3),
                 lambda: mx.MXWeight(*w[:8], 1), lambda: mx.MXWeight(*w[:5], 7, *w[6:])):
        with pytest.raises(ops.ShapeError):
            make()
    assert all(torch.equal(a, b) for a, b in zip(plain.unpack(rows), plain.unpack(mx.MXRows(*rows))))


def test_blocks_are_measured_before_a_kernel_fills_them(no_gpu):
    """Attention writes [T, padded] elements and [T, padded / 32] scales: tensors that are smaller than the fields beside them are refused."""
    like = torch.zeros(3, 4)
    for form in ("mxfp8", "mxfp4"):
        rows = mx.empty_rows(3, 600, form)._replace(device=-1)      # the device number of a tensor on the host
        small, other = mx.empty_rows(3, 512, form), mx.empty_rows(3, 600, "mxfp4" if form == "mxfp8" else "mxfp8")
        ops._need_blocks(rows, 3, 600, like)
        off = torch.empty(3 * rows.elements.shape[1] + 8, dtype=torch.uint8)[8:].view(3, -1).view(rows.elements.dtype)
        for bad in (rows._replace(elements=small.elements), rows._replace(scales=small.scales), rows._replace(elements=rows.elements[:2]),
                    rows._replace(elements=other.elements), rows._replace(bits=other.bits), rows._replace(form=other.form), rows._replace(padded=512),
                    rows._replace(scales=rows.scales[:1]), rows._replace(elements=off), rows._replace(scales=rows.scales.view(torch.uint8).to(torch.int16)),
                    rows[:3], None):
            with pytest.raises(ops.ShapeError):
                ops._need_blocks(bad, 3, 600, like)


def test_parts_of_k_go_with_a_variant(no_gpu):
    """A number of parts that nothing would follow is refused, and so is none."""
    x, w = _rows(3, 1200)[2], mx.lay_weight(_rows(40, 1200, "mxfp4")[2])
    for args in (dict(splits=2), dict(splits=1), dict(splits=4, partials_ok=True), dict(variant=3, splits=0), dict(variant=0, splits=0), dict(variant=0, splits=-1)):
        with pytest.raises(ops.ShapeError):
            mx.gemm(x, w, **args)
    with pytest.raises(AssertionError, match="launched"):
        mx.gemm(x, w, variant=3, splits=3)
