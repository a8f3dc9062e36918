"""Registers that spill to memory, and memory that a lane has of its own, in the microscaled kernels: none."""
import pytest

from arle_amd.kernels import build
from test_kernel_registers import _code_objects, _kernels


@pytest.mark.parametrize("library", ["mx_rows", "mx_gemm"])
def test_the_microscaled_kernels_stay_in_their_registers(library):
    with open(build.ensure(library), "rb") as fh:
        data = fh.read()
    found = {}
    for elf in _code_objects(data):
        found.update(_kernels(elf))
    assert len(found) > 20
    spilt = {name: k[".vgpr_spill_count"] for name, k in found.items() if k[".vgpr_spill_count"] or k[".private_segment_fixed_size"]}
    assert not spilt
