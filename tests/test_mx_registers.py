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


def test_portions_that_leave_rows_are_not_charged_for_blocks():
    """The portions kernel of head_dim 128 keeps as many scalars in registers as it did before its results could leave in blocks, an ending of
    its own: with all endings behind a branch it had 13 to 16 more in memory (56 to 66 of them)."""
    with open(build.ensure("attention_mfma"), "rb") as fh:
        data = fh.read()
    notes = {}
    for elf in _code_objects(data):
        notes.update((n, k) for n, k in _kernels(elf).items() if "attn_prefill_dma_kernel" in n)
    assert len(notes) == 6 + 8      # whole tiles or not, one group or two or one beside decoded tokens; the first four in blocks of 8 and of 4 bits
    for n, k in notes.items():
        assert k[".vgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0 and k[".sgpr_spill_count"] <= 52, n
