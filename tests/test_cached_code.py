"""Properties of the cached attention's machine code that no result shows, read from the built
library."""
import os

import pytest

import code_objects

vh = pytest.importorskip("vestra_hip")

LIBRARY = os.path.join(os.path.dirname(os.path.abspath(vh.__file__)), "libvestra_hip.so")


@pytest.mark.parametrize("kernel", ["attention_tile_kernel", "attention_few_kernel"])
def test_every_offset_is_inside_the_bounds_check(kernel):
    """A buffer load checks the lane's and the instruction's own offset against the buffer's
    size; the scalar offset comes on top of that, unchecked.  A block past the end of the keys
    is read within its buffer only where no load has a scalar offset."""
    found = code_objects.kernels(LIBRARY, kernel)
    assert len(found) == 16  # two formats, four scorings, masked or not
    for name, (_, code) in found.items():
        loads = [x for x in code if x.startswith("buffer_load")]
        assert loads, name
        for x in loads:
            scalar = x.split(", ")[3].split()[0]
            assert scalar == "0", (name, x)


@pytest.mark.parametrize("kernel", ["attention_few_kernel", "attention_row_kernel",
                                    "attention_join_kernel"])
def test_short_chains_hold_nothing_in_scratch(kernel):
    """Kernels that are bound by the latency of one chain: no spilled vector register and no
    array or choice of addresses that lives in memory."""
    found = code_objects.kernels(LIBRARY, kernel)
    assert found
    for name, (values, code) in found.items():
        assert values["private_segment_fixed_size"] == 0 and values["vgpr_spill_count"] == 0, name
        assert not [x for x in code if x.startswith(("scratch_", "flat_"))], name
