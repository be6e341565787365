"""Properties of the feed-forward products' machine code that no result shows, read from the
built library."""
import os

import pytest

import code_objects

vh = pytest.importorskip("vestra_hip")

LIBRARY = os.path.join(os.path.dirname(os.path.abspath(vh.__file__)), "libvestra_hip.so")


@pytest.mark.parametrize("kernel", ["gated_kernel", "gated_grad_kernel", "gradients_kernel",
                                    "gated_few_kernel", "linear_i8_kernel", "linear_i8_few_kernel",
                                    "linear_i8_rows_kernel", "quantise_rows_kernel"])
def test_nothing_in_scratch(kernel):
    """Sums and fragments stay in registers: a tile's are most of what a wave has."""
    found = code_objects.kernels(LIBRARY, kernel)
    assert found
    for name, (values, code) in found.items():
        assert values["private_segment_fixed_size"] == 0 and values["vgpr_spill_count"] == 0, name
        assert not [x for x in code if x.startswith("scratch_")], name


@pytest.mark.parametrize("kernel", ["gated_kernel", "gated_grad_kernel", "linear_i8_kernel",
                                    "gradients_kernel"])
def test_stages_land_before_a_barrier(kernel):
    """The loads into LDS are counted by hand: every kernel that has them waits for vmcnt before
    it meets the others, and never reads a stage without having met them."""
    for name, (_, code) in code_objects.kernels(LIBRARY, kernel).items():
        first = next(i for i, x in enumerate(code)
                     if x.startswith("buffer_load") and x.endswith("lds"))
        waited = [i for i, x in enumerate(code)
                  if i > first and x.startswith("s_waitcnt") and "vmcnt" in x]
        met = next(i for i, x in enumerate(code) if i > first and x.startswith("s_barrier"))
        product = next(i for i, x in enumerate(code) if x.startswith("v_mfma"))
        assert waited and waited[0] < met < product, name
