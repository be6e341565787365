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
