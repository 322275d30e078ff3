"""What the sources of the 8-bit cache's kernels must not contain."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "diffuse-rs_b200", "csrc")


@pytest.mark.parametrize("name", ["kv8.cuh", "attn_kv8_rows.cuh", "attn_kv8_tile.cuh"])
def test_no_read_only_loads(name):
    # These kernels start while the kernel before them runs, so that what they
    # read may still be written after their start: no read-only loads, nor
    # pointers that let the compiler make them.
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert not re.search(r"__ldg\s*\(|ld\.global\.nc|__restrict__", code)
