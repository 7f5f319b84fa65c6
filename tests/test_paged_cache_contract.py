"""What the paged-cache operators promise and no device is needed to check."""
import os
import re

import pytest

from mlx_server_runtime_b200 import _lib

CSRC = os.path.join(os.path.dirname(_lib.__file__), "csrc")


def source(name):
    """A source file without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        s = f.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", " ", s, flags=re.S)


@pytest.mark.parametrize("name", ["paged_attn.cu", "paged_attn_tc.cu", "paged_cache.cu",
                                  "rows_units.cuh", "kv_dequant.cuh"])
def test_no_read_only_loads(name):
    """With launch overlap these kernels start while the kernel that writes the pools, tables
    and queries they read may still run. A load through the read-only path needs data that
    does not change for as long as the kernel lives, so none is made: neither by hand, nor by
    parameters that allow the compiler to."""
    s = source(name)
    assert not re.search(r"__ldg\b|\bld\.global(\.\w+)*\.nc\b", s)
    assert not re.search(r"\bconst\b[^;,(){}]*\*\s*__restrict__", s)
