"""What the sources of the 8-bit operators must not contain. Their kernels may start while the kernel before them in the
stream still writes their inputs, and a stale line read then shows in no test that can be relied on."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "elips_b200" / "csrc"


@pytest.mark.parametrize("name", ["int8_kernels.cuh", "int8_gemm.cuh"])
def test_no_non_coherent_loads(name):
    """Neither __ldg nor ld.global.nc, nor a const __restrict__ pointer that lets the compiler choose them: that path is
    for data that is read-only for the kernel's whole life."""
    code = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    assert not re.search(r"__ldg|global\.nc|__restrict__", code)
