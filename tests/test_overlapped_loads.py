"""Kernels that begin under the kernel ahead of them load what it writes with ordinary loads.

The non-coherent path (`__ldg`, `ld.global.nc`, and what the compiler may make of a `const __restrict__`
pointer) is for memory that nobody writes while the kernel lives.  A kernel launched by launch_overlapped
lives from under the tail of its predecessor on, which may be the writer of its operands; its
griddepcontrol.wait orders ordinary loads.  Checked from the text, without a GPU.
"""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "pantheon_b200" / "csrc"


def _code(path: Path) -> str:
    text = re.sub(r"/\*.*?\*/", "", path.read_text(), flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


OVERLAPPED = sorted(p for p in CSRC.glob("*.cu") if "wait_previous_grid()" in _code(p))


def test_the_overlapped_kernels_are_found():
    assert len(OVERLAPPED) == 5
    for p in CSRC.glob("*.cu"):
        if "launch_overlapped(" in _code(p):
            assert p in OVERLAPPED, f"{p.name}: an overlapped launch without its wait"


def test_no_non_coherent_loads_in_overlapped_kernels():
    shared = [CSRC / n for n in ("qg_launch.cuh", "qg_rows.cuh", "qg_mxfp4.cuh", "qg_mxfp4_mma.cuh", "qg_gated.cuh")]
    for p in OVERLAPPED + shared:
        code = _code(p)
        assert "__ldg" not in code and ".nc" not in code and "__restrict__" not in code, p.name
