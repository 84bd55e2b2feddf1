"""How kernels that start before the one ahead of them has ended may read: found in their source, without a GPU."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "mkernel_b200" / "csrc"


def code(path):
    """The source without its comments."""
    return re.sub(r"/\*.*?\*/", "", re.sub(r"//[^\n]*", "", path.read_text()), flags=re.S)


def test_no_operand_is_read_as_if_nobody_wrote_it():
    """All kernels are launched with programmatic serialization: while they are resident the kernel ahead still writes
    their operands, which the read-only path (__ldg, ld.global.nc, __restrict__ const) does not allow for."""
    sources = [p for p in sorted(CSRC.iterdir()) if p.suffix in (".cu", ".cuh", ".h")]
    assert len(sources) > 6
    for p in sources:
        for word in ("__ldg", "ld.global.nc", "__restrict__"):
            assert word not in code(p), f"{p.name}: {word}"


def test_every_such_kernel_waits_first():
    """Each __global__ kernel of these files has the wait, and lets the next kernel start only behind it."""
    for name in ("w4.cu", "w4_tile.cu", "rotary.cu"):
        text = code(CSRC / name)
        kernels = text.count("__global__")
        assert kernels > 0 and text.count("grid_dependency_wait()") == kernels, name
        assert len(re.findall(r"grid_dependency_wait\(\);\s*ptx::grid_launch_dependents\(\);", text)) == kernels, name
