"""The HIP sources themselves: what a file compiles is launched there."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "turing-bf16_amd" / "csrc"
KERNEL = re.compile(r"__global__[^;{]*?\bvoid\s+(\w+)\s*\(", re.S)


def kernels(path):
    return KERNEL.findall(re.sub(r"//[^\n]*", "", path.read_text()))


def included(path):
    """The headers beside a file that it includes, directly or through others."""
    found, todo = set(), [path]
    while todo:
        for name in re.findall(r'#include "([\w.]+)"', todo.pop().read_text()):
            if (CSRC / name).exists() and name not in found:
                found.add(name)
                todo.append(CSRC / name)
    return [CSRC / name for name in sorted(found)]


def test_kernels_are_found():
    assert "paged_write_kernel" in kernels(CSRC / "paged.hip") and "pingpong_kernel" in kernels(CSRC / "gemm_tiles.h")


@pytest.mark.parametrize("source", sorted(p.name for p in CSRC.glob("*.hip")))
def test_every_kernel_that_a_file_compiles_is_launched_in_it(source):
    text = re.sub(r"//[^\n]*", "", (CSRC / source).read_text())
    for path in (CSRC / source, *included(CSRC / source)):
        for name in kernels(path):
            assert re.search(rf"\b{name}\s*(<[^;]*?)?<<<", text, re.S), f"{name} ({path.name}) is compiled into {source} and launched nowhere there"
