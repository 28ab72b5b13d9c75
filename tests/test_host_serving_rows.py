"""What the lanes of the paged attention load of a row, by the kernel's own rules compiled for the
CPU: every load ends inside the row, for every head dim. No GPU."""
import pathlib
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "turing-bf16_amd" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "paged_rows.h"
using namespace tbf16;
int main() {
  for (int D = 8; D <= 256; D += 8) {
    const int DP = D <= 64 ? 64 : D <= 128 ? 128 : 256;
    for (int g = 0; g < 4; ++g)
      for (int i = 0; i < key_pieces(DP); ++i) printf("k %d %d %d\n", D, key_piece(D, g, i), kKeyPiece);
    for (int r = 0; r < 16; ++r)
      for (int i = 0; i < value_pieces(DP); ++i) printf("v %d %d %d\n", D, value_piece(D, DP, r, i), value_piece_size(DP));
  }
}
"""


@pytest.fixture(scope="module")
def loads(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("rows")
    (d / "rows.cpp").write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", f"-I{CSRC}", str(d / "rows.cpp"), "-o", str(d / "rows")], check=True)
    out = {}
    for line in subprocess.run([str(d / "rows")], check=True, capture_output=True, text=True).stdout.splitlines():
        kind, D, at, size = line.split()
        out.setdefault((kind, int(D)), []).append((int(at), int(size)))
    return out


@pytest.mark.parametrize("kind", ["k", "v"])
@pytest.mark.parametrize("D", range(8, 257, 8))
def test_loads_stay_in_the_row(loads, kind, D):
    pieces = loads[kind, D]
    assert all(0 <= at and at + size <= D and at % min(size, 8) == 0 for at, size in pieces), pieces
    covered = {e for at, size in pieces for e in range(at, at + size)}
    assert covered == set(range(D))  # and all of the row is loaded
    assert len(pieces) == {"k": 4 * (2 if D <= 64 else 4 if D <= 128 else 8), "v": 16 * (2 if D > 128 else 1)}[kind]
