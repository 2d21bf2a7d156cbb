"""The places that the 4-bit attention's asynchronous copies write to, gone through lane by lane on the CPU."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "lunara_b200" / "csrc"

PROGRAM = """
#include <cstdio>
#include "scale_copy.h"
template <int KT, int DP>
void all(int dim) {
  for (int lane = 0; lane < 32; ++lane) {
    const lunara::ScaleCopy s = lunara::scale_copy<KT, DP>(lane, dim / 16);
    if (s.copies) std::printf("%d %d %d %d %d\\n", dim, s.kv, s.group, s.piece, s.place);
  }
}
int main() {
  all<32, 64>(32); all<32, 64>(64); all<32, 128>(96); all<32, 128>(128);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_scale_copies_write_every_byte_once(tmp_path):
    """The scales of a tile's 32 keys, for every head dimension that the streaming kernel takes with 4 bits: each
    piece is copied once, to a place of its own (asynchronous copies of a warp have no order among themselves)."""
    (tmp_path / "places.cc").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(tmp_path / "places.cc"), "-o", str(tmp_path / "places")], check=True)
    lines = subprocess.run([str(tmp_path / "places")], capture_output=True, text=True, check=True).stdout.splitlines()
    rows = [tuple(map(int, line.split())) for line in lines]
    for dim in (32, 64, 96, 128):
        srow, padded = dim // 16, 64 if dim <= 64 else 128
        for kv in (0, 1):
            mine = [r for r in rows if r[0] == dim and r[1] == kv]
            written = [place + i for *_, place in mine for i in range(16)]
            assert sorted(written) == list(range(32 * srow)), (dim, kv)   # every byte that is read, and each of them once
            assert max(written) < 32 * (padded // 16)
            assert all(place == group * 8 * srow + 16 * piece and 16 * piece < 8 * srow for _, _, group, piece, place in mine)
