"""How the norms' kernels cut a row into 16-byte copies, on the CPU: the header that the
kernels use is compiled for the host. An asynchronous 16-byte copy needs both of its
addresses aligned, whatever it reads."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include "frattn_row_pieces.h"
int main() {
  for (int off = 0; off < 16; ++off)
    for (int bytes = 1; bytes <= 130; ++bytes)
      for (int n = 1; n <= 32; n *= 4)
        for (int t = 0; t < n; ++t)
          frattn::row_pieces(off, bytes, t, n, [&](int at, int from, int size) {
            std::printf("%d %d %d %d %d %d %d\n", off, bytes, n, t, at, from, size);
          });
}
"""


@pytest.fixture(scope="module")
def pieces(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("pieces")
    (d / "p.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", "-I", os.path.join(ROOT, "fused_rope_attn_b200", "csrc"), "-o",
                    str(d / "p"), str(d / "p.cpp")], check=True)
    out = subprocess.run([str(d / "p")], check=True, capture_output=True, text=True).stdout
    rows = {}
    for line in out.splitlines():
        off, nbytes, n, t, at, src, size = map(int, line.split())
        rows.setdefault((off, nbytes, n), []).append((t, at, src, size))
    assert len(rows) == 16 * 130 * 3
    return rows


def test_every_address_is_aligned(pieces):
    for (off, nbytes, n), ps in pieces.items():
        for t, at, src, size in ps:
            assert at % 16 == 0 and src % 16 == 0 and 0 <= size <= 16, (off, nbytes, n, t, at, src, size)


def test_the_row_is_covered_once_and_zeros_follow(pieces):
    for (off, nbytes, n), ps in pieces.items():
        end = off + nbytes
        ats = sorted(at for _, at, _, _ in ps)
        assert ats == list(range(0, ats[-1] + 16, 16))  # each piece once, no gap
        assert end <= ats[-1] < end + 16  # the last is all zeros
        for _, at, src, size in ps:
            assert size == max(0, min(16, end - at))
            assert 0 <= src and src + size <= end  # nothing past the row's end
            assert size == 0 or src == at
            assert src < end  # a piece that the row touches
