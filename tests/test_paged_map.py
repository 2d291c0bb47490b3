"""Where the kernels look a position's page up, in the kernels' own header, on the CPU."""

import subprocess

import pytest

from exp3_amd import build

PROGRAM = r"""
#include <cstdio>
#include <cstring>
#include "paged.h"
int main() {
  const int32_t memory[] = {2, 0, 1, 3, 2, 9, -1, 1 << 30, 4};     // two rows of three, 2 in front of each
  spx::PagedMap m{};
  m.table = memory + 1;
  m.table_stride = 4;
  m.width = 3;
  m.pages = 4;
  m.page_shift = 4;
  const int rows[] = {0, 1};
  for (int b : rows)
    for (int p : {-1, 0, 15, 16, 47, -16, -2147483647 - 1}) printf("%d ", m.page(b, p));
}
"""


def test_pages_of_positions(tmp_path):
    """A position of -1, the last one of a sequence without keys, has no page, and the entry in
    front of the table's row is not read for it (its value would be a page)."""
    source = tmp_path / "map.hip"
    source.write_text(PROGRAM)
    program = tmp_path / "map"
    done = subprocess.run([build._hipcc(), *build.HIPCC_FLAGS, "-O1", f"-I{build.CSRC}", str(source), "-o",
                           str(program)], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    got = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert got.returncode == 0
    assert [int(x) for x in got.stdout.split()] == [-1, 0, 0, 1, 3, -1, -1,
                                                    -1, -1, -1, -1, -1, -1, -1]
