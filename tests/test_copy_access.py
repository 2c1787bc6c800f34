"""The width in which dispatch copies rows, from its rule compiled for the host: an access never is
wider than its address is aligned (the hardware may tolerate it, the compiler need not)."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "mtp_amd" / "csrc"
PROGRAM = """
#include <cstdio>
#include "access.h"
int main() {
  for (long row = 2; row <= 64; row += 2)
    for (long p = 0; p < 16; p += 2)
      for (long q = 0; q < 16; q += 2)
        std::printf("%ld %ld %ld %d\\n", row, p, q,
                    copy_access_bytes(row, (void*)(4096 + p), (void*)(8192 + q)));
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_copies_are_as_wide_as_everything_is_aligned(tmp_path):
    (tmp_path / "a.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", "a.cpp", "-o", "a"], cwd=tmp_path, check=True)
    lines = subprocess.run([tmp_path / "a"], capture_output=True, text=True, check=True).stdout
    cases = [tuple(map(int, line.split())) for line in lines.splitlines()]
    assert len(cases) == 32 * 8 * 8
    for row, p, q, width in cases:
        want = next(w for w in (16, 4, 2) if row % w == p % w == q % w == 0)
        assert width == want, (row, p, q)
