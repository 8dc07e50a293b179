"""CPU test of the walk that the paged token kernels take through a run of key blocks (csrc/paged_token.hpp), compiled
for the host with the package's own flags."""

from __future__ import annotations

import importlib
import shutil
import subprocess

import pytest

build = importlib.import_module("collaborative-edge-system_amd.build")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "paged_token.hpp"

// Runs measured on lengths that have changed by the time that the walk reads them: every unit lies in a row that
// there is, and every walk ends.
int main() {
  srand(7);
  int past = 0;
  for (int turn = 0; turn < 20000; ++turn) {
    const int rows = 1 + rand() % 5, units = 1 + rand() % 4;
    std::vector<int> then(rows), now(rows);
    for (int b = 0; b < rows; ++b) then[b] = 1 + rand() % 6, now[b] = turn % 2 ? then[b] : 1 + rand() % 6;
    int b = rand() % rows, unit = rand() % units, lo = rand() % then[b], blocks = then[b], total = 0;
    for (int x = b; x < rows; ++x) total += then[x] * units;
    total -= unit * then[b] + lo;                        // blocks from here to the line's end
    int left = turn % 3 ? 1 + rand() % total : total, want = left, seen = 0, steps = 0;
    while (true) {
      if (b < 0 || b >= rows || unit < 0 || unit >= units || left <= 0 || ++steps > 1000) {
        printf("turn %d: row %d of %d, unit %d of %d, left %d\n", turn, b, rows, unit, units, left);
        return 1;
      }
      const int hi = blocks < lo + left ? blocks : lo + left;
      seen += hi - lo;
      if (!cea::next_unit(b, unit, lo, left, blocks, hi - lo, units, rows, [&](int row) {
            if (row < 0 || row >= rows) ++past;
            return now[row < rows ? row : 0];
          }))
        break;
    }
    if (past != 0 || (turn % 2 && seen != want)) {
      printf("turn %d: %d of %d blocks, %d lengths read past the last row\n", turn, seen, want, past);
      return 1;
    }
  }
  puts("ok");
  return 0;
}
"""


@pytest.mark.skipif(shutil.which(build.HIPCC) is None and not build.HIPCC.startswith("/"),
                    reason="hipcc not available")
def test_runs_end_at_the_last_row(tmp_path):
    src, exe = tmp_path / "runs.hip", tmp_path / "runs"
    src.write_text(PROGRAM)
    flags = [f for f in build.COMMON_FLAGS if f != "-fPIC"]
    subprocess.run([build.HIPCC, *flags, str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    got = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert got.returncode == 0 and got.stdout == "ok\n", got.stdout + got.stderr
