"""CPU: the tiles that an expert's rows take (csrc/grouped.cuh, the function that the kernel calls), compiled for the host."""
import os
import shutil
import subprocess

import pytest


def _tiles(pairs, where):
  from faster_weathernext import _build
  source, program = os.path.join(where, "tiles.cpp"), os.path.join(where, "tiles")
  with open(source, "w") as f:
    f.write('#include <cstdio>\n#include "grouped.cuh"\nint main() {\n  int rows, unit;\n'
            '  while (scanf("%d %d", &rows, &unit) == 2) printf("%d\\n", fwn::group_tiles(rows, unit));\n}\n')
  cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_build.nvcc()))), "include")
  subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-I", _build.CSRC, "-I", cuda, source, "-o", program], check=True)
  out = subprocess.run([program], input="\n".join(f"{r} {u}" for r, u in pairs), text=True, capture_output=True, check=True).stdout
  return [int(v) for v in out.split()]


def test_tiles_of_an_expert(tmp_path):
  """Up to the largest tensor (2^31 - 1,025 rows) and the longest run (2^20 stages of 64 rows): their sum passes 2^31. One expert
  of 2^31 - 1,025 rows and 8 x 8 weights plans runs of some 15 million rows."""
  most = 2 ** 31 - 1025
  rows = [0, 1, 63, 64, 65, 255, 256, 257, 40_962, 2 ** 30, most - 1, most]
  units = [64, 128, 256, 64 * 9, 64 * 233_017, 2 ** 26]
  pairs = [(r, u) for r in rows for u in units]
  if not shutil.which("g++"):
    pytest.skip("no host compiler")
  assert _tiles(pairs, tmp_path) == [-(-r // u) for r, u in pairs]
  assert _tiles([(r, 0) for r in rows], tmp_path) == [1] * len(rows)
