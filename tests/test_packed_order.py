"""The order of the blocks of packed prompts (batch.hpp, host code): the count of
a sequence's blocks of at least L tiles against the blocks one by one."""
import pathlib
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

PROGRAM = r"""
#include <cstdio>
#include "batch.hpp"

int main() {
  long cases = 0;
  const int pasts[] = {0, 1, 5, 31, 32, 33, 64, 100, 4095};
  for (int block : {32, 64, 128})
    for (int G : {1, 2, 3, 4, 8, 33, 200})
      for (int past : pasts)
        for (int rows : {1, 2, 7, 31, 32, 33, 64, 65, 100, 257}) {
          const int tile = 32, blocks = (rows * G + block - 1) / block;
          const int most = (past + rows + tile - 1) / tile;
          for (int L = 1; L <= most + 2; ++L) {
            int want = 0;
            for (int b = 0; b < blocks; ++b) {
              const int last = ((b + 1) * block < rows * G ? (b + 1) * block : rows * G) - 1;
              want += (past + last / G + 1 + tile - 1) / tile >= L;
            }
            const int got = ikv::blocks_of_tiles(rows, past, G, block, tile, L);
            ++cases;
            if (got != want) {
              std::printf("block %d G %d past %d rows %d L %d: %d, not %d\n", block, G, past, rows, L, got, want);
              return 1;
            }
          }
        }
  std::printf("%ld cases\n", cases);
  return 0;
}
"""


def test_blocks_of_at_least_so_many_tiles(tmp_path):
    if not pathlib.Path(HIPCC).exists():
        pytest.skip("hipcc not available")
    src, exe = tmp_path / "order.hip", tmp_path / "order"
    src.write_text(PROGRAM)
    subprocess.run([HIPCC, "--offload-host-only", "-std=c++20", "-O1", "-I", str(ROOT / "infer-llm_amd" / "csrc"),
                    "-o", str(exe), str(src)], check=True, capture_output=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
    assert int(done.stdout.split()[0]) > 1000
