"""The places of x that the adapters' kernels read (madi_amd/csrc/lora_places.h), on the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <stdio.h>
#include "lora_places.h"
int main() {
  // a row is taken in chunks of 2048 elements, four to a load: every place of its last chunk, inside the row or not
  for (uint32_t k = 64; k <= 4160; k += 64)
    for (uint32_t at = 0; at < (k + 2047) / 2048 * 2048; at += 4) {
      const uint32_t place = madi::lora_x_place(at, k);
      if (place % 4 || place + 4 > k || (at < k && place != at)) return printf("k %u: %u read at %u\n", k, at, place), 1;
    }
  return 0;
}
"""


def test_no_load_of_x_leaves_its_row(tmp_path):
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "madi_amd", "csrc"), str(tmp_path / "t.cpp"),
                    "-o", str(tmp_path / "t")], check=True)
    run = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_the_kernel_reads_x_there():
    text = open(os.path.join(ROOT, "madi_amd", "csrc", "lora.hip")).read()
    tile = text[text.index("void lora_tile_kernel("):]
    body = tile[tile.index("const auto load_x"):]
    assert "x + lora_x_place(" in body[:body.index("};")]
