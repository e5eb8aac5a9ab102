"""Where ranges of weight cut a query tile's key tiles (attention_index.h, cut_of), compiled for the host: in order,
no part shorter than the multiple that is cut at, pairs of under 16 tiles whole."""
import os
import subprocess

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lunaflux_amd", "csrc", "kernels")

SOURCE = r"""
#define LF_DEVICE static inline
#include "attention_index.h"
#include <stdio.h>
using namespace attn;
int main() {
  if (cut_tiles(511, 64) != 4 || cut_tiles(512, 64) != 8 || cut_tiles(1, 32) != 8) return puts("cut_tiles"), 1;
  for (int cut = 4; cut <= 8; cut += 4) {
    for (int tiles = 1; tiles < 200; ++tiles) {
      const int64_t begin = 1000, weight = 64 * tiles + 256;
      const int least = tiles < 4 * kCut ? kCut : cut;
      int before = 0;
      for (int64_t u = begin - 3; u <= begin + weight + 3; ++u) {
        const int c = cut_of(u, begin, weight, tiles, cut);
        bool wrong = c < before || c > tiles || (c != before && c - before < least && c - before != tiles);
        if (c != 0 && c != tiles) wrong |= tiles < 2 * kCut || c % least != 0 || tiles - c < least;
        if (u <= begin) wrong |= c != 0;
        if (u >= begin + weight) wrong |= c != tiles;
        if (wrong) return printf("cut %d of %d tiles at %lld: %d after %d\n", cut, tiles, (long long)(u - begin), c, before), 1;
        before = c;
      }
    }
  }
  // as much as a range can weigh
  const int64_t weight = (int64_t(1) << 31) + 512;
  if (cut_of(weight / 2, 0, weight, 1 << 25, 4) != 1 << 24) return puts("large"), 1;
  return 0;
}
"""


def test_cuts(tmp_path):
    source, exe = tmp_path / "cuts.cpp", tmp_path / "cuts"
    source.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", KERNELS, str(source), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout + run.stderr
