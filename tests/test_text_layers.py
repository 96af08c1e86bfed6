"""Chunks of keys and the layers that they leave, counted as the host and the kernels do (no GPU: the
functions are compiled for the host)."""
import shutil
import subprocess

import pytest

from wuxianhuabu_b200.build import CSRC

SRC = r'''
#include <algorithm>
#include <cstdint>
#include <cstdio>
#define __host__
#define __device__
%s
int main() {
  const int chunks[] = {0, 64, 96, 128, 256}, mosts[] = {4, 8, 16, 32};
  for (int chunk : chunks)
    for (int most : mosts) {
      int seen = 0;  // of all lengths up to lk
      for (int lk = 0; lk < 70000; ++lk) {
        const int layers = layers_of(chunk, most, lk);
        // the units of a walk, one after the other, until the keys are out
        int units = 1;
        if (chunk)
          for (int at = chunk_of(chunk, most, lk); at < lk; at += chunk_of(chunk, most, lk)) ++units;
        seen = std::max(seen, layers);
        if (units != layers || layers > most || most_layers(chunk, most, lk) < seen)
          return printf("chunk %%d most %%d keys %%d: %%d units, %%d layers, room for %%d\n", chunk, most, lk, units, layers,
                        most_layers(chunk, most, lk)), 1;
      }
      for (int64_t keys : {int64_t(1) << 30, (int64_t(1) << 31) - 1, int64_t(1) << 34})
        if (most_layers(chunk, most, keys) != (chunk ? most : 1))
          return printf("%%d of %%d: %%lld\n", chunk, most, (long long)keys), 1;
    }
  return 0;
}
'''


def test_layers_are_the_units_of_a_walk(tmp_path):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no host compiler")
    text = (CSRC / "wx_text_dev.cuh").read_text()
    a = text.index("__host__ __device__ inline int chunk_of")
    b = text.index("}", text.index("inline int most_layers")) + 1
    (tmp_path / "b.cpp").write_text(SRC % text[a:b])
    subprocess.run([gxx, "-O1", "-ftrapv", str(tmp_path / "b.cpp"), "-o", str(tmp_path / "b")], check=True)
    out = subprocess.run([str(tmp_path / "b")], text=True, capture_output=True)
    assert out.returncode == 0, out.stdout
