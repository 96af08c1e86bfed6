"""The bounds of the keys that a query row sees, in 32-bit arithmetic as the kernels form them, against
the same in whole numbers (no GPU: key_hi and key_lo are compiled for the host)."""
import itertools
import shutil
import subprocess

import pytest

from wuxianhuabu_b200.build import CSRC

INT_MAX = 2 ** 31 - 1

SRC = r'''
#include <cstdio>
#include <algorithm>
#define __device__
#define __forceinline__ inline
using std::max;
using std::min;
struct TextAttnParams { int causal, window; };
struct Seq { long long q0, k0; int lq, lk; };
%s
int main() {
  long long causal, window, lq, lk, tok;
  while (scanf("%%lld %%lld %%lld %%lld %%lld", &causal, &window, &lq, &lk, &tok) == 5) {
    TextAttnParams p{(int)causal, (int)window};
    Seq s{0, 0, (int)lq, (int)lk};
    printf("%%d %%d\n", key_lo(p, s, (int)tok), key_hi(p, s, (int)tok));
  }
}
'''


def test_key_bounds_hold_at_the_integer_limits(tmp_path):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no host compiler")
    text = (CSRC / "wx_text_dev.cuh").read_text()
    a = text.index("__device__ __forceinline__ int key_hi")
    b = text.index("}", text.index("int key_lo")) + 1
    (tmp_path / "b.cpp").write_text(SRC % text[a:b])
    # -ftrapv: an addition that overflows ends the program instead of wrapping
    subprocess.run([gxx, "-O0", "-ftrapv", str(tmp_path / "b.cpp"), "-o", str(tmp_path / "b")], check=True)
    lengths = [0, 1, 5, 20, 130, 70000, 2 ** 30, INT_MAX]
    cases = []
    for lq, lk, window in itertools.product(lengths, lengths, [0, 1, 16, 4096, 2 ** 30, INT_MAX - 7, INT_MAX]):
        for tok in {0, lq // 2, lq - 1}:
            if 0 <= tok < lq:
                cases.append((1, window, lq, lk, tok))
    out = subprocess.run([str(tmp_path / "b")], input="\n".join(" ".join(map(str, c)) for c in cases), text=True,
                         capture_output=True, check=True).stdout.split("\n")
    for c, line in zip(cases, out):
        _, window, lq, lk, tok = c
        at = tok + lk - lq  # the key at which the row stands
        hi = max(0, min(lk, at + 1))
        lo = max(0, at - window + 1) if window else 0
        got = tuple(map(int, line.split()))
        assert got == (lo, hi), (c, got, (lo, hi))
