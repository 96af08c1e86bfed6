"""The number of pieces that items of new prompts behind a shared prefix are cut into (no GPU: the host's rule
is compiled by itself)."""
import random
import shutil
import subprocess

import pytest

from wuxianhuabu_b200.build import CSRC

SRC = r'''
#include <cmath>
#include <cstdint>
#include <cstdio>
constexpr int kTfMinTiles = 8;
constexpr int64_t kTfPartBytes = int64_t(256) << 20;
%s
int main() {
  int sms, hd, wide;
  double some, tiles;
  long long rows;
  while (scanf("%%d %%lf %%lf %%lld %%d %%d", &sms, &some, &tiles, &rows, &hd, &wide) == 6)
    printf("%%d\n", prefix_pieces(sms, some, tiles, rows, hd, wide != 0));
}
'''


@pytest.fixture(scope="module")
def pieces(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no host compiler")
    at = tmp_path_factory.mktemp("pieces")
    text = (CSRC / "wx_text_flash.cu").read_text()
    assert "kTfMinTiles = 8;" in text and "kTfPartBytes = int64_t(256) << 20;" in text
    a = text.index("inline int prefix_pieces")
    (at / "b.cpp").write_text(SRC % text[a:text.index("\n}", a) + 2])
    subprocess.run([gxx, "-O1", str(at / "b.cpp"), "-o", str(at / "b")], check=True)

    def run(cases):
        out = subprocess.run([str(at / "b")], input="\n".join(" ".join(map(str, c)) for c in cases), text=True,
                             capture_output=True, check=True).stdout
        return list(map(int, out.split()))
    return run


def test_room_is_bounded_and_pieces_have_their_tiles(pieces):
    rng = random.Random(1)
    cases = []
    for _ in range(3000):
        rows = int(2 ** rng.uniform(4, 26))
        cases.append((148, max(1.0, rows / 256 * rng.uniform(1, 4)), 2 ** rng.uniform(0, 11), rows, rng.choice([64, 128]),
                      rng.choice([0, 1])))
    for (_, some, tiles, rows, hd, _), n in zip(cases, pieces(cases)):
        assert n == 1 or (8 * n <= tiles and n * rows * (4 * hd + 8) <= 256 << 20), (some, tiles, rows, hd, n)


def test_many_rounds_are_not_cut(pieces):
    # 80,000 new tokens behind 128,000 (32 / 8 heads), 99,939 behind the same (64 / 8): what a part of a round saves is
    # less than the pieces' sums cost; 148 items of 50 tiles fill a round by themselves
    assert pieces([(148, 10080, 1007, 80000 * 32, 128, 0), (148, 25000, 1007, 99939 * 64, 128, 0),
                   (148, 148, 49, 33852, 128, 1)]) == [1, 1, 1]


def test_few_long_items_are_cut(pieces):
    # 8 and 16 items of 200 tiles: as many pieces as fit beside one another; a little more than one round: in three
    assert pieces([(148, 8, 200, 8 * 256, 128, 0), (148, 16, 200, 16 * 256, 128, 0),
                   (148, 160, 63.2, 160 * 256, 128, 0)]) == [18, 9, 3]
