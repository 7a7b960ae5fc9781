"""Plans of the token operators that need no GPU: how the norm of any width shares its rows out."""

from __future__ import annotations

import subprocess

from arthip_b200 import build

SHAPES = r"""
#include <cstdio>
#include "kernels/token_norm_shape.h"
struct Print {
  int channels;
  template <int GROUP, int LANES, int N>
  int operator()() const { return std::printf("%d %d %d %d\n", channels, GROUP, LANES, N); }
};
int main() {
  for (int c = 1; c <= 8192; ++c) ah::token_norm::staged_shape(c, Print{c});
}
"""


def test_every_width_of_the_staged_norm_holds_its_rows(tmp_path):
    """Of a lane's N elements only the last two are tested against the row's end, so at every
    width all others have to lie within it; and the lanes have to hold the row."""
    (tmp_path / "shapes.cc").write_text(SHAPES)
    exe = tmp_path / "shapes"
    subprocess.run(["g++", "-std=c++17", "-I", str(build.CSRC), str(tmp_path / "shapes.cc"), "-o", str(exe)], check=True)
    lines = [tuple(map(int, l.split())) for l in subprocess.run([str(exe)], capture_output=True, text=True,
                                                                check=True).stdout.splitlines()]
    assert [l[0] for l in lines] == list(range(1, 8193))
    for c, group, lanes, n in lines:
        assert group in (32, 64, 128, 256) and (lanes == group or (group == 32 and 32 % lanes == 0)), c
        assert n % 2 == 0 and (n - 2) * lanes <= c <= n * lanes, (c, lanes, n)
