"""The order in which a launch's workgroups take their items (csrc/tile_item.h), run
on the host: every item once, and sorted work spread evenly over the XCDs."""

from __future__ import annotations

import math
import shutil
import subprocess

import numpy as np
import pytest

from trnsparse_amd import build_lib

PROGRAM = """
#include <stdio.h>
#include "tile_item.h"
int main() {
  const int heads[] = {1, 2, 3, 4, 5, 7, 8, 9, 12, 16}, items[] = {1, 7, 44, 140, 301};
  for (int sorted = 0; sorted < 2; ++sorted)
    for (int H : heads)
      for (int P : items)
        for (int64_t g = 0; g < tsp::head_grid(P, H); ++g) {
          int64_t h = -1, i = -1;
          if ((sorted ? tsp::sorted_item : tsp::head_item)((uint32_t)g, P, H, h, i))
            printf("%d %d %d %lld %lld %lld\\n", sorted, H, P, (long long)g, (long long)h, (long long)i);
        }
}
"""


@pytest.fixture(scope="module")
def order(tmp_path_factory):
    if not shutil.which(build_lib.HIPCC):
        pytest.skip("no hipcc")
    d = tmp_path_factory.mktemp("order")
    (d / "order.hip").write_text(PROGRAM)
    subprocess.run([build_lib.HIPCC, "--offload-host-only", "-O1", "-std=c++17", f"-I{build_lib.CSRC}",
                    str(d / "order.hip"), "-o", str(d / "order")], check=True, capture_output=True, timeout=120)
    out = subprocess.run([str(d / "order")], check=True, capture_output=True, text=True, timeout=60).stdout
    return np.array([[int(v) for v in line.split()] for line in out.splitlines()])


def test_every_item_once(order):
    for sorted_, H, P in {tuple(r) for r in order[:, :3].tolist()}:
        rows = order[(order[:, :3] == (sorted_, H, P)).all(1)]
        at = rows[:, 4] * P + rows[:, 5]
        assert len(rows) == H * P and (np.sort(at) == np.arange(H * P)).all()
    assert len({tuple(r) for r in order[:, :3].tolist()}) == 2 * 10 * 5


def test_sorted_work_is_even(order):
    """Items as long as their places from the end: of each head an XCD has every n-th item
    (n = 8 / gcd(heads, 8)), and two such sums differ by the longest item at most."""
    rows = order[order[:, 0] == 1]
    for H, P in {tuple(r) for r in rows[:, 1:3].tolist()}:
        r = rows[(rows[:, 1] == H) & (rows[:, 2] == P)]
        share = np.bincount(r[:, 3] % 8, weights=P - r[:, 5], minlength=8)
        assert share.max() - share.min() <= H // math.gcd(H, 8) * P, (H, P, share)
