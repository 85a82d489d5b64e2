"""Into parts of which length paged attention cuts its keys (CPU): the rule's source, compiled for the host."""

from __future__ import annotations

import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "bioemu2_amd" / "csrc"
SOURCE = """
#include "paged_parts.h"
extern "C" unsigned part_length(const unsigned* tiles, int n, unsigned items, unsigned groups, unsigned least, int search,
                                unsigned* counted) {
  unsigned total = 0, live = 0;
  for (int i = 0; i < n; ++i) total += tiles[i] * items, live += tiles[i] ? items : 0;
  return bioemu::part_length(total, live, groups, least, search != 0, [&](unsigned part) {
    unsigned c = 0;
    for (int i = 0; i < n; ++i) c += (tiles[i] + part - 1) / part;
    ++*counted;
    return c * items;
  });
}
"""


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    where = tmp_path_factory.mktemp("parts")
    (where / "parts.cpp").write_text(SOURCE)
    gxx = shutil.which("g++") or shutil.which("clang++")
    if gxx is None:
        pytest.skip("no host compiler")
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(where / "parts.cpp"),
                    "-o", str(where / "parts.so")], check=True)
    lib = ctypes.CDLL(str(where / "parts.so"))

    def length(tiles, items, groups=512, least=4, search=True):
        counted = ctypes.c_uint(0)
        got = lib.part_length((ctypes.c_uint * len(tiles))(*tiles), len(tiles), items, groups, least, int(search),
                              ctypes.byref(counted))
        assert counted.value <= 16
        return got

    return length


def parts(tiles, items, part):
    return items * sum(-(-t // part) for t in tiles)


def check(rule, tiles, items, groups=512, least=4, search=True):
    total, live = items * sum(tiles), items * sum(t > 0 for t in tiles)
    each = total // groups
    got = rule(tiles, items, groups, least, search)
    n = parts(tiles, items, got)
    assert got >= max(least, 1) and n <= groups + live      # what the workspace holds
    most = each + (max(48, each // 6 + 4) if search else max(24, each // 6 + 4))
    if search:
        if parts(tiles, items, max(most, least)) <= groups:
            assert n <= groups, (tiles, items, got, n)
            # and none six tiles shorter would do, where an even cut is not little longer than a share
            if got - 6 > each and got - 6 >= least and got > each + min(24, each // 6 + 4):
                assert parts(tiles, items, got - 6) > groups, (tiles, items, got)
        else:
            assert got == max(each + 24, least)
    else:
        if live < groups and -(-total // (groups - live)) <= most:
            assert n <= groups, (tiles, items, got, n)
    return got


@pytest.mark.parametrize("tiles,items", [([4096, 3704], 32), ([4096, 3615, 1498, 1587], 16), ([40000, 39000], 8)])
def test_long_parts_run_at_once(rule, tiles, items):
    """Two contexts of 131072 and 118528 keys with 32 key heads (and others): one part more than runs at once takes nearly
    another pass."""
    got = check(rule, tiles, items)
    assert parts(tiles, items, got) <= 512 and got <= 1.17 * items * sum(tiles) / 512 + 48


@pytest.mark.parametrize("most", [3, 30, 130, 1000, 4096, 60000])
def test_any_lengths(rule, most):
    r = random.Random(most)
    for _ in range(1500):
        n = r.choice([1, 2, 3, 4, 8, 17, 64])
        tiles = [r.choice([0, r.randint(1, most), r.randint(most // 2 + 1, most), most]) for _ in range(n)]
        items = r.choice([1, 2, 4, 8, 16, 32])
        if sum(tiles) * items >= 2 ** 31:
            continue
        check(rule, tiles, items, r.choice([512, 512, 1024, 16]), r.choice([4, 8]), r.random() < 0.8)


def test_no_keys(rule):
    assert check(rule, [0, 0], 8) >= 1 and check(rule, [0] * 64, 1, search=False) >= 1
