"""The planning of prompts' attention over the 4-bit cache, on the CPU: the
length of a piece, and that pieces and their partial results fit their arrays."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from libllmcpu_b200 import build

SHARES, MIN_PIECE = 296, 8

MAIN = r'''
#include <cstdio>
#include "kv4_plan.h"
int main()
{
	long long total;
	int n_kv;
	while (scanf("%lld %d", &total, &n_kv) == 2) printf("%d\n", nncu::kv4_longest(total, n_kv));
}
'''

# (blocks, tiles of a block, KV heads): one block, a prompt, a long chunk, a batch, then two million new tokens with 16
# heads a KV head over a context as long (2^32 tiles), and the most that a call can ask for
CASES = [(1, 1, 8), (32, 64, 8), (8, 250, 4), (700, 33, 2), (5, 3000, 1), (1, 1 << 21, 700), (1 << 18, 1 << 14, 8),
         (1 << 22, 1 << 25, 256)]


@pytest.fixture(scope="module")
def longest(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("plan")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run([gxx, "-std=c++17", f"-I{build.CSRC}", str(d / "main.cpp"), "-o", str(d / "plan")], check=True)
    given = "".join(f"{b * t} {kv}\n" for b, t, kv in CASES)
    r = subprocess.run([str(d / "plan")], input=given, capture_output=True, text=True, check=True)
    return dict(zip(CASES, map(int, r.stdout.split())))


@pytest.mark.parametrize("case", CASES)
def test_pieces_fit(longest, case):
    blocks, tiles, n_kv = case
    most = longest[case]
    assert most == min(max(MIN_PIECE, -(-blocks * tiles * n_kv // SHARES)), 2 ** 31 - 1)
    pieces = -(-tiles // most)
    assert blocks * pieces <= blocks + SHARES
    if pieces > 1:
        assert blocks * pieces * n_kv <= 2 * SHARES  # partial results
    each = -(-tiles // pieces)
    assert tiles - (pieces - 1) * each > 0  # the last piece has tiles too
