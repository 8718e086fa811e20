"""What the checks of the 8-bit products remember, on the CPU: every stream
learns of a wait that ran out, once, whichever stream is checked first."""
from __future__ import annotations

import shutil
import subprocess

import pytest

from libllmcpu_b200 import build

MAIN = r'''
#include <cstdio>
#include "i8_seen.h"
int main()
{
	nncu::I8Seen seen;
	int device;
	unsigned long long stream;
	unsigned count;
	while (scanf("%d %llu %u", &device, &stream, &count) == 3) printf("%d\n", (int)seen.more(device, stream, count));
}
'''


@pytest.fixture(scope="module")
def seen(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("seen")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run([gxx, "-std=c++17", "-pthread", f"-I{build.CSRC}", str(d / "main.cpp"), "-o", str(d / "seen")], check=True)

    def run(checks):
        given = "".join("%d %d %d\n" % c for c in checks)
        r = subprocess.run([str(d / "seen")], input=given, capture_output=True, text=True, check=True)
        return [x == "1" for x in r.stdout.split()]

    return run


# (device, stream, waits that ran out so far) of one check after another, and whether each reports
@pytest.mark.parametrize("checks,reports", [
    ([(0, 1, 0), (0, 2, 0)], [False, False]),
    # a product of stream 2 times out, stream 1 is checked first: both learn of it, once
    ([(0, 1, 0), (0, 2, 0), (0, 1, 7), (0, 2, 7), (0, 1, 7), (0, 2, 7)], [False, False, True, True, False, False]),
    # once more
    ([(0, 1, 7), (0, 1, 9), (0, 2, 9), (0, 2, 9), (0, 1, 9)], [True, True, True, False, False]),
    # devices count apart; a stream that is checked for the first time may have had them
    ([(0, 1, 3), (1, 1, 0), (1, 1, 3), (0, 1, 3), (0, 3, 3)], [True, False, True, False, True]),
])
def test_no_check_hides_a_wait_from_another(seen, checks, reports):
    assert seen(checks) == reports
