"""The plans of the 8-bit products and of the log probabilities, on the CPU:
each call of variants.py goes to the kernel that it is there for, and every plan
is one that its kernel can run."""
from __future__ import annotations

import random
import shutil
import subprocess

import pytest

import variants as V
from libllmcpu_b200 import build

MAIN = r'''
#include <cstdio>
#include "i8_plan.h"
#include "logprobs_plan.h"
using namespace nncu;
int main()
{
	char what;
	int a, b, c;
	while (scanf(" %c %d %d %d", &what, &a, &b, &c) == 4)
		if (what == 'i')
		{
			const I8Plan p = i8_plan(a, b, c);
			printf("%d %d %d %d %d %d %d %d\n", (int)p.pair, p.bn, p.split, p.panels, p.tiles_o, p.tiles_t, i8_stages(p), i8_smem(p));
		}
		else
		{
			const LpPlan p = lp_plan(a, b, c > 0);
			printf("%d %d %d\n", p.wide ? LP_WIDE : LP_NARROW, (int)p.ahead, p.parts);
		}
}
'''


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("plans")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run([gxx, "-std=c++17", "-O1", f"-I{build.CSRC}", str(d / "main.cpp"), "-o", str(d / "plans")], check=True)

    def run(what, calls):
        given = "".join(f"{what} %d %d %d\n" % c for c in calls)
        r = subprocess.run([str(d / "plans")], input=given, capture_output=True, text=True, check=True)
        return [tuple(map(int, line.split())) for line in r.stdout.splitlines()]

    return run


def test_each_product_takes_its_variant(plans):
    for case, (pair, bn, split, panels, tiles_o, tiles_t, _, _) in zip(V.LINEAR, plans("i", [c[:3] for c in V.LINEAR])):
        assert (pair, bn, split, panels, tiles_o * tiles_t) == case[6:], case


def test_the_pairs_cases_reach_what_they_are_for(plans):
    """74 pairs: three tiles and more of one pair, with and without what is added; several tiles of tokens under more than
    32 tiles of channels; tiles of fewer stages than the ring has, and of more."""
    got = list(zip(V.LINEAR, plans("i", [c[:3] for c in V.LINEAR])))
    walks = [(c, p) for c, p in got if p[0] and p[4] * p[5] > 2 * 74]
    assert {bool(c[4]) for c, _ in walks} == {False, True} and {bool(c[3]) for c, _ in walks} == {False, True}
    assert {p[3] for _, p in walks} == {1, 2}
    assert any(p[4] > 32 and p[4] % 32 and p[5] > 1 for _, p in walks)
    stages = [(-(-c[2] // (128 * p[3])), p[6]) for c, p in walks]
    assert any(n < ring for n, ring in stages) and any(n > ring and n % ring for n, ring in stages)
    splits = {(p[0], p[2]) for _, p in got}
    assert splits >= {(1, s) for s in (1, 2, 3, 4)} | {(0, s) for s in (1, 2, 3, 4, 6, 8)}


def test_the_other_products_take_theirs(plans):
    assert [p[0] for p in plans("i", [(n, r, 131071) for n, r, _ in V.LARGEST])] == [k for _, _, k in V.LARGEST]
    assert [p[0] for p in plans("i", [(b - a, *V.BATCH) for a, b, _ in V.SLICES])] == [k for _, _, k in V.SLICES]
    assert [p[0] for p in plans("i", [(n, *V.TOGETHER) for n, _ in V.TOKENS])] == [k for _, k in V.TOKENS]


def test_each_row_of_logits_takes_its_variant(plans):
    for case, plan in zip(V.LOGPROBS, plans("l", [c[:3] for c in V.LOGPROBS])):
        assert plan == case[3:], case
        assert case[1] // (plan[2] * plan[0] * 16) >= V.GROUPS - 1, case  # (the last one may be cut)


def test_every_variant_of_the_log_probabilities_has_a_case(plans):
    rng = random.Random(1)
    calls = [(int(2100 ** rng.random()), int(2000 * 150 ** rng.random()), rng.randint(0, 1)) for _ in range(40000)]
    reached = {(bool(c[2]), *p) for c, p in zip(calls, plans("l", calls))}
    assert reached <= {(bool(c[2]), *c[3:]) for c in V.LOGPROBS}


def test_every_plan_can_be_run(plans):
    """Stages to load while others are read, memory that a CTA may ask for, sizes that the tensor cores take, a share of
    the columns for each that splits them."""
    rng = random.Random(2)
    calls = [(int((1 << 20) ** rng.random()), int((1 << 20) ** rng.random()), int(131071 ** rng.random())) for _ in range(40000)]
    calls += [(1 << 30, 1, 1), (1, 1 << 30, 131071), (1 << 30, 64, 131071), (64, 1 << 30, 1)]
    for (n, r, c), (pair, bn, split, panels, tiles_o, tiles_t, stages, smem) in zip(calls, plans("i", calls)):
        assert 16 <= bn <= 256 and bn % (32 if pair else 16) == 0 and tiles_t == -(-n // bn)
        assert tiles_o == -(-r // (256 if pair else 128)) and panels in (1, 2)
        assert panels + 1 <= stages <= 12 and smem <= 216 * 1024
        assert 1 <= split <= (4 if pair else 8) and split * panels <= -(-c // 128)
