"""Kernels that begin while the one before them on the stream ends, on the CPU:
what such a kernel reads may still be written when it begins, so that its source
holds no non-coherent load (which asks for memory that is read-only for the
whole life of the kernel)."""
from __future__ import annotations

import glob
import os
import re

import pytest

from libllmcpu_b200 import build


def code(path):
    """The source without its comments."""
    with open(path) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


SOURCES = {os.path.basename(p): code(p) for p in glob.glob(os.path.join(build.CSRC, "*.cu*"))}
DEPENDENT = sorted(n for n, s in SOURCES.items() if n.endswith(".cu") and "griddep_wait()" in s)
HEADERS = sorted(n for n in SOURCES if n.endswith(".cuh"))


def test_the_dependent_kernels_are_found():
    assert {"k_decode.cu", "k_decode_tc.cu", "k_i8.cu", "k_i8_linear.cu", "k_logprobs.cu"} <= set(DEPENDENT)


@pytest.mark.parametrize("name", DEPENDENT + HEADERS)
def test_no_non_coherent_loads(name):
    assert not re.findall(r"__ldg\w*|\bld\.global(?:\.\w+)*\.nc\b", SOURCES[name])


@pytest.mark.parametrize("name", DEPENDENT)
def test_no_promise_that_would_allow_them(name):
    """(A const __restrict__ argument of a kernel lets the compiler take such loads.)"""
    assert "__restrict__" not in SOURCES[name]
