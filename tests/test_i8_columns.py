"""Arrays whose rows lie between one another's, columns of one buffer: taken where
no byte is in common, on the CPU (a call that is not refused comes as far as the
device)."""
from __future__ import annotations

import os

import pytest

import libllmcpu_b200 as N
from libllmcpu_b200 import build


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(N.LIB_PATH):
        build.build()
    return N.lib()


BASE = 1 << 24


def at(i):
    return (i + 2) << 24


def meets(rc, L):
    text = L.nncu_last_error().decode()
    assert rc != 0  # (no device, or addresses that are none)
    if rc != N.ERR_INVALID_ARGUMENT:
        return False
    assert "meet" in text or "device memory" in text, text
    return "meet" in text


def linear(L, n=5, rows=40, **kw):
    d = dict(n_tok=n, rows=rows, cols=16, x=at(0), x_scales=at(1), w=at(2), w_scales=at(3), y=BASE, y_stride=100)
    return meets(L.nncu_i8_linear_dev(N.i8_linear(**{**d, **kw}), None), L)


@pytest.mark.parametrize("place,met", [(40, False), (60, False), (50, False), (39, True), (61, True), (0, True), (99, True),
                                       (140, False), (139, True), (-60, False), (-61, True), (-59, False), (-39, True), (240, False)])
def test_what_is_added_beside_y(L, place, met):
    """y: columns 0 to 40 of rows of 100 floats, add: 40 columns from `place` on."""
    assert linear(L, add=BASE + 4 * place, add_stride=100) == (met and place != 0)  # (add may be y)


def test_other_distances_and_single_rows(L):
    assert linear(L, add=BASE + 160, add_stride=101)  # somewhere they meet, for all that is known
    assert not linear(L, n=1, add=BASE + 160)  # one row behind the other
    assert linear(L, n=1, add=BASE + 156)
    assert not linear(L, bias=BASE + 4 * 140)  # a row between two rows of y
    assert linear(L, bias=BASE + 4 * 161)  # ... and into the next one
    assert linear(L, w_scales=BASE + 4 * 30)
    # codes between rows of y: 64 of 400 bytes
    assert not linear(L, x=BASE + 160, x_stride=400)
    assert linear(L, x=BASE + 144, x_stride=400)


def test_rows_out_between_others(L):
    look = dict(n=5, cols=40, n_rows=5, codes=BASE + 160, code_stride=400, scales=at(1), ids=at(2), out=BASE, out_stride=100)
    assert not meets(L.nncu_i8_lookup_dev(N.i8_lookup(**look), None), L)
    assert meets(L.nncu_i8_lookup_dev(N.i8_lookup(**{**look, "codes": BASE + 368}), None), L)  # into the next row
    rows = dict(n=5, cols=40, x=BASE, x_stride=100, codes=BASE + 160, code_stride=400, scales=at(1))
    assert not meets(L.nncu_i8_quantise_dev(N.i8_rows(**rows), None), L)
    assert meets(L.nncu_i8_quantise_dev(N.i8_rows(**{**rows, "codes": BASE + 144}), None), L)
    assert meets(L.nncu_i8_quantise_dev(N.i8_rows(**{**rows, "scales": BASE + 200}), None), L)  # side by side: into a row
