"""The 8-bit operators' and the log probabilities' refusals, on the CPU: bad
arguments fail before any device work, with the reason in nncu_last_error."""
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


def at(i):  # aligned addresses that are never read: every call here is refused (or has nothing to do)
    return (i + 1) << 24


ROWS = dict(n=4, cols=100, x=at(0), codes=at(1), scales=at(2), gamma=at(3), norm=1, code_stride=112)
LOOKUP = dict(n=4, cols=100, n_rows=9, codes=at(0), scales=at(1), out=at(2), ids=at(3), code_stride=112)
LINEAR = dict(n_tok=4, rows=50, cols=100, x=at(0), x_scales=at(1), w=at(2), w_scales=at(3), y=at(4), bias=at(5),
              add=at(6), x_stride=112, w_stride=112)
LOGPROBS = dict(n=4, n_vocab=100, logits=at(0), tokens=at(1), logprob=at(2), rank=at(3), entropy=at(4), top=5,
                top_ids=at(5), top_logprobs=at(6))


def refused(rc, L, text):
    assert rc == N.ERR_INVALID_ARGUMENT
    assert text in L.nncu_last_error().decode(), L.nncu_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(n=-1), "n or cols"), (dict(cols=0), "n or cols"), (dict(cols=(1 << 24) + 1), "cols"), (dict(x_type=3), "x_type"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(x=None), "NULL"), (dict(codes=None), "NULL"), (dict(scales=None), "NULL"),
    (dict(x=at(0) + 2), "aligned"), (dict(x=at(0) + 1, x_type=N.KV_BF16), "aligned"), (dict(gamma=at(3) + 2), "aligned"),
    (dict(codes=at(1) + 8), "16-byte"), (dict(code_stride=104), "16-byte"), (dict(code_stride=96), "strides"),
    (dict(x_stride=99), "strides"), (dict(x_stride=1 << 60), "strides"), (dict(codes=at(0)), "meet"),
    (dict(scales=at(1) + 16), "meet"), (dict(scales=at(3)), "meet"),
])
def test_quantise_refuses(L, change, text):
    refused(L.nncu_i8_quantise_dev(N.i8_rows(**{**ROWS, **change}), None), L, text)


@pytest.mark.parametrize("change,text", [
    (dict(n=-1), "bad n"), (dict(cols=0), "cols"), (dict(cols=(1 << 24) + 1), "cols"), (dict(n_rows=0), "n_rows"), (dict(mult=float("inf")), "mult"),
    (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(out=None), "NULL"), (dict(ids=at(3) + 1), "aligned"),
    (dict(out=at(2) + 2), "aligned"), (dict(codes=at(0) + 4), "16-byte"), (dict(code_stride=100), "16-byte"),
    (dict(code_stride=96), "strides"), (dict(out_stride=99), "strides"), (dict(out_stride=1 << 61), "strides"),
    (dict(out=at(0) + 800), "meet"), (dict(out=at(3)), "meet"), (dict(ids=None, n=10), "ids"),
])
def test_lookup_refuses(L, change, text):
    refused(L.nncu_i8_lookup_dev(N.i8_lookup(**{**LOOKUP, **change}), None), L, text)


@pytest.mark.parametrize("change,text", [
    (dict(n_tok=-1), "n_tok"), (dict(rows=0), "rows"), (dict(rows=(1 << 30) + 1, n_tok=1), "rows"),
    (dict(n_tok=(1 << 30) + 1, rows=1), "n_tok"), (dict(cols=0), "cols"), (dict(cols=131072), "cols"),
    (dict(n_tok=1 << 30, rows=1 << 10), "2^36"), (dict(x=None), "NULL"), (dict(w=None), "NULL"),
    (dict(y=None), "NULL"), (dict(x_scales=None), "NULL"), (dict(w_scales=None), "NULL"),
    (dict(x=at(0) + 8), "16-byte"), (dict(w=at(2) + 1), "16-byte"), (dict(x_stride=100), "16-byte"),
    (dict(w_stride=104), "16-byte"), (dict(x_stride=96), "strides"), (dict(w_stride=96), "strides"),
    (dict(y_stride=49), "strides"), (dict(add_stride=49), "strides"), (dict(w_stride=1 << 60), "strides"),
    (dict(y=at(4) + 2), "aligned"), (dict(bias=at(5) + 1), "aligned"), (dict(add=at(6) + 2), "aligned"),
    (dict(y=at(0)), "meet"), (dict(y=at(1) - 16), "meet"), (dict(y=at(5)), "meet"), (dict(add=at(4) + 4), "meet"),
    (dict(add=at(4), add_stride=52), "meet"),
])
def test_linear_refuses(L, change, text):
    refused(L.nncu_i8_linear_dev(N.i8_linear(**{**LINEAR, **change}), None), L, text)


@pytest.mark.parametrize("change,text", [
    (dict(n=-1), "bad n"), (dict(n_vocab=0), "n_vocab"), (dict(n_vocab=(1 << 30) + 1), "n_vocab"), (dict(top=33), "top"), (dict(top=-1), "top"),
    (dict(top=5, n_vocab=4), "top"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(logits=None), "logits"),
    (dict(tokens=None), "tokens"), (dict(tokens=None, logprob=None), "tokens"),
    (dict(logprob=None, rank=None, entropy=None, top=0), "output"), (dict(stride=99), "stride"),
    (dict(stride=1 << 60), "stride"), (dict(logits=at(0) + 2), "aligned"), (dict(rank=at(3) + 1), "aligned"),
    (dict(logprob=at(0) + 400), "meet"), (dict(rank=at(2)), "meet"), (dict(top_ids=at(6) + 40), "meet"),
])
def test_logprobs_refuses(L, change, text):
    refused(L.nncu_logprobs_dev(N.logprobs(**{**LOGPROBS, **change}), None), L, text)


def test_nothing_to_do_is_no_error(L):
    assert L.nncu_i8_quantise_dev(N.i8_rows(**{**ROWS, "n": 0, "x": None}), None) == 0
    assert L.nncu_i8_lookup_dev(N.i8_lookup(**{**LOOKUP, "n": 0}), None) == 0
    assert L.nncu_i8_linear_dev(N.i8_linear(**{**LINEAR, "n_tok": 0, "x": None}), None) == 0
    assert L.nncu_logprobs_dev(N.logprobs(**{**LOGPROBS, "n": 0, "logits": None}), None) == 0


def test_null_structs_are_refused(L):
    for f in (L.nncu_i8_quantise_dev, L.nncu_i8_lookup_dev, L.nncu_i8_linear_dev, L.nncu_logprobs_dev):
        refused(f(None, None), L, "NULL")


def test_host_tensors_and_other_types_are_refused():
    torch = pytest.importorskip("torch")
    z = torch.zeros
    with pytest.raises(ValueError, match="GPU"):
        N.i8_rows(**{**ROWS, "x": z(4, 100)})
    with pytest.raises(ValueError, match="not torch.float64"):
        N.i8_rows(**{**ROWS, "x": z(4, 100, dtype=torch.float64)})
    with pytest.raises(ValueError, match="int8"):
        N.i8_linear(**{**LINEAR, "w": z(50, 112)})
    with pytest.raises(ValueError, match="int32"):
        N.logprobs(**{**LOGPROBS, "tokens": z(4, dtype=torch.int64)})
    with pytest.raises(ValueError, match="float32"):
        N.logprobs(**{**LOGPROBS, "logits": z(4, 100, dtype=torch.bfloat16)})
