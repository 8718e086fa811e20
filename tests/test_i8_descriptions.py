"""What the descriptions of the 8-bit operators and the log probabilities refuse
of tensors, on the CPU: memory that a call would reach past its end, rows that
it would read or write in another layout."""
from __future__ import annotations

import numpy as np
import pytest

import libllmcpu_b200 as N


class Device:
    type = "cuda"

    def __eq__(self, other):
        return isinstance(other, Device)


class Tensor:
    """As much of a GPU tensor as a description looks at, over memory of its own or another one's."""

    def __init__(self, *shape, dtype="float32", stride=None, memory=None, offset=0):
        self.shape, self.ndim, self.device = shape, len(shape), Device()
        self.dtype = f"torch.{dtype}"
        self.size = {"int8": 1, "bfloat16": 2, "float16": 2}.get(dtype, 4)
        dense = [int(np.prod(shape[i + 1:])) for i in range(len(shape))]
        self.strides = tuple(dense if stride is None else stride)
        ends = [(n - 1) * s for n, s in zip(shape, self.strides)]
        self.memory = self.size * (offset + sum(ends) + 1) if memory is None else memory
        self.offset = offset

    def stride(self, i):
        return self.strides[i]

    def __getitem__(self, i):
        assert i == 0
        return Tensor(*self.shape[1:], dtype=self.dtype.rpartition(".")[2], stride=self.strides[1:], memory=self.memory,
                      offset=self.offset)

    def numel(self):
        return int(np.prod(self.shape))

    def element_size(self):
        return self.size

    def storage_offset(self):
        return self.offset

    def untyped_storage(self):
        return self

    def nbytes(self):
        return self.memory

    def data_ptr(self):
        return 1 << 24


def floats(*shape, **kw):
    return Tensor(*shape, **kw)


def whole(*shape, **kw):
    return Tensor(*shape, dtype="int32", **kw)


def codes(*shape, **kw):
    return Tensor(*shape, dtype="int8", **kw)


def rows(**kw):
    return N.i8_rows(**{**dict(n=4, cols=100, x=floats(4, 100), codes=codes(4, 112), scales=floats(4)), **kw})


# ---- the type of x ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,own", [("float32", N.KV_F32), ("bfloat16", N.KV_BF16), ("float16", N.KV_F16)])
def test_a_tensor_says_its_type(dtype, own):
    x = floats(4, 100, dtype=dtype)
    assert rows(x=x).x_type == own and rows(x=x, x_type=own).x_type == own
    for other in {N.KV_F32, N.KV_BF16, N.KV_F16} - {own}:  # (16-bit rows read as floats would be twice as long)
        with pytest.raises(ValueError, match="x_type"):
            rows(x=x, x_type=other)


def test_a_pointer_does_not():
    assert rows(x=1 << 24).x_type == N.KV_F32
    assert rows(x=1 << 24, x_type=N.KV_BF16).x_type == N.KV_BF16


# ---- arrays without a stride -------------------------------------------------------------------

def report(**kw):
    return N.logprobs(**{**dict(n=6, n_vocab=100, logits=floats(6, 100), tokens=whole(6), logprob=floats(6), rank=whole(6),
                                entropy=floats(6), top=5, top_ids=whole(6, 5), top_logprobs=floats(6, 5)), **kw})


@pytest.mark.parametrize("name,make", [("top_ids", whole), ("top_logprobs", floats)])
def test_rows_of_alternatives_are_as_long_as_asked(name, make):
    for shape in ((6, 5), (9, 5), (30,), (2, 3, 5), (40,)):
        report(**{name: make(*shape)})
    for shape in ((6, 32), (6, 6), (2, 3, 32), (30, 2)):  # rows would be written 5 apart into longer ones
        with pytest.raises(ValueError, match=name):
            report(**{name: make(*shape)})
    with pytest.raises(ValueError, match=name):
        report(**{name: make(6, 4)})
    report(**{name: make(6, 32)}, top=0)  # none are written
    report(n=1, **{name: make(6, 32)})  # one row: at its place
    report(top=1, top_ids=whole(2, 3), top_logprobs=floats(6, 1))
    with pytest.raises(ValueError, match=name):
        report(top=1, **{"top_ids": whole(6, 1), "top_logprobs": floats(6, 1), name: make(2, 3, 32)})


@pytest.mark.parametrize("name,make", [("tokens", whole), ("rank", whole), ("logprob", floats), ("entropy", floats)])
def test_vectors_lie_side_by_side(name, make):
    for shape in ((6,), (9,), (6, 1), (1, 6), (2, 3), (3, 3)):
        report(**{name: make(*shape)})
    for shape in ((6, 2), (7, 32)):
        with pytest.raises(ValueError, match=name):
            report(**{name: make(*shape)})


# ---- rows -----------------------------------------------------------------------------------------

def lookup(**kw):
    return N.i8_lookup(**{**dict(n=6, cols=100, n_rows=9, codes=codes(9, 112), scales=floats(9), out=floats(6, 100)), **kw})


def linear(**kw):
    return N.i8_linear(**{**dict(n_tok=6, rows=50, cols=100, x=codes(6, 112), x_scales=floats(6), w=codes(50, 112),
                                 w_scales=floats(50), y=floats(6, 50), bias=floats(50), add=floats(6, 50)), **kw})


# (an array of rows, its stride's field, how it is made, rows, values of a row)
ROW_ARRAYS = [(rows, "x", "x_stride", floats, 4, 100), (rows, "codes", "code_stride", codes, 4, 112),
              (lookup, "codes", "code_stride", codes, 9, 112), (lookup, "out", "out_stride", floats, 6, 100),
              (linear, "x", "x_stride", codes, 6, 112), (linear, "w", "w_stride", codes, 50, 112),
              (linear, "y", "y_stride", floats, 6, 50), (linear, "add", "add_stride", floats, 6, 50),
              (report, "logits", "stride", floats, 6, 100)]


@pytest.mark.parametrize("call,name,field,make,n,row", ROW_ARRAYS)
def test_rows_of_more_dimensions(call, name, field, make, n, row):
    given = lambda t: getattr(call(**{name: t}), field)  # noqa: E731
    assert given(make(n, row)) == row and given(make(n + 3, row + 48)) == row + 48
    assert given(make(1, n, row)) == row and given(make(1, 1, n, row)) == row  # a batch of one
    assert given(make(1, n, row + 48)) == row + 48
    assert given(make(n, 2, row // 2)) == row  # heads
    # (a batch's rows would be read as far apart as its prompts are, past their end)
    for shape in ((n // 2 + 1, 2, row), (n - 1, 3, row), (1, n - 1, row), (1, n, row // 4), (1, 1, n * row)):
        with pytest.raises(ValueError, match=f"^{name}:"):
            call(**{name: make(*shape)})


@pytest.mark.parametrize("call,name,field,make,n,row", ROW_ARRAYS)
def test_rows_end_within_their_memory(call, name, field, make, n, row):
    used = 100 if row == 112 else row  # (what a call reads of a row of codes)
    wide = row + 16
    call(**{name: make((n - 1) * wide + used), field: wide})
    call(**{name: make(n, row, stride=(wide, 1))})
    call(**{name: make(n, used, stride=(row, 1)), field: row})
    call(**{name: make(n, row, offset=5, memory=make(1).size * (5 + (n - 1) * wide + used)), field: wide})
    for bad in (make((n - 1) * wide + used - 1), make(n, row), make(n * row),
                make(n, row, offset=6, memory=make(1).size * (5 + (n - 1) * wide + used))):
        with pytest.raises(ValueError, match=f"^{name}: .*{field} of {wide}"):
            call(**{name: bad, field: wide})
