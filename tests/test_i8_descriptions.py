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
