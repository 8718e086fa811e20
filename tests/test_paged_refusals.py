"""More of the paged operators' refusals, on the CPU: arrays that meet, scales
and sizes that no kernel can serve, tensors that are not what a call reads."""
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


A, GAP = 1 << 20, 4096  # addresses that are never read: every call here is refused


def refused(rc, L, text):
    assert rc == N.ERR_INVALID_ARGUMENT
    assert text in L.nncu_last_error().decode(), L.nncu_last_error()


ARRAYS = ("past", "n_new", "held", "queue", "ring", "block_table", "held_out", "queue_out", "seq_len", "q_start",
          "positions", "slots", "token_req")
WRITTEN = ("held_out", "queue_out", "seq_len", "q_start", "positions", "slots", "token_req")


def step(**change):
    at = {name: A + i * GAP for i, name in enumerate(ARRAYS)}
    return N.paged_step(**{**dict(n_req=4, page_size=16, n_pages=8, max_blocks=4, max_tok=8), **at, **change}), at


def meets(L, **change):
    refused(L.nncu_paged_step_dev(step(**change)[0], None), L, "must not")


@pytest.mark.parametrize("out", WRITTEN)
@pytest.mark.parametrize("other", ARRAYS)
def test_step_arrays_must_not_be_one(L, out, other):
    if out != other:
        meets(L, **{out: step()[1][other]})


def test_step_arrays_must_not_meet(L):
    at = step()[1]
    meets(L, ring=at["past"] + 12)         # the ring's first entry is past's last
    meets(L, seq_len=at["n_new"] - 12)     # the last of seq_len is n_new's first
    meets(L, q_start=at["held_out"] - 16)  # (n_req + 1 entries)
    meets(L, queue_out=at["queue"] - 12)
    meets(L, queue=at["slots"] + 28)
    # rows of 4 entries, 16 apart: in the second row, into the third from before it, before the table
    for p in (16 * 4 + 8, 2 * 16 * 4 - 4, -4):
        meets(L, table_stride=16, held=at["block_table"] + p)


POOL = dict(pages=A, n_pages=8, page_size=64, n_kv=2, head_dim=128)
ATTN = dict(n_req=2, n_tok=2, n_head=8, max_new=1, max_blocks=4, block_table=A, seq_len=A, q_start=A, q=A, out=A,
            workspace=A, workspace_bytes=1 << 40)


@pytest.mark.parametrize("change", [dict(scale=float("inf")), dict(scale=float("-inf")), dict(softcap=float("inf"))])
def test_attention_wants_finite_scales(L, change):
    """Their products with a score of zero are NaN."""
    refused(L.nncu_kv4_attention_dev(N.kv4_attn(N.kv4_pool(**POOL), **{**ATTN, **change}), None), L, "scale or softcap")


@pytest.mark.parametrize("n_tok", [2 ** 31 - 1, 2 ** 31 - 592])
def test_rope_axes_counts_with_32_bits(L, n_tok):
    """A CTA takes every 592nd token, and stops at the first number past the last one."""
    rope = N.rope_axes(n_tok=n_tok, n_head=1, n_kv=1, head_dim=2, positions=A, inv_freq=A, q=A, pos_stride=n_tok)
    refused(L.nncu_rope_axes_dev(rope, None), L, "n_tok")


def test_tensors_of_other_types_are_refused():
    torch = pytest.importorskip("torch")
    z = torch.zeros
    i32, rows = torch.int32, dict(n_tok=4, n_head=2, n_kv=2, head_dim=64, inv_freq=A)
    pool = N.kv4_pool(z(8, dtype=torch.uint8), 8, 64, 2, 128)
    with pytest.raises(ValueError, match="positions.*int32.*int64"):
        N.rope_axes(**rows, positions=torch.arange(4), q=A)
    with pytest.raises(ValueError, match="q: .*float32.*bfloat16"):
        N.rope_axes(**rows, positions=A, q=z(4, 128, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="slots.*int32"):
        N.kv4_rows(pool, slots=z(4), n_tok=4, k=A, v=A)
    with pytest.raises(ValueError, match="seq_len.*int32"):
        N.kv4_attn(pool, **{**ATTN, "seq_len": z(2, dtype=torch.int64)})
    with pytest.raises(ValueError, match="past.*int32"):
        step(past=z(4, dtype=torch.int64))
    with pytest.raises(TypeError, match="no_such"):
        step(no_such=A)
    assert step(past=z(4, dtype=i32))[0].past


def test_tensors_whose_values_lie_apart_are_refused():
    torch = pytest.importorskip("torch")
    z, i32 = torch.zeros, torch.int32
    rope = dict(n_tok=4, n_head=2, n_kv=2, head_dim=64, inv_freq=A)
    apart = "lie side by side"
    with pytest.raises(ValueError, match=apart):  # every other entry of a vector
        N.rope_axes(**rope, positions=z(8, dtype=i32)[::2], q=A)
    with pytest.raises(ValueError, match=apart):
        step(n_new=z(4, 2, dtype=i32)[:, 0])
    with pytest.raises(ValueError, match=apart):  # heads with a gap behind each, or in another order
        N.rope_axes(**rope, positions=A, q=z(4, 2, 80)[..., :64])
    with pytest.raises(ValueError, match=apart):
        N.rope_axes(**rope, positions=A, q=z(2, 4, 64).transpose(0, 1))
    # rows apart are served, and what has one entry lies side by side whatever its strides
    r = N.rope_axes(**rope, positions=z(4, 1, dtype=i32).T, q=z(4, 3, 64)[:, :2], k=z(8, 2, 64)[::2])
    assert (r.q_stride, r.k_stride) == (3 * 64, 2 * 2 * 64)
    r = N.rope_axes(**{**rope, "n_tok": 1}, positions=z(1, 3, dtype=i32).T, q=A, sections=[16, 8, 8])
    assert r.pos_stride == 1
