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
