"""The paged operators' refusals, on the CPU: bad arguments fail before any
device work, with the reason in nncu_last_error."""
from __future__ import annotations

import os

import numpy as np
import pytest

import libllmcpu_b200 as N
from libllmcpu_b200 import build


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(N.LIB_PATH):
        build.build()
    return N.lib()


A = 1 << 20  # an aligned address that is never read: every call here is refused (or has nothing to do)
STEP = dict(n_req=4, page_size=16, n_pages=8, max_blocks=4, max_tok=8, past=A, n_new=A, held=A, queue=A, ring=A,
            block_table=A, held_out=A + 64, queue_out=A + 64, seq_len=A, q_start=A, positions=A, slots=A, token_req=A)
ROPE = dict(n_tok=2, n_head=4, n_kv=2, head_dim=128, positions=A, inv_freq=A, q=A, k=A)
POOL = dict(pages=A, n_pages=8, page_size=64, n_kv=2, head_dim=128)
ROWS = dict(slots=A, n_tok=2, k=A, v=A)
ATTN = dict(n_req=2, n_tok=2, n_head=8, max_new=1, max_blocks=4, block_table=A, seq_len=A, q_start=A, q=A, out=A,
            workspace=A, workspace_bytes=1 << 40)


def refused(rc, L, text):
    assert rc == N.ERR_INVALID_ARGUMENT
    assert text in L.nncu_last_error().decode(), L.nncu_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(n_req=0), "n_req"), (dict(n_req=8193), "n_req"), (dict(page_size=0), "page_size"),
    (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 28), "n_pages"), (dict(max_tok=-1), "max_tok"),
    (dict(table_stride=3), "table"), (dict(past=None), "NULL"), (dict(ring=None), "NULL"), (dict(slots=None), "NULL"),
    (dict(held_out=A), "must not be"), (dict(queue_out=A), "must not be"),
])
def test_step_refuses(L, change, text):
    refused(L.nncu_paged_step_dev(N.paged_step(**{**STEP, **change}), None), L, text)


@pytest.mark.parametrize("change,text", [
    (dict(n_tok=-1), "n_tok"), (dict(q=None, k=None), "no rows"), (dict(head_dim=127), "head_dim"),
    (dict(head_dim=1024), "head_dim"), (dict(n_rot=130), "n_rot"), (dict(n_rot=63), "n_rot"),
    (dict(rope_mode=2), "mode"), (dict(sections=[10, 20]), "sections"), (dict(sections=[-4, 68]), "section"),
    (dict(sections=[10, 54], interleaved=1), "interleaved"), (dict(positions=None), "NULL"),
    (dict(inv_freq=None), "NULL"), (dict(q_stride=100), "strides"), (dict(q_stride=600), "two strides"),
    (dict(sections=[32, 32], pos_stride=1), "pos_stride"), (dict(sections=[64, 0, 0, 0, 0]), "axes"),
])
def test_rope_axes_refuses(L, change, text):
    refused(L.nncu_rope_axes_dev(N.rope_axes(**{**ROPE, **change}), None), L, text)


@pytest.mark.parametrize("change,text", [
    (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
    (dict(page_size=512), "page_size"), (dict(n_pages=0), "n_pages"), (dict(n_kv=0), "n_kv"),
    (dict(n_pages=1 << 26), "n_pages"), (dict(pages=None), "pages"), (dict(pages=A + 8), "aligned"),
])
def test_pool_is_checked(L, change, text):
    pool = N.kv4_pool(**{**POOL, **change})
    refused(L.nncu_kv4_append_dev(N.kv4_rows(pool, **ROWS), None), L, text)
    refused(L.nncu_kv4_read_dev(N.kv4_rows(pool, **ROWS), None), L, text)
    attn = dict(ATTN, n_head=4 * max(pool.n_kv, 1))
    refused(L.nncu_kv4_attention_dev(N.kv4_attn(pool, **attn), None), L, text)


@pytest.mark.parametrize("change,text", [
    (dict(n_tok=-1), "n_tok"), (dict(slots=None), "NULL"), (dict(k=None, v=None), "NULL"), (dict(k=A + 4), "aligned"),
    (dict(v_stride=258), "aligned"), (dict(k_stride=128), "strides"),
])
def test_rows_are_checked(L, change, text):
    rows = N.kv4_rows(N.kv4_pool(**POOL), **{**ROWS, **change})
    refused(L.nncu_kv4_append_dev(rows, None), L, text)
    refused(L.nncu_kv4_read_dev(rows, None), L, text)


@pytest.mark.parametrize("change,text", [
    (dict(n_req=-1), "n_req"), (dict(max_new=-1), "max_new"), (dict(window=-1), "window"), (dict(n_head=7), "n_head"),
    (dict(n_head=0), "n_head"), (dict(max_blocks=1 << 26), "max_blocks"), (dict(table_stride=3), "table"),
    (dict(block_table=None), "NULL"), (dict(q=None), "NULL"), (dict(q=A + 4), "aligned"),
    (dict(out_stride=1026), "aligned"), (dict(q_stride=512), "strides"), (dict(softcap=-1.0), "softcap"),
    (dict(scale=float("nan")), "scale"), (dict(n_tok=1 << 30), "2^31"), (dict(n_req=2000000000), "2^31"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=16), "workspace"),
    (dict(workspace=A + 8), "workspace"),
])
def test_attention_refuses(L, change, text):
    refused(L.nncu_kv4_attention_dev(N.kv4_attn(N.kv4_pool(**POOL), **{**ATTN, **change}), None), L, text)


def test_nothing_to_do_is_no_error(L):
    assert L.nncu_rope_axes_dev(N.rope_axes(**{**ROPE, "n_tok": 0}), None) == 0
    assert L.nncu_kv4_append_dev(N.kv4_rows(N.kv4_pool(**POOL), **{**ROWS, "n_tok": 0}), None) == 0
    for change in (dict(n_req=0), dict(n_tok=0), dict(max_new=0)):
        assert L.nncu_kv4_attention_dev(N.kv4_attn(N.kv4_pool(**POOL), **{**ATTN, **change}), None) == 0


def test_null_structs_are_refused(L):
    for f in (L.nncu_paged_step_dev, L.nncu_rope_axes_dev, L.nncu_kv4_append_dev, L.nncu_kv4_read_dev,
              L.nncu_kv4_attention_dev, L.nncu_kv4_check):
        refused(f(None, None), L, "NULL")


def test_pool_bytes(L):
    # 0.5625 bytes a value, K and V
    assert N.kv4_bytes(10, 64, 8, 128) == 10 * 64 * 8 * 128 * 9 // 16 * 2
    with pytest.raises(N.NnncError):
        N.kv4_bytes(10, 64, 8, 80)


def test_strides_come_from_the_tensors():
    x = np.zeros((4, 520), np.float32)[:, :512]
    with pytest.raises(AssertionError):  # not contiguous: host arrays are refused as ever
        N.rope_axes(**{**ROPE, "q": x})
    torch = pytest.importorskip("torch")
    y = torch.zeros(4, 520)[:, :512]
    assert N.rope_axes(**{**ROPE, "q": y}).q_stride == 520
    with pytest.raises(ValueError):
        N.rope_axes(**{**ROPE, "q": torch.zeros(512, 4).T})


def test_paged_bench_parses_its_arguments():
    from libllmcpu_b200 import paged_bench

    with pytest.raises(SystemExit) as e:
        paged_bench.main(["--help"])
    assert e.value.code == 0
