"""The paged operators at the edges of their arguments: lengths that no sum can
hold, scales of any sign, long spans, workspaces after a wait that ran out."""
from __future__ import annotations

import os
import subprocess
import sys

import numpy as np
import pytest

import paged_helpers as P

pytestmark = pytest.mark.gpu

SUM_END = (1 << 30) - 1  # where the tables' running sums stop


def dev(torch, x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=dtype, device="cuda")


class Step:
    """One paged_step call over `past`, `new`, `held`; its tables as numpy arrays."""

    def __init__(self, torch, N, past, new, held, queue, ring, table, page, max_blocks, max_tok):
        i32, n = torch.int32, len(past)
        z = lambda k: torch.full((k,), -99, dtype=i32, device="cuda")  # noqa: E731
        self.out = dict(held_out=z(n), queue_out=z(4), seq_len=z(n), q_start=z(n + 1), positions=z(max_tok),
                        slots=z(max_tok), token_req=z(max_tok))
        self.ring = dev(torch, ring, i32)
        N.paged_step_dev(N.paged_step(n_req=n, page_size=page, n_pages=len(ring), max_blocks=max_blocks,
                                      max_tok=max_tok, past=dev(torch, past, i32), n_new=dev(torch, new, i32),
                                      held=dev(torch, held, i32), queue=dev(torch, queue, i32), ring=self.ring,
                                      block_table=table, **self.out))
        torch.cuda.synchronize()

    def check_all(self, want, end=(1 << 31) - 1):
        for name, key in (("held_out", "held"), ("queue_out", "queue"), ("seq_len",) * 2, ("q_start",) * 2,
                          ("positions",) * 2, ("slots",) * 2, ("token_req",) * 2):
            np.testing.assert_array_equal(self.out[name].cpu().numpy(),
                                          np.minimum(np.asarray(want[key], np.int64), end), err_msg=name)
        np.testing.assert_array_equal(self.ring.cpu().numpy(), np.asarray(want["ring"]))

    def check(self, want):
        self.check_all(want, SUM_END)


@pytest.mark.parametrize("new", [[1 << 30, 1 << 30, 3, 2], [3, (1 << 31) - 1, (1 << 31) - 1, 5], [1 << 30] * 40 + [4]])
def test_step_of_lengths_past_any_sum(nncu, torch_cuda, new):
    """New tokens whose sum passes 2^31: nobody behind them is served, and the sums stay at their end."""
    n, page, n_pages, max_blocks, max_tok = len(new), 16, 12, 6, 40
    past, held = [5] * n, [1] * n
    table = np.arange(n * max_blocks).reshape(n, max_blocks) % n_pages
    ring = np.arange(n_pages)
    want = P.step(past, new, held, [3, 9], ring, table, page, n_pages, max_blocks, max_tok)
    Step(torch_cuda, nncu, past, new, held, [3, 9], ring, dev(torch_cuda, table, torch_cuda.int32), page, max_blocks,
         max_tok).check(want)


def test_step_of_more_lacking_pages_than_any_sum(nncu, torch_cuda):
    """1025 requests that lack 2^20 pages each, then one that lacks a single page: the sum has reached its end, but the
    ring suffices for none of them."""
    torch = torch_cuda
    n, page, max_blocks, n_pages = 1026, 16, 1 << 20, 64
    past, new, held = [(1 << 24) - 1] * (n - 1) + [0], [1] * (n - 1) + [3], [0] * n
    table = torch.empty(n, max_blocks, dtype=torch.int32, device="cuda")
    want = P.step(past, new, held, [60, 40], np.arange(n_pages), np.zeros((n, 1)), page, n_pages, max_blocks, n + 8)
    want["queue"][2] = SUM_END  # (pages that were missing)
    Step(torch, nncu, past, new, held, [60, 40], np.arange(n_pages), table, page, max_blocks, n + 8).check(want)


def test_step_of_lengths_near_the_largest(nncu, torch_cuda):
    """Pages of one token, a table of 2^31 - 1 a request: a need as large, then a small one; neither is served, and no
    entry of the table is touched."""
    torch = torch_cuda
    most, n_pages = (1 << 31) - 1, 64
    past, new, held = [most - 1, 0], [1, 3], [0, 0]
    table = torch.empty(2 * most, dtype=torch.int32, device="cuda").view(2, most)
    want = P.step(past, new, held, [5, 40], np.arange(n_pages), np.zeros((2, 4)), 1, n_pages, most, 20)
    assert want["seq_len"] == past
    want["queue"][2] = SUM_END
    Step(torch, nncu, past, new, held, [5, 40], np.arange(n_pages), table, 1, most, 20).check_all(want)
    del table
    torch.cuda.empty_cache()


def steps_of(counts):
    import torch

    import libllmcpu_b200 as N

    for n in counts:
        rng = np.random.default_rng(n)
        past, new = rng.integers(0, 60, n), rng.integers(0, 3, n)
        held = -(-past // 16)
        n_pages, max_tok = int(held.sum()) + 900, int(new.sum()) + 5
        ids, at = rng.permutation(n_pages), 0
        table = np.full((n, 5), -7)
        for r in range(n):
            table[r, :held[r]] = ids[at:at + held[r]]
            at += held[r]
        ring = np.full(n_pages, -9)
        ring[:n_pages - at] = ids[at:]
        want = P.step(past, new, held, [0, n_pages - at], ring, table, 16, n_pages, 5, max_tok)
        Step(torch, N, past, new, held, [0, n_pages - at], ring, dev(torch, table, torch.int32), 16, 5,
             max_tok).check(want)


def test_step_whose_sums_just_fill_48_kb(nncu, torch_cuda):
    """4090 to 4095 requests: their sums fill the 48 KB that a kernel has unasked, less its other shared words. In a
    process of its own, where no larger call has asked for more before."""
    here = os.path.dirname(os.path.abspath(__file__))
    code = "import test_gpu_paged_edges as t; t.steps_of([4089, 4090, 4093, 4095, 4096])"
    path = os.pathsep.join([here, os.path.dirname(here), os.environ.get("PYTHONPATH", "")])
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": path})
    assert r.returncode == 0, r.stderr[-2000:]


class Cache:
    """Requests' keys and values in a pool: random pages, written by the append, read back as the values they stand for."""

    def __init__(self, torch, N, lens, n_kv, d, page, seed=0, rise=0.0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.torch, self.N, self.lens, self.n_kv, self.d = torch, N, lens, n_kv, d
        blocks = [-(-n // page) for n in lens]
        n_pages = sum(blocks) + 3
        ids = np.random.default_rng(seed).permutation(n_pages)
        self.table = np.full((len(lens), max(blocks)), -1)
        self.kv, at = [], 0
        self.pages = torch.zeros(N.kv4_bytes(n_pages, page, n_kv, d), dtype=torch.uint8, device="cuda")
        self.pool = N.kv4_pool(self.pages, n_pages, page, n_kv, d)
        # keys along `axis` grow with their position: scores of a query that lies along it rise by `rise`
        self.axis = torch.randn(d, generator=gen, device="cuda")
        self.axis /= self.axis.norm()
        for r, n in enumerate(lens):
            self.table[r, :blocks[r]] = ids[at:at + blocks[r]]
            at += blocks[r]
            k, v = (torch.randn(n, n_kv, d, generator=gen, device="cuda") for _ in range(2))
            k += rise * torch.linspace(0, 1, n, device="cuda")[:, None, None] * self.axis
            back = [torch.zeros(n, n_kv * d, device="cuda") for _ in range(2)]
            slots = dev(torch, self.table[r, np.arange(n) // page] * page + np.arange(n) % page, torch.int32)
            N.kv4_append_dev(N.kv4_rows(self.pool, slots=slots, n_tok=n, k=k, v=v))
            N.kv4_read_dev(N.kv4_rows(self.pool, slots=slots, n_tok=n, k=back[0], v=back[1]))
            self.kv.append([x.view(n, n_kv, d).double().cpu().numpy() for x in back])
        self.vmax = max([float(np.abs(kv[1]).max()) for kv in self.kv if kv[1].size] + [0.0])

    def attn(self, new, group, scale, window=0, softcap=0.0, along=0.0, seed=1):
        """The call of `new` tokens a request; self.out has its rows, self.q its queries."""
        torch, N = self.torch, self.N
        gen = torch.Generator(device="cuda").manual_seed(seed)
        nh, n_tok, i32 = self.n_kv * group, sum(new), torch.int32
        self.group, self.new, self.args = group, new, (window, scale, softcap)
        q = torch.randn(n_tok, nh, self.d, generator=gen, device="cuda") + along * self.axis
        self.q = q.view(n_tok, nh * self.d)
        self.out = torch.full_like(self.q, 5.0)
        self.start = np.concatenate([[0], np.cumsum(new)])
        call = N.kv4_attn(self.pool, n_req=len(new), n_tok=n_tok, n_head=nh, max_new=max(new),
                          max_blocks=self.table.shape[1], block_table=dev(torch, self.table, i32),
                          seq_len=dev(torch, self.lens, i32), q_start=dev(torch, self.start, i32), q=self.q,
                          out=self.out, window=window, scale=scale, softcap=softcap)
        self.ws = torch.zeros(N.kv4_workspace_bytes(call), dtype=torch.uint8, device="cuda")
        call.workspace, call.workspace_bytes = self.ws.data_ptr(), self.ws.numel()
        return call

    def rows(self, r, tokens, heads=None):
        """(what the call gave, what the definition gives) for tokens of request r, [rows, head_dim]."""
        window, scale, softcap = self.args
        got, want = [], []
        for t in tokens:
            for h in range(self.n_kv * self.group) if heads is None else heads:
                at = (int(self.start[r]) + t, slice(h * self.d, (h + 1) * self.d))
                kv = [x[:, h // self.group] for x in self.kv[r]]
                got.append(self.out[at].double().cpu().numpy())
                want.append(P.attention(self.q[at].cpu().numpy(), *kv, self.lens[r] - self.new[r] + t, window, scale,
                                        softcap))
        return np.array(got), np.array(want)


@pytest.mark.parametrize("new", [1, 90])
def test_check_reports_and_clears(nncu, torch_cuda, new):
    """The error word that a wait which ran out leaves (written here by the host): reported once, the workspace is
    cleared, and the next call is right."""
    torch = torch_cuda
    c = Cache(torch, nncu, [2000, 1500], 2, 128, 64)
    call = c.attn([new] * 2, 4, 128 ** -0.5)
    nncu.kv4_attention_dev(call)
    nncu.kv4_check(call)
    first = c.out.clone()
    c.ws[:4].view(torch.int32)[0] = 1
    c.ws[256:4096] = 7  # and counters that a call was left with
    with pytest.raises(nncu.NnncError) as e:
        nncu.kv4_check(call)
    assert e.value.status == nncu.ERR_TIMEOUT and "ran out" in str(e.value)
    assert int(c.ws.count_nonzero()) == 0
    nncu.kv4_check(call)
    c.out.fill_(5.0)
    nncu.kv4_attention_dev(call)
    nncu.kv4_check(call)
    assert torch.equal(c.out, first)


# The relative size (2-norm) of an output's error over long spans. A tensor-memory product cuts its accumulator off
# towards zero, 2^-24 of it in the mean. O takes 8 products a tile of 64 keys and starts anew every 6 tiles: 48 cuts of a
# sum that grows from nothing, half of 48 * 2^-24 = 1.4e-6. Scores (up to 7 in base 2, 2 in the mean) take up to 16
# products: 2 * 16 / 2 * 2^-24 * ln 2 = 0.7e-6. The exponential 2^-22 and the halves of q and of the weights (2^-22
# each), at random among the keys: 0.5e-6. Together 2.6e-6; without the new starts a piece of 50 tiles or more has 200
# cuts at half its size and more: 12e-6.
LONG = 4e-6


@pytest.mark.parametrize("d,n_kv,group,keys,new,page", [
    (64, 8, 4, 16000, 1024, 16), (128, 8, 4, 16000, 1000, 32), (256, 4, 2, 16000, 1001, 16), (128, 8, 4, 15990, 900, 256),
])
def test_prompts_in_long_pieces(nncu, torch_cuda, d, n_kv, group, keys, new, page):
    """Pieces of 50 tiles and more: sums added up many times, tables read in many parts; again the same, bit for bit."""
    torch = torch_cuda
    c = Cache(torch, nncu, [keys], n_kv, d, page)
    call = c.attn([new], group, d ** -0.5)
    nncu.kv4_attention_dev(call)
    nncu.kv4_check(call)
    first = c.out.clone()
    for t in (0, 131, 514, new - 1):
        got, want = c.rows(0, [t])
        assert np.linalg.norm(got - want) <= LONG * np.linalg.norm(want), t
    for _ in range(3):
        c.out.fill_(5.0)
        nncu.kv4_attention_dev(call)
        assert torch.equal(c.out, first)


# With scores that rise to 13 in base 2 each product may cut off 2^-24 of them, always towards zero: D / 16 times
# 13 * 2^-24 * ln 2, 8.6e-6 for 256 values, beside the above.
@pytest.mark.parametrize("d,n_kv,group,keys,new,page", [(64, 8, 4, 16000, 1024, 32), (128, 8, 4, 9000, 2000, 16),
                                                        (256, 4, 2, 16000, 1000, 64)])
def test_scores_that_rise_along_long_pieces(nncu, torch_cuda, d, n_kv, group, keys, new, page):
    """The held score moves after sums have been put aside: they follow it."""
    c = Cache(torch_cuda, nncu, [keys], n_kv, d, page, rise=9.0)
    call = c.attn([new], group, d ** -0.5, along=d ** 0.5)
    nncu.kv4_attention_dev(call)
    nncu.kv4_check(call)
    for t in (0, new // 2, new - 1):
        got, want = c.rows(0, [t])
        assert np.linalg.norm(got - want) <= (LONG + d / 16 * 0.54e-6) * np.linalg.norm(want), t


@pytest.mark.parametrize("rise", [0.0, 9.0])
@pytest.mark.parametrize("d,n_kv,group,lens,new,page", [
    (128, 8, 4, [16000, 15000, 16000, 9000], 1, 16), (64, 8, 4, [16000] * 4, 8, 16), (128, 8, 4, [16000] * 4, 8, 32),
    (256, 4, 2, [30000, 16001], 3, 16), (64, 8, 4, [16000, 12345, 16000], 1, 64),
])
def test_decode_in_long_runs(nncu, torch_cuda, d, n_kv, group, lens, new, page, rise):
    """Runs of more tiles than a table read has (8 at 16 keys a page), and segments cut anywhere."""
    torch = torch_cuda
    c = Cache(torch, nncu, lens, n_kv, d, page, rise=rise)
    call = c.attn([new] * len(lens), group, d ** -0.5, along=d ** 0.5 if rise else 0.0)
    nncu.kv4_attention_dev(call)
    nncu.kv4_check(call)
    first = c.out.clone()
    for r in range(len(lens)):
        got, want = c.rows(r, [new - 1])
        assert np.linalg.norm(got - want) <= (LONG + d / 16 * 0.54e-6 * (rise > 0)) * np.linalg.norm(want), r
    nncu.kv4_attention_dev(call)
    assert torch.equal(c.out, first)


def test_long_prompts_side_by_side(nncu, torch_cuda):
    """Two calls on two streams with workspaces of their own, whose prompt parts were left full of ones: the places that
    their sums are kept in are each call's own, and found free."""
    torch = torch_cuda
    c = [Cache(torch, nncu, [16000], 8, 128, 64, seed=s) for s in (3, 4)]
    calls = [x.attn([1000], 4, 128 ** -0.5) for x in c]
    for call in calls:
        nncu.kv4_attention_dev(call)
        nncu.kv4_check(call)
    first = [x.out.clone() for x in c]
    streams = [torch.cuda.Stream() for _ in c]
    for x in c:
        x.ws[-(1 << 25):].fill_(255)
    for _ in range(3):
        for x, call, st in zip(c, calls, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                x.out.fill_(5.0)
                nncu.kv4_attention_dev(call, st)
        torch.cuda.synchronize()
        assert all(torch.equal(x.out, f) for x, f in zip(c, first))
    for call in calls:
        nncu.kv4_check(call)


# Weights are good to 6e-6 for scores up to 40 in base 2 (their rounding and the products' sums 2^-24 of their size, the
# exponential 2^-22, the halves of q and of the weights 2^-21), and an output is a mean of values no larger than vmax.
@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.1, -0.25, 1e-38, 0.3])
@pytest.mark.parametrize("d,new", [(64, 3), (64, 150), (128, 130), (256, 150)])
def test_any_scale(nncu, torch_cuda, d, new, scale, softcap):
    """A scale of zero weighs all keys alike, a negative one turns the order round: masked keys stay masked."""
    c = Cache(torch_cuda, nncu, [new + 70], 2, d, 16)
    nncu.kv4_attention_dev(c.attn([new], 2, scale, softcap=softcap))
    got, want = c.rows(0, sorted({0, 1, new // 2, new - 1}))
    assert np.abs(got - want).max() <= 1e-5 * c.vmax


@pytest.mark.parametrize("scale", [-0.125, 0.0, 1e-4])
def test_any_scale_of_tiny_queries(nncu, torch_cuda, scale):
    """Queries near 2^-100, whose scores vanish: a mean of the values."""
    c = Cache(torch_cuda, nncu, [300], 1, 64, 16)
    call = c.attn([200], 2, scale)
    c.q *= 2.0 ** -100
    nncu.kv4_attention_dev(call)
    got, want = c.rows(0, [0, 100, 199])
    assert np.abs(got - want).max() <= 1e-5 * c.vmax


@pytest.mark.parametrize("window", [(1 << 31) - 1, (1 << 31) - 50, 1000])
@pytest.mark.parametrize("keys,new", [(1, 5), (3, 40), (70, 300), (900, 4)])
def test_windows_of_any_size(nncu, torch_cuda, keys, new, window):
    """More new tokens than keys (the first see none), and a window that all positions fit in."""
    c = Cache(torch_cuda, nncu, [keys], 2, 128, 16)
    nncu.kv4_attention_dev(c.attn([new], 2, 128 ** -0.5, window=window))
    got, want = c.rows(0, sorted({0, max(0, new - keys - 1), max(0, new - keys), new - 1}))
    assert np.abs(got - want).max() <= 1e-5 * c.vmax
