"""Serve requests from a paged 4-bit cache, one layer of a named model shape,
and time the step's four operators:

    python -m libllmcpu_b200.paged_bench --model qwen3-8b --requests 64 --context 4096 --steps 50

Prompts first: every request gets a prompt of its own length (up to
``--context``) through the tables, the rotation, the cache write and the
attention, then ``--steps`` decode steps of ``--tokens`` tokens each. The
tables are built on the device from the requests' lengths, so the decode step
is captured once as a CUDA graph pair (the table's state alternates) and
replayed. One JSON line: the prompts' time, the median decode step, its
operators timed one by one, the cache's size. q, k and v are random rows in
place of the projections.
"""
from __future__ import annotations

import argparse
import json

import numpy as np

from . import (kv4_append_dev, kv4_attention_dev, kv4_attn, kv4_bytes, kv4_check, kv4_pool, kv4_rows,
               kv4_workspace_bytes, paged_step, paged_step_dev, rope_axes, rope_axes_dev)
from .forward_bench import MODELS


class PagedLayer:
    """One layer's paged cache and the buffers of its steps: `max_tok` tokens a
    step from `n_req` requests of up to `max_blocks` pages each."""

    def __init__(self, torch, n_head: int, n_kv: int, head_dim: int, n_req: int, page: int, n_pages: int,
                 max_blocks: int, max_tok: int, max_new: int):
        i32 = torch.int32
        z = lambda *n: torch.zeros(*n, dtype=i32, device="cuda")  # noqa: E731
        f = lambda *n: torch.empty(*n, device="cuda")  # noqa: E731
        self.torch, self.turn = torch, 0
        self.past, self.new, self.seq_len, self.q_start = z(n_req), z(n_req), z(n_req), z(n_req + 1)
        self.held, self.queue = [z(n_req), z(n_req)], [z(4), z(4)]
        self.queue[0][1] = n_pages
        self.positions, self.slots, self.token_req = z(max_tok), z(max_tok), z(max_tok)
        self.table, self.ring = z(n_req, max_blocks), torch.arange(n_pages, dtype=i32, device="cuda")
        self.pages = torch.zeros(kv4_bytes(n_pages, page, n_kv, head_dim), dtype=torch.uint8, device="cuda")
        self.q, self.k, self.v = f(max_tok, n_head * head_dim), f(max_tok, n_kv * head_dim), f(max_tok, n_kv * head_dim)
        self.out = torch.zeros_like(self.q)
        half = head_dim // 2
        self.inv_freq = torch.as_tensor((1e6 ** (-np.arange(half) / half)).astype(np.float32), device="cuda")
        self.steps = [paged_step(n_req=n_req, page_size=page, n_pages=n_pages, max_blocks=max_blocks, max_tok=max_tok,
                                 past=self.past, n_new=self.new, held=self.held[i], queue=self.queue[i],
                                 ring=self.ring, block_table=self.table, held_out=self.held[1 - i],
                                 queue_out=self.queue[1 - i], seq_len=self.seq_len, q_start=self.q_start,
                                 positions=self.positions, slots=self.slots, token_req=self.token_req)
                      for i in (0, 1)]
        self.rope = rope_axes(n_tok=max_tok, n_head=n_head, n_kv=n_kv, head_dim=head_dim, positions=self.positions,
                              inv_freq=self.inv_freq, q=self.q, k=self.k)
        pool = kv4_pool(self.pages, n_pages, page, n_kv, head_dim)
        self.rows = kv4_rows(pool, slots=self.slots, n_tok=max_tok, k=self.k, v=self.v)
        self.attn = kv4_attn(pool, n_req=n_req, n_tok=max_tok, n_head=n_head, max_new=max_new, max_blocks=max_blocks,
                             block_table=self.table, seq_len=self.seq_len, q_start=self.q_start, q=self.q, out=self.out)
        self.workspace = torch.zeros(kv4_workspace_bytes(self.attn), dtype=torch.uint8, device="cuda")
        self.attn.workspace, self.attn.workspace_bytes = self.workspace.data_ptr(), self.workspace.numel()

    def operators(self, stream=None):
        """The step's calls in order, by name (each step takes the other half of the tables' state)."""
        self.turn ^= 1
        step = self.steps[self.turn ^ 1]
        return [("tables", lambda: paged_step_dev(step, stream)), ("rope", lambda: rope_axes_dev(self.rope, stream)),
                ("append", lambda: kv4_append_dev(self.rows, stream)),
                ("attention", lambda: kv4_attention_dev(self.attn, stream))]

    def step(self, stream=None) -> None:
        for _, call in self.operators(stream):
            call()


def _resize(layer: PagedLayer, n_tok: int, max_new: int) -> None:
    """Fewer tokens a step in the same buffers (a decode step after the prompts)."""
    for s in layer.steps:
        s.max_tok = n_tok
    layer.rope.n_tok = layer.rows.n_tok = layer.attn.n_tok = n_tok
    layer.attn.max_new = max_new


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--model", choices=sorted(MODELS), default="qwen3-8b")
    ap.add_argument("--requests", type=int, default=64)
    ap.add_argument("--context", type=int, default=4096, help="the longest prompt")
    ap.add_argument("--page", type=int, default=64)
    ap.add_argument("--tokens", type=int, default=1, help="tokens of a request in a decode step")
    ap.add_argument("--steps", type=int, default=50)
    a = ap.parse_args(argv)

    import torch

    _, n_head, n_kv, hd, _ = MODELS[a.model]
    rng = np.random.default_rng(0)
    prompts = np.maximum(1, (a.context * rng.uniform(0.1, 1.0, a.requests)).astype(np.int64))
    prompts[0] = a.context
    most = a.context + a.tokens * (a.steps + 20)
    max_blocks = -(-most // a.page)
    n_pages = int(sum(-(-(int(p) + most - a.context) // a.page) for p in prompts)) + 1
    layer = PagedLayer(torch, n_head, n_kv, hd, a.requests, a.page, n_pages, max_blocks, int(prompts.sum()),
                       int(prompts.max()))
    gen = torch.Generator(device="cuda").manual_seed(0)
    for x in (layer.q, layer.k, layer.v):
        x.normal_(generator=gen)

    def event():
        return torch.cuda.Event(enable_timing=True)

    layer.new.copy_(torch.as_tensor(prompts, dtype=torch.int32))
    b, e = event(), event()
    b.record()
    layer.step()
    e.record()
    kv4_check(layer.attn)
    prompt_ms = b.elapsed_time(e)
    if int(layer.queue[layer.turn][2]) or not torch.equal(layer.seq_len.cpu(), torch.as_tensor(prompts, dtype=torch.int32)):
        raise RuntimeError("a prompt was not served")

    _resize(layer, a.requests * a.tokens, a.tokens)
    layer.new.fill_(a.tokens)

    def advance():
        layer.past.copy_(layer.seq_len)

    # the operators one by one, then whole steps as a pair of graphs
    times = {}
    for it in range(6):
        advance()
        for name, call in layer.operators():
            b, e = event(), event()
            b.record()
            call()
            e.record()
            e.synchronize()
            if it > 1:
                times.setdefault(name, []).append(b.elapsed_time(e) * 1e3)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            advance()
            layer.step(torch.cuda.current_stream())
        graphs.append(g)
    steps = []
    for it in range(a.steps):
        b, e = event(), event()
        b.record()
        graphs[it & 1].replay()
        e.record()
        e.synchronize()
        steps.append(b.elapsed_time(e) * 1e3)
    kv4_check(layer.attn)
    keys = int(layer.seq_len.sum())
    if keys != int(prompts.sum()) + a.requests * a.tokens * (6 + a.steps) or not bool(torch.isfinite(layer.out).all()):
        raise RuntimeError("the decode steps did not advance every request")
    print(json.dumps(dict(what="paged 4-bit serving step", model=a.model, requests=a.requests, context=a.context,
                          page=a.page, tokens=a.tokens, prompt_tokens=int(prompts.sum()), prompts_ms=round(prompt_ms, 3),
                          step_us=round(float(np.median(steps)), 2),
                          operators_us={k: round(float(np.median(v)), 2) for k, v in times.items()},
                          cached_keys=keys, cache_MB=round(layer.pages.numel() / 1e6, 1),
                          bf16_cache_MB=round(layer.pages.numel() / 0.5625 * 2 / 1e6, 1))))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
