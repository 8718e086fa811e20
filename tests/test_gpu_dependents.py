"""Kernels that begin while the one before them ends, on one buffer that they
write and read in turn: a prompt's chunks scored one after another."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_i8 import code_rows, dev

pytestmark = pytest.mark.gpu

CHUNKS = 24


@pytest.mark.parametrize("n,vocab,cols,top", [
    (3, 40000, 256, 5), (40, 5003, 512, 0), (200, 3001, 128, 3), (300, 20011, 640, 0), (600, 6000, 256, 20),
    (64, 151936, 64, 5)])
def test_chunks_scored_through_one_buffer_of_logits(nncu, torch_cuda, n, vocab, cols, top):
    """Product, log probabilities, product, log probabilities, nothing between, every time other logits in the same
    buffer: called, and as one graph."""
    torch, N = torch_cuda, nncu
    rng = np.random.default_rng(n + vocab)
    w = code_rows(torch, rng.integers(-127, 128, (vocab, cols), dtype=np.int8), rng)
    ws = dev(torch, rng.uniform(1e-3, 2e-3, vocab).astype(np.float32))
    logits = torch.full((n, vocab), float("nan"), device="cuda")
    calls, outs = [], []
    for _ in range(CHUNKS):
        x = code_rows(torch, rng.integers(-127, 128, (n, cols), dtype=np.int8), rng)
        xs, tok = dev(torch, rng.uniform(0.01, 0.05, n).astype(np.float32)), dev(torch, rng.integers(0, vocab, n, dtype=np.int32))
        out = dict(logprob=torch.zeros(n, device="cuda"), entropy=torch.zeros(n, device="cuda"),
                   rank=torch.zeros(n, dtype=torch.int32, device="cuda"))
        if top:
            out |= dict(top_ids=torch.zeros(n, top, dtype=torch.int32, device="cuda"),
                        top_logprobs=torch.zeros(n, top, device="cuda"))
        calls.append((N.i8_linear(n_tok=n, rows=vocab, cols=cols, x=x, x_scales=xs, w=w, w_scales=ws, y=logits),
                      N.logprobs(n=n, n_vocab=vocab, logits=logits, tokens=tok, top=top, **out)))
        outs.append(out)
    want = []
    for (product, report), out in zip(calls, outs):  # each alone
        N.i8_linear_dev(product)
        torch.cuda.synchronize()
        N.logprobs_dev(report)
        torch.cuda.synchronize()
        want.append({k: v.clone() for k, v in out.items()})
    assert not torch.equal(want[0]["entropy"], want[1]["entropy"])

    def chunks(stream):
        for product, report in calls:
            N.i8_linear_dev(product, stream)
            N.logprobs_dev(report, stream)

    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        chunks(torch.cuda.current_stream())
    for it in range(6):
        for out in outs:
            for v in out.values():
                v.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay() if it % 2 else chunks(stream)
        torch.cuda.synchronize()
        for out, one in zip(outs, want):
            for k, v in out.items():
                assert torch.equal(v, one[k]), k
    N.i8_check()


def test_a_check_keeps_to_its_stream(nncu, torch_cuda):
    """While one stream is captured another one is checked; the captured one's own check is refused, and leaves the
    capture as it is."""
    torch, N = torch_cuda, nncu
    rng = np.random.default_rng(1)
    w, x = (code_rows(torch, rng.integers(-127, 128, (n, 64), dtype=np.int8), rng) for n in (40, 3))
    y = torch.zeros(3, 40, device="cuda")
    one = torch.ones(40, device="cuda")
    call = N.i8_linear(n_tok=3, rows=40, cols=64, x=x, x_scales=one, w=w, w_scales=one, y=y)
    other, stream = torch.cuda.Stream(), torch.cuda.Stream()
    N.i8_linear_dev(call, other)
    N.i8_check(other)
    want = y.clone()
    torch.cuda.synchronize()
    y.zero_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        N.i8_linear_dev(call, torch.cuda.current_stream())
        N.i8_check(other)
        with pytest.raises(N.NnncError, match="captured"):
            N.i8_check(torch.cuda.current_stream())
    assert not bool(y.any())
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    N.i8_check(stream)
