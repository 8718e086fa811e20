"""The 8-bit operators and the log probabilities as they are used: one after
another around the paged cache, captured and replayed, on several streams,
behind whatever wrote their inputs."""
from __future__ import annotations

import numpy as np
import pytest

import i8_helpers as H
from test_gpu_i8 import code_rows, dev, exact_linear

pytestmark = pytest.mark.gpu

EMBD, HEADS, KV, HD, VOCAB, PAGE = 208, 6, 2, 64, 1003, 16


def host(x):
    return x.detach().cpu().numpy()


def values(scales, codes, cols):
    return host(codes)[:, :cols], host(scales)


def served(torch, seed, n_req, max_tok, max_new, max_rows, n_pages=40):
    from libllmcpu_b200.paged_bench import I8Matrix, ServedLayer

    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda r, c: torch.randn(r, c, generator=g, device="cuda")  # noqa: E731
    table = I8Matrix(torch, VOCAB, EMBD, rnd(VOCAB, EMBD) * EMBD ** -0.5)
    wqkv = I8Matrix(torch, (HEADS + 2 * KV) * HD, EMBD, (rnd((HEADS + 2 * KV) * HD, EMBD) * 0.1).to(torch.bfloat16))
    wo = I8Matrix(torch, EMBD, HEADS * HD, (rnd(EMBD, HEADS * HD) * 0.05).to(torch.float16))
    gains = 1 + 0.2 * rnd(2, EMBD)
    layer = ServedLayer(torch, HEADS, KV, HD, n_req, PAGE, n_pages, 8, max_tok, max_new, table, wqkv, wo, gains, max_rows)
    layer.ids.random_(0, VOCAB, generator=g)
    layer.chosen.random_(0, VOCAB, generator=g)
    return layer, table, wqkv, wo, gains


def check_quantised(x, gamma, norm, codes, scales):
    want_c, want_s = H.quantise(x, gamma, norm, 1e-6)
    np.testing.assert_array_equal(host(codes)[:, :x.shape[1]], want_c)
    assert (np.abs(host(scales) - want_s) <= 1.01 * H.U * want_s).all()


def check_product(torch, got, codes, scales, m, add=None):
    x, xs = values(scales, codes, m.cols)
    w, ws = values(m.scales, m.codes, m.cols)
    want, tol = exact_linear(torch, x, xs, w, ws, None, add)
    assert (np.abs(host(got) - want) <= tol).all()


def test_a_step_around_the_paged_cache(nncu, torch_cuda):
    """Prompts, then decode steps: every operator's output against its definition, from what the one before it left."""
    torch, N = torch_cuda, nncu
    from libllmcpu_b200.paged_bench import _resize

    prompts, n_req = [37, 1, 70], 3
    layer, table, wqkv, wo, gains = served(torch, 1, n_req, sum(prompts), max(prompts), 4)
    layer.new.copy_(torch.tensor(prompts, dtype=torch.int32))
    for step in range(4):
        n = sum(prompts) if step == 0 else n_req
        if step == 1:
            _resize(layer, n_req, 1)
            layer.new.fill_(1)
        layer.past.copy_(layer.seq_len)
        tokens = host(layer.ids)[:n]
        for name, call in layer.operators():
            before = host(layer.hidden)[:n].copy()
            call()
            torch.cuda.synchronize()
            if name == "embed":
                c, s = values(table.scales, table.codes, EMBD)
                want = c[tokens].astype(np.float64) * (s[tokens].astype(np.float64) * np.float32(EMBD ** 0.5))[:, None]
                assert (np.abs(host(layer.hidden)[:n] - want) <= 2.01 * H.U * np.abs(want)).all()
            elif name == "qkv":
                check_quantised(before, host(gains[0]), 1, layer.codes[:n], layer.scales[:n])
                check_product(torch, layer.qkv[:n], layer.codes[:n], layer.scales[:n], wqkv)
            elif name == "attention":
                slots, seq = host(layer.slots)[:n], host(layer.seq_len)
                assert (slots >= 0).all() and list(seq) == [p + step for p in prompts]
            elif name == "output":
                check_quantised(host(layer.out)[:n], None, 0, layer.attn_codes[:n], layer.attn_scales[:n])
                check_product(torch, layer.hidden[:n], layer.attn_codes[:n], layer.attn_scales[:n], wo, before)
            elif name == "logits":
                check_quantised(before, host(gains[1]), 1, layer.codes[:n], layer.scales[:n])
                check_product(torch, layer.logits[:n], layer.codes[:n], layer.scales[:n], table)
            elif name == "logprobs":
                for r in range(n):
                    want, off = H.logprobs(host(layer.logits)[r], 1.0, int(layer.chosen[r]), layer.TOP)
                    for k in ("rank", "top_ids"):
                        np.testing.assert_array_equal(host(layer.report[k])[r], want[k])
                    for k in ("logprob", "entropy", "top_logprobs"):
                        assert (np.abs(host(layer.report[k])[r] - want[k]) <= off[k]).all()
        assert [name for name, _ in layer.operators()][-1] == ("output" if step == 0 else "logprobs")
        layer.turn ^= 1  # (looking at the operators took a turn)
        if step:
            layer.ids[:n_req].copy_(layer.report["top_ids"][:n_req, 0])
    N.kv4_check(layer.attn)
    N.i8_check()


def test_a_replayed_step_gives_what_calls_give(nncu, torch_cuda):
    """Decode steps as graphs (every kernel a programmatic dependent of the one before) and call by call: the same bits."""
    torch = torch_cuda
    runs = []
    for graphed in (False, True):
        layer, *_ = served(torch, 5, 4, 4, 1, 4)
        layer.new.fill_(1)

        def step(stream):
            layer.past.copy_(layer.seq_len)
            layer.step(stream)
            layer.ids.copy_(layer.report["top_ids"][:, 0])

        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            graphs = []
            if graphed:
                for _ in range(2):
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g, stream=stream):
                        step(torch.cuda.current_stream())
                    graphs.append(g)
                layer.turn = 0
            seen = []
            for it in range(12):
                if graphed:
                    graphs[it & 1].replay()
                else:
                    step(stream)
                seen.append([x.clone() for x in (layer.hidden, layer.logits, layer.ids, *layer.report.values())])
        torch.cuda.synchronize()
        runs.append(seen)
    for a, b in zip(*runs):
        for x, y in zip(a, b):
            assert torch.equal(x, y)
    assert len({tuple(s[0][0].tolist()) for s in runs[0]}) > 1  # (the steps do not all repeat the first)


def test_kernels_wait_for_what_they_read(nncu, torch_cuda):
    """Inputs of every kind rewritten right before each call, by torch's kernels and by these operators, many times over:
    nothing stale is read, nothing is overwritten early."""
    torch, N = torch_cuda, nncu
    n, rows, cols = 40, 700, 2048
    st = torch.cuda.current_stream()
    g = torch.Generator(device="cuda").manual_seed(3)
    sources = [torch.randn(n, cols, generator=g, device="cuda") for _ in range(3)]
    weights = [torch.randn(rows, cols, generator=g, device="cuda") for _ in range(3)]
    x, w = torch.empty_like(sources[0]), torch.empty_like(weights[0])
    xc, wc = (torch.empty(r, cols, dtype=torch.int8, device="cuda") for r in (n, rows))
    xs, ws, y = torch.empty(n, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(n, rows, device="cuda")
    lp, tok = torch.empty(n, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    qx = N.i8_rows(n=n, cols=cols, x=x, codes=xc, scales=xs, norm=1)
    qw = N.i8_rows(n=rows, cols=cols, x=w, codes=wc, scales=ws)
    mul = N.i8_linear(n_tok=n, rows=rows, cols=cols, x=xc, x_scales=xs, w=wc, w_scales=ws, y=y)
    ask = N.logprobs(n=n, n_vocab=rows, logits=y, tokens=tok, logprob=lp)
    back = N.i8_lookup(n=n, cols=cols, n_rows=n, codes=xc, scales=xs, out=x)

    def once(a, b):
        x.copy_(sources[a])
        w.copy_(weights[b])
        N.i8_quantise_dev(qx, st)
        N.i8_quantise_dev(qw, st)
        N.i8_linear_dev(mul, st)
        tok.fill_(b)
        N.logprobs_dev(ask, st)
        N.i8_lookup_dev(back, st)  # writes what the first call read
        return y.clone(), lp.clone(), x.clone()

    want = {}
    for a in range(3):
        for b in range(3):
            want[a, b] = once(a, b)
            torch.cuda.synchronize()
    got = [((it * 7) % 3, (it * 5 + it // 3) % 3) for it in range(150)]
    outs = [once(a, b) for a, b in got]
    torch.cuda.synchronize()
    for k, o in zip(got, outs):
        for u, v in zip(o, want[k]):
            assert torch.equal(u, v)
    N.i8_check()


def test_calls_on_two_streams_at_once(nncu, torch_cuda):
    """Products (both kernels), rows and log probabilities at once on two streams, nothing shared but the weights."""
    torch, N = torch_cuda, nncu
    rng = np.random.default_rng(2)
    rows, cols = 1500, 1024
    w = code_rows(torch, rng.integers(-127, 128, (rows, cols), dtype=np.int8), rng)
    ws = dev(torch, rng.uniform(0.01, 1, rows).astype(np.float32))
    jobs = []
    for n in (3, 900):
        xc = code_rows(torch, rng.integers(-127, 128, (n, cols), dtype=np.int8), rng)
        xs, y = dev(torch, rng.uniform(0.01, 1, n).astype(np.float32)), torch.zeros(n, rows, device="cuda")
        ids = torch.zeros(n, 7, dtype=torch.int32, device="cuda")
        tl, codes, sc = torch.zeros(n, 7, device="cuda"), torch.zeros(n, 1504, dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
        jobs.append((N.i8_linear(n_tok=n, rows=rows, cols=cols, x=xc, x_scales=xs, w=w, w_scales=ws, y=y),
                     N.logprobs(n=n, n_vocab=rows, logits=y, top=7, top_ids=ids, top_logprobs=tl),
                     N.i8_rows(n=n, cols=rows, x=y, codes=codes, scales=sc), (y, ids, tl, codes, sc)))

    def run(job, stream):
        N.i8_linear_dev(job[0], stream)
        N.logprobs_dev(job[1], stream)
        N.i8_quantise_dev(job[2], stream)

    want = []
    for job in jobs:
        run(job, torch.cuda.current_stream())
        torch.cuda.synchronize()
        want.append([t.clone() for t in job[3]])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(40):
        for job in jobs:
            for t in job[3]:
                t.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for job, st in zip(jobs, streams):
                run(job, st)
        torch.cuda.synchronize()
        for job, ts in zip(jobs, want):
            for a, b in zip(job[3], ts):
                assert torch.equal(a, b)
    N.i8_check()


def test_two_graphs_replayed_at_once(nncu, torch_cuda):
    """Graphs that hold the same weights, replayed on two streams at once, share nothing else (there is no workspace)."""
    torch, N = torch_cuda, nncu
    rng = np.random.default_rng(4)
    w = code_rows(torch, rng.integers(-127, 128, (640, 4096), dtype=np.int8), rng)
    ws = torch.ones(640, device="cuda")
    graphs, ys, want = [], [], []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        x = code_rows(torch, rng.integers(-127, 128, (5, 4096), dtype=np.int8), rng)
        y = torch.zeros(5, 640, device="cuda")
        call = N.i8_linear(n_tok=5, rows=640, cols=4096, x=x, x_scales=torch.ones(5, device="cuda"), w=w, w_scales=ws, y=y)
        N.i8_linear_dev(call)
        torch.cuda.synchronize()
        want.append(y.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            for _ in range(5):
                N.i8_linear_dev(call, torch.cuda.current_stream())
        graphs.append((g, call))
        ys.append(y)
    for _ in range(30):
        for y in ys:
            y.zero_()
        torch.cuda.synchronize()
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for y, v in zip(ys, want):
            assert torch.equal(y, v)


def test_memory_that_is_not_the_gpus_is_refused(nncu, torch_cuda):
    """Raw addresses of host memory are refused before anything is launched."""
    torch, N = torch_cuda, nncu
    pinned = torch.zeros(64, 64).pin_memory()
    z = torch.zeros(64, 64, device="cuda")
    c = torch.zeros(64, 64, dtype=torch.int8, device="cuda")
    one = torch.ones(64, device="cuda")
    for call in (lambda: N.i8_quantise_dev(N.i8_rows(n=4, cols=64, x=z, codes=np.zeros((4, 64), np.int8).ctypes.data // 16 * 16, scales=one)),
                 lambda: N.i8_lookup_dev(N.i8_lookup(n=4, cols=64, n_rows=64, codes=c, scales=one, out=pinned.data_ptr())),
                 lambda: N.i8_linear_dev(N.i8_linear(n_tok=4, rows=64, cols=64, x=c, x_scales=one, w=c, w_scales=one, y=pinned.data_ptr())),
                 lambda: N.logprobs_dev(N.logprobs(n=4, n_vocab=64, logits=pinned.data_ptr(), entropy=one))):
        before = N.launch_count()
        with pytest.raises(N.NnncError):
            call()
        assert N.launch_count() == before
    torch.cuda.synchronize()


def test_served_bench_runs(nncu, torch_cuda, capsys):
    from libllmcpu_b200 import paged_bench

    assert paged_bench.main(["--model", "llama3.2-1b", "--requests", "5", "--context", "200", "--page", "16", "--steps", "4",
                             "--vocab", "5000"]) == 0
    assert '"logprobs"' in capsys.readouterr().out
