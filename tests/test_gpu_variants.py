"""Every variant of the 8-bit product and of the log probabilities against the
definitions in 64 bits: the calls of variants.py, whose plans are checked on the
CPU."""
from __future__ import annotations

import numpy as np
import pytest

import i8_helpers as H
import variants as V
from test_gpu_i8 import pitch
from test_gpu_logprobs import check, run

pytestmark = pytest.mark.gpu


def codes(torch, g, n, cols, low=-128):
    """Random rows of codes on 16 bytes, with noise between them."""
    return torch.randint(low, 128, (n, pitch(cols)), generator=g, dtype=torch.int8, device="cuda")[:, :cols]


def product(torch, x, xs, w, ws, bias, add):
    """(y, how far float32 results may be off) in 64 bits on the GPU: i8_helpers.linear, a part of the channels at a time
    (whole sums below 2^53 are exact)."""
    xd = x.double()
    for a in range(0, w.shape[0], 4096):
        p = (xd @ w[a:a + 4096].double().T) * xs.double()[:, None] * ws[a:a + 4096].double()
        tol = 3 * H.U * p.abs()
        for more in (None if bias is None else bias[a:a + 4096], None if add is None else add[:, a:a + 4096]):
            if more is not None:
                p = p + more.double()
                tol = tol + H.U * p.abs()
        yield a, p, 1.001 * tol + 1e-43


@pytest.mark.parametrize("case", V.LINEAR)
def test_linear(nncu, torch_cuda, case):
    torch, N = torch_cuda, nncu
    n, r, c, has_bias, has_add, slack = case[:6]
    g = torch.Generator(device="cuda").manual_seed(n + r + c)
    u = lambda lo, hi, *s: lo + (hi - lo) * torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    x, w = codes(torch, g, n, c), codes(torch, g, r, c)
    xs, ws = u(1e-3, 1, n), u(1e-4, 1e-3, r)
    bias = 50 * torch.randn(r, generator=g, device="cuda") if has_bias else None
    add = 50 * torch.randn(n, r, generator=g, device="cuda") if has_add else None
    y = torch.full((n + 1, r + slack), -7.0, device="cuda")
    given = None
    if has_add == 2:
        y[:n, :r] = add
        given = y
    elif has_add:
        given = torch.full((n, r + 2), float("nan"), device="cuda")
        given[:, :r] = add
    N.i8_linear_dev(N.i8_linear(n_tok=n, rows=r, cols=c, x=x, x_scales=xs, w=w, w_scales=ws, bias=bias, add=given, y=y))
    torch.cuda.synchronize()
    N.i8_check()
    assert bool((y[n] == -7).all()) and bool((y[:, r:] == -7).all())
    for a, want, tol in product(torch, x, xs, w, ws, bias, add):
        off = (y[:n, a:a + want.shape[1]].double()[:, :r - a] - want).abs()
        assert bool((off <= tol).all()), a


@pytest.mark.parametrize("n,r", [(n, r) for n, r, _ in V.LARGEST])
def test_largest_sums(nncu, torch_cuda, n, r):
    torch, N = torch_cuda, nncu
    c = 131071
    x, w = (torch.full((m, c + 1), -128, dtype=torch.int8, device="cuda") for m in (n, r))
    one = torch.ones(max(n, r), device="cuda")
    y = torch.zeros(n, r, device="cuda")
    N.i8_linear_dev(N.i8_linear(n_tok=n, rows=r, cols=c, x=x, x_scales=one, w=w, w_scales=one, y=y))
    N.i8_check()
    assert bool((y == float(2 ** 31 - 2 ** 14)).all())


def test_a_token_does_not_go_by_its_batch(nncu, torch_cuda):
    """The same token among others, by single CTAs and by pairs: the same bits."""
    torch, N = torch_cuda, nncu
    r, c = V.BATCH
    n = max(b for _, b, _ in V.SLICES)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = codes(torch, g, n, c, -127), codes(torch, g, r, c, -127)
    xs, ws = torch.rand(n, generator=g, device="cuda"), torch.rand(r, generator=g, device="cuda")
    bias = torch.randn(r, generator=g, device="cuda")
    got = []
    for a, b, _ in V.SLICES:
        y = torch.zeros(b - a, r, device="cuda")
        N.i8_linear_dev(N.i8_linear(n_tok=b - a, rows=r, cols=c, x=x[a:b], x_scales=xs[a:b], w=w, w_scales=ws, bias=bias, y=y))
        got.append(y)
    N.i8_check()
    for (a, b, _), y in zip(V.SLICES, got):
        assert torch.equal(y, got[0][a:b])


def test_both_kernels_on_two_streams_at_once(nncu, torch_cuda):
    """Single CTAs and pairs, with the log probabilities of what they give, at once on two streams, new inputs each time."""
    torch, N = torch_cuda, nncu
    r, c = V.TOGETHER
    g = torch.Generator(device="cuda").manual_seed(2)
    w, ws = codes(torch, g, r, c, -127), torch.rand(r, generator=g, device="cuda") * 1e-3
    jobs = []
    for n, _ in V.TOKENS:
        sets = []
        xs, y = torch.rand(n, generator=g, device="cuda") * 0.05, torch.zeros(n, r, device="cuda")
        for _ in range(3):
            ids, ent = torch.zeros(n, 7, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
            x = codes(torch, g, n, c, -127)
            sets.append((N.i8_linear(n_tok=n, rows=r, cols=c, x=x, x_scales=xs, w=w, w_scales=ws, y=y),
                         N.logprobs(n=n, n_vocab=r, logits=y, top=7, top_ids=ids, entropy=ent), ids, ent))
        jobs.append(sets)
    want = []
    for sets in jobs:
        for linear, logprobs, ids, ent in sets:
            N.i8_linear_dev(linear)
            torch.cuda.synchronize()
            N.logprobs_dev(logprobs)
            torch.cuda.synchronize()
            want.append((ids.clone(), ent.clone()))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for sets in jobs:
            for _, _, ids, ent in sets:
                ids.zero_(), ent.zero_()
        torch.cuda.synchronize()
        for k in range(3):
            for sets, st in zip(jobs, streams):
                N.i8_linear_dev(sets[k][0], st)
                N.logprobs_dev(sets[k][1], st)
        torch.cuda.synchronize()
        for one, (ids, ent) in zip([s for sets in jobs for s in sets], want):
            assert torch.equal(one[2], ids) and torch.equal(one[3], ent)
    N.i8_check()


# ---- log probabilities -----------------------------------------------------------------------

def odd(x, at):
    """Rows that are masked whole or but for one, equal throughout, of the lowest and largest values, with NaN and
    infinities, signed zeros, among the others: into the rows `at`."""
    f, v = np.finfo(np.float32), x.shape[1]
    for i, r in enumerate(at):
        k = i % 11
        if k == 0:
            x[r] = -np.inf
        elif k == 1:
            x[r], x[r, v // 2] = -np.inf, 3.0
        elif k == 2:
            x[r] = 1.25
        elif k == 3:
            x[r] = f.min
        elif k == 4:
            x[r, : v // 2] = f.min
        elif k == 5:
            x[r, v // 3] = np.nan
        elif k == 6:
            x[r, v - 1] = np.inf
        elif k == 7:
            x[r] = np.where(np.arange(v) % 3, 0.0, -0.0)
        elif k == 8:
            x[r] = np.where(np.arange(v) % 2, f.max, f.min)
        elif k == 9:
            x[r] = np.nan
        else:
            x[r] = -np.arange(v) * np.float32(0.01)


@pytest.mark.parametrize("case", V.LOGPROBS)
def test_logprobs(nncu, torch_cuda, case):
    """Ordinary rows and odd ones among them; of many, some of the ordinary ones are checked."""
    n, v, top = case[:3]
    rng = np.random.default_rng(n + v + top)
    x = rng.standard_normal((n, v), dtype=np.float32) * np.float32(3)
    x[:, rng.integers(0, v, 3)] += 9
    if v % 2:  # many equal ones, half of them masked
        x = np.round(x * 4) / np.float32(4)
        x[rng.random((n, v), dtype=np.float32) < 0.5] = -np.inf
    at = rng.choice(n, min(n // 2, 22), replace=False)
    odd(x, at)
    tokens = rng.integers(0, v, n)
    tokens[n // 3] = -1
    got = run(nncu, torch_cuda, x, 0.9, tokens, top, slack=n % 4, lead=v % 4)
    some = np.unique(np.concatenate([at, [0, n // 3, n - 1], rng.integers(0, n, 12)]))
    check(x[some], 0.9, tokens[some], top, {k: a[some] for k, a in got.items()})
    some = np.setdiff1d(np.arange(n), some)  # the others: no call leaves one out
    assert np.isfinite(got["entropy"][some]).all() and (got["entropy"][some] > 0).all()
    assert (got["rank"][some] >= 0).all() and (got["rank"][some] < v).all()


def test_columns_of_one_buffer(nncu, torch_cuda):
    """What is added and what comes out in columns of one buffer, looked up into a third part of it, in between its rows."""
    torch, N = torch_cuda, nncu
    g = torch.Generator(device="cuda").manual_seed(4)
    for n, r, c in ((5, 40, 48), (300, 700, 256)):
        x, w = codes(torch, g, n, c), codes(torch, g, r, c)
        xs, ws = torch.rand(n, generator=g, device="cuda"), torch.rand(r, generator=g, device="cuda")
        wide = torch.full((n, 2 * r + c + 10), -7.0, device="cuda")
        wide[:, r:2 * r] = torch.randn(n, r, generator=g, device="cuda")
        add, y, out = wide[:, r:2 * r], wide[:, :r], wide[:, 2 * r + 4:2 * r + 4 + c]
        kept = add.clone()
        N.i8_lookup_dev(N.i8_lookup(n=n, cols=c, n_rows=n, codes=x, scales=xs, out=out))
        N.i8_linear_dev(N.i8_linear(n_tok=n, rows=r, cols=c, x=x, x_scales=xs, w=w, w_scales=ws, add=add, y=y))
        N.i8_check()
        assert torch.equal(add, kept) and torch.equal(out, x.float() * xs[:, None])
        assert bool((wide[:, 2 * r:2 * r + 4] == -7).all()) and bool((wide[:, 2 * r + 4 + c:] == -7).all())
        for a, want, tol in product(torch, x, xs, w, ws, None, kept):
            assert bool(((y.double() - want).abs() <= tol).all())
