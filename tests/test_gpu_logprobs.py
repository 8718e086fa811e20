"""Log probabilities, ranks, entropies and the likeliest tokens on the GPU
against their definitions in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import i8_helpers as H

pytestmark = pytest.mark.gpu

FLOATS, WHOLE = ("logprob", "entropy", "top_logprobs"), ("rank", "top_ids")


def run(N, torch, x, scale, tokens, top, slack=0, lead=0):
    """The call on rows `slack` floats further apart than they are long, from `lead` floats past 16 bytes."""
    n, v = x.shape
    flat = torch.full((lead + (n + 1) * (v + slack),), float("nan"), device="cuda")
    rows = flat[lead:lead + n * (v + slack)].view(n, v + slack)
    rows[:, :v] = torch.as_tensor(x, device="cuda")
    f = lambda *s: torch.full(s, -7.0, device="cuda")  # noqa: E731
    i = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")  # noqa: E731
    out = dict(logprob=f(n + 1), entropy=f(n + 1), rank=i(n + 1), top_ids=i(n + 1, top), top_logprobs=f(n + 1, top))
    N.logprobs_dev(N.logprobs(n=n, n_vocab=v, logits=rows, stride=v + slack, scale=scale,
                              tokens=torch.as_tensor(tokens, dtype=torch.int32, device="cuda"), top=top, **out))
    torch.cuda.synchronize()
    got = {k: a.cpu().numpy() for k, a in out.items()}
    for k, a in got.items():
        assert (a[n] == -7).all(), k  # nothing behind the last row
    return {k: a[:n] for k, a in got.items()}


def check(x, scale, tokens, top, got):
    for r in range(x.shape[0]):
        want, off = H.logprobs(x[r], scale, int(tokens[r]), top)
        for k in WHOLE:
            np.testing.assert_array_equal(got[k][r], want[k], err_msg=f"{k} of row {r}")
        for k in FLOATS:
            a, b = np.asarray(got[k][r], np.float64), np.asarray(want[k], np.float64)
            fine = np.isfinite(b)
            np.testing.assert_array_equal(np.where(fine, 0, a), np.where(fine, 0, b), err_msg=f"{k} of row {r}")
            far = np.abs(np.where(fine, a, 0) - np.where(fine, b, 0))
            assert (far <= off[k]).all(), (k, r, far, off[k])


CASES = [  # rows, vocabulary, top, scale, masked, logits in steps of a 16-bit float, slack, lead
    (1, 1, 1, 1.0, 0, 0, 0, 0), (1, 2, 2, 1.0, 0, 0, 0, 0), (5, 3, 0, 0.5, 0, 0, 1, 1), (3, 31, 31, 1.0, 0, 1, 0, 0),
    (4, 33, 32, 2.0, 0.5, 1, 2, 3), (2, 1000, 5, 1.0, 0, 0, 0, 0), (200, 1001, 3, 1.43, 0.9, 1, 0, 1),
    (1, 4096, 20, 1.0, 0, 0, 0, 0), (1, 32001, 20, 1.0, 0, 1, 0, 2), (7, 50257, 8, 0.7, 0, 0, 4, 0),
    (1, 262144, 32, 1.0, 0, 0, 0, 0), (3, 262144, 20, 1.0, 0.99, 0, 0, 0), (64, 32000, 5, 1.25, 0.9, 1, 0, 0),
    (16, 128256, 0, 1.0, 0, 0, 0, 0), (40, 65537, 32, 1.0, 0, 1, 0, 0), (160, 20000, 1, 1.0, 0, 0, 0, 0),
    (300, 8193, 20, 1.0, 0.2, 0, 3, 1), (1, 500001, 7, 1.0, 0, 0, 0, 0),
    (450, 5003, 5, 1.0, 0.3, 0, 1, 1), (400, 5000, 0, 0.8, 0, 1, 0, 0), (100, 33990, 0, 1.0, 0.5, 0, 2, 3),
    (64, 43807, 9, 1.0, 0, 0, 0, 0), (340, 43807, 5, 1.0, 0, 1, 1, 2), (300, 33990, 0, 2.0, 0, 0, 0, 0), (700, 5001, 32, 1.0, 0.9, 1, 0, 0),
    (150, 43807, 20, 1.0, 0.99, 0, 0, 0),
]


@pytest.mark.parametrize("case", CASES)
def test_logprobs(nncu, torch_cuda, case):
    n, v, top, scale, masked, steps, slack, lead = case
    rng = np.random.default_rng(n + v + top)
    x = (rng.standard_normal((n, v)) * 3).astype(np.float32)
    x[:, rng.integers(0, v, 3)] += 9
    if steps:  # many equal ones
        x = np.round(x * 4) / np.float32(4)
    x[rng.random((n, v)) < masked] = -np.inf
    tokens = rng.integers(0, v, n)
    if n > 2:
        tokens[1], tokens[2] = -1, v
    check(x, scale, tokens, top, run(nncu, torch_cuda, x, scale, tokens, top, slack, lead))


@pytest.mark.parametrize("v", [1, 40, 5000, 70001])
def test_odd_rows(nncu, torch_cuda, v):
    """Rows that are masked whole or but for one token, equal throughout, of the type's lowest and largest values,
    rising, falling, with NaN and infinities, signed zeros."""
    f = np.finfo(np.float32)
    rng = np.random.default_rng(v)
    x = rng.standard_normal((13, v)).astype(np.float32)
    x[0] = -np.inf
    x[1] = -np.inf
    x[1, v // 2] = 3.0
    x[2] = 1.25
    x[3] = f.min
    x[4, : v // 2] = f.min
    x[5] = np.arange(v) * np.float32(0.01)
    x[6] = -np.arange(v) * np.float32(0.01)
    x[7, v // 3] = np.nan
    x[8, v - 1] = np.inf
    x[9] = np.where(rng.random(v) < 0.5, 0.0, -0.0)
    x[10] = np.where(rng.random(v) < 0.5, f.max, f.min)
    x[11, :] = np.nan
    x[12] = -80.0
    x[12, 0] = 20.0
    top = min(v, 20)
    for tokens in (np.full(13, v - 1), np.zeros(13, int), rng.integers(0, v, 13)):
        check(x, 1.0, tokens, top, run(nncu, torch_cuda, x, 1.0, tokens, top))


@pytest.mark.parametrize("n", [1, 5, 300])
def test_likeliest_tokens_side_by_side(nncu, torch_cuda, n):
    """All of the largest logits in one thread's, warp's or CTA's share, at every distance that a share could have."""
    v, top = 40000, 32
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n, v)).astype(np.float32)
    for r in range(n):
        gap = [1, 2, 4, 8, 16, 32, 128, 256, 512, 1000, 1024][r % 11]
        at = (rng.integers(0, v) + gap * np.arange(40)) % v
        x[r, at] = 10 + rng.permutation(40) // 2
    tokens = rng.integers(0, v, n)
    check(x, 1.0, tokens, top, run(nncu, torch_cuda, x, 1.0, tokens, top))


def test_outputs_may_be_left_out(nncu, torch_cuda):
    torch, N = torch_cuda, nncu
    x = torch.randn(3, 999, device="cuda")
    tok = torch.tensor([5, 7, 998], dtype=torch.int32, device="cuda")
    full = dict(logprob=torch.zeros(3, device="cuda"), rank=torch.zeros(3, dtype=torch.int32, device="cuda"),
                entropy=torch.zeros(3, device="cuda"), top_ids=torch.zeros(3, 4, dtype=torch.int32, device="cuda"),
                top_logprobs=torch.zeros(3, 4, device="cuda"))
    N.logprobs_dev(N.logprobs(n=3, n_vocab=999, logits=x, tokens=tok, top=4, **full))
    for k, a in full.items():
        one = torch.zeros_like(a)
        N.logprobs_dev(N.logprobs(n=3, n_vocab=999, logits=x, tokens=tok if k in ("logprob", "rank") else None,
                                  top=4 if k.startswith("top") else 0, **{k: one}))
        assert torch.equal(one, a), k
