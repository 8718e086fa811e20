"""Rows in 8 bits on the GPU against their definitions in 64 bits: quantised
with their norm, looked up, multiplied."""
from __future__ import annotations

import numpy as np
import pytest

import i8_helpers as H

pytestmark = pytest.mark.gpu


def dev(torch, x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=dtype, device="cuda")


def rows(torch, x, slack, fill):
    """x's rows on the device, `slack` values further apart than they are long, whose values are `fill`."""
    wide = torch.full((x.shape[0], x.shape[1] + slack), fill, dtype=torch.from_numpy(x[:1, :1].copy()).dtype, device="cuda")
    wide[:, :x.shape[1]] = dev(torch, x)
    return wide[:, :x.shape[1]]


def pitch(cols):
    return -(-cols // 16) * 16


def code_rows(torch, x, rng, more=0):
    """int8 rows on 16 bytes, with noise between them."""
    wide = dev(torch, rng.integers(-128, 128, (x.shape[0], pitch(x.shape[1]) + 16 * more), dtype=np.int8))
    wide[:, :x.shape[1]] = dev(torch, x)
    return wide[:, :x.shape[1]]


# ---- quantised -----------------------------------------------------------------------------

QUANTISE = [  # rows, cols, type, gain, norm, values between rows
    (1, 1, "float32", 0, 0, 0), (3, 7, "float32", 1, 1, 2), (5, 64, "bfloat16", 1, 1, 0), (2, 100, "float16", 0, 1, 3),
    (64, 2048, "float32", 1, 1, 0), (9, 2560, "bfloat16", 0, 0, 8), (33, 4096, "float32", 0, 1, 4),
    (7, 4095, "float32", 1, 0, 0), (2, 5000, "float16", 1, 1, 0), (3, 16384, "float32", 1, 1, 0),
    (2, 33000, "bfloat16", 1, 1, 1), (1, 131071, "float32", 1, 1, 0), (700, 1030, "float32", 1, 1, 2),
    # many rows
    (2500, 1030, "float32", 1, 1, 2), (2401, 2048, "bfloat16", 1, 1, 0), (9001, 64, "float32", 1, 0, 0),
    (5003, 500, "float16", 0, 1, 4), (4750, 301, "float32", 0, 1, 3), (700, 8192, "float32", 1, 1, 0),
    (2600, 1500, "float32", 1, 1, 1),
]


def typed(x, kind):
    """float32 values that the type holds."""
    import torch

    return torch.from_numpy(x).to(getattr(torch, kind)).float().numpy()


def quantised(N, torch, x, kind, gamma, norm, eps=1e-6, slack=0):
    n, cols = x.shape
    xt = rows(torch, x, slack, float("nan")).to(getattr(torch, kind)) if kind == "float32" else None
    if xt is None:
        wide = torch.full((n, cols + slack), float("nan"), dtype=getattr(torch, kind), device="cuda")
        wide[:, :cols] = dev(torch, x).to(getattr(torch, kind))
        xt = wide[:, :cols]
    codes = torch.full((n + 1, pitch(cols) + 16), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((n + 1,), -7.0, device="cuda")
    g = None if gamma is None else dev(torch, gamma)
    N.i8_quantise_dev(N.i8_rows(n=n, cols=cols, x=xt, x_stride=cols + slack, codes=codes,
                                code_stride=codes.shape[1], scales=scales, gamma=g, norm=norm, eps=eps))
    torch.cuda.synchronize()
    c, s = codes.cpu().numpy(), scales.cpu().numpy()
    assert (c[n] == 99).all() and (c[:, cols:] == 99).all() and s[n] == -7.0  # nothing past a row or behind the last
    return c[:n, :cols].astype(np.int64), s[:n]


def check_rows(x, got, gamma, norm, eps=1e-6):
    codes, scales = H.quantise(x, gamma, norm, eps)
    np.testing.assert_array_equal(got[0], codes)
    np.testing.assert_array_equal(np.isnan(got[1]), np.isnan(scales))
    fine = ~np.isnan(scales)
    # the step is the definition's own; with the norm it is rounded once more (a hundredth for the sums in 64 bits)
    off = np.abs(got[1][fine] - scales[fine])
    assert (off <= (1.01 * H.U * scales[fine] + 1e-45 if norm else 0)).all()


@pytest.mark.parametrize("case", QUANTISE)
def test_quantise(nncu, torch_cuda, case):
    n, cols, kind, gain, norm, slack = case
    rng = np.random.default_rng(sum(map(int, (n, cols, gain, norm))))
    x = rng.standard_normal((n, cols)).astype(np.float32) * np.exp(rng.uniform(-5, 5, (n, 1))).astype(np.float32)
    x[:, rng.integers(0, cols, max(1, cols // 200))] *= 20
    x = typed(x, kind)
    gamma = (1 + 0.3 * rng.standard_normal(cols)).astype(np.float32) if gain else None
    check_rows(x, quantised(nncu, torch_cuda, x, kind, gamma, norm, slack=slack), gamma, norm)


@pytest.mark.parametrize("cols", [254, 4096, 40000])
def test_quantise_at_the_borders(nncu, torch_cuda, cols):
    """Values half way between two codes, and next to that, with steps of every size of mantissa."""
    rng = np.random.default_rng(cols)
    x = np.zeros((40, cols), np.float32)
    for r in range(40):
        top = np.float32(rng.uniform(1, 2) * 2.0 ** rng.integers(-60, 60)) if r % 3 else np.float32(127 * 2.0 ** (r - 20))
        step = top / np.float32(127)
        half = ((rng.integers(-126, 126, cols) + 0.5) * np.float64(step)).astype(np.float32)
        side = rng.integers(-1, 2, cols)
        x[r] = np.where(side < 0, np.nextafter(half, np.float32(-np.inf)), np.where(side > 0, np.nextafter(half, np.float32(np.inf)), half))
        x[r, r % cols] = top
    check_rows(x, quantised(nncu, torch_cuda, x, "float32", None, 0), None, 0)


@pytest.mark.parametrize("kind,top", [(k, t) for k in ("float32", "bfloat16", "float16")
                                      for t in (2.0 ** -119, 1.7 * 2.0 ** -119, 2.0 ** -10, 1.99 * 2.0 ** 120)
                                      if k != "float16" or t == 2.0 ** -10])  # (the others are past its range)
def test_quantise_next_to_every_border(nncu, torch_cuda, kind, top):
    """For many steps (the least, whose halves are no floats, among them) the values at, just below and just above all 254
    borders between codes; of 16-bit inputs the nearest ones that there are."""
    import torch as t

    rng = np.random.default_rng(8)
    most = typed((top * rng.uniform(1, 2, 60)).astype(np.float32), kind)
    step = (most * (np.float32(1) / np.float32(127))).astype(np.float64)[:, None]
    border = ((np.arange(-127, 127) + 0.5) * step).astype(np.float32)
    x = np.concatenate([np.nextafter(border, np.float32(-np.inf)), border, np.nextafter(border, np.float32(np.inf)), most[:, None]], 1)
    x = t.from_numpy(x).to(getattr(t, kind)).float().numpy()
    x = np.concatenate([x, np.zeros((60, 5), np.float32)], 1)  # 768 values
    for cols in (768, 767):  # with and without code for odd ends
        check_rows(x[:, :cols].copy(), quantised(nncu, torch_cuda, x[:, :cols].copy(), kind, None, 0), None, 0)


@pytest.mark.parametrize("cols", [17, 2048, 2051, 70000])
def test_quantise_odd_rows(nncu, torch_cuda, cols):
    """Rows of zeros, of subnormal and of the largest values, with NaN and infinities, signed zeros."""
    f = np.finfo(np.float32)
    x = np.random.default_rng(cols).standard_normal((9, cols)).astype(np.float32)
    x[0] = 0
    x[1] = -0.0
    x[2] *= np.float32(1e-40)
    x[3] = np.where(x[3] > 0, f.max, -f.max)
    x[4, cols // 2] = np.nan
    x[5, cols - 1] = -np.inf
    x[6, 0] = np.inf
    x[7] *= np.float32(1e25)  # squares past float32
    x[8] *= np.float32(1e-25)
    for norm, eps in ((0, 0.0), (1, 1e-6), (1, 0.0)):
        check_rows(x, quantised(nncu, torch_cuda, x, "float32", None, norm, eps), None, norm, eps)


# ---- looked up -----------------------------------------------------------------------------

@pytest.mark.parametrize("n,cols,vocab,slack", [(1, 1, 1, 0), (5, 100, 7, 3), (64, 2048, 1000, 0), (3, 4097, 20, 1),
                                                (1000, 2560, 300, 4), (2, 131071, 5, 0)])
def test_lookup(nncu, torch_cuda, n, cols, vocab, slack):
    torch, N = torch_cuda, nncu
    rng = np.random.default_rng(n + cols)
    table = rng.integers(-128, 128, (vocab, cols), dtype=np.int8)
    scales = rng.uniform(1e-4, 1, vocab).astype(np.float32)
    ids = rng.integers(0, vocab, n).astype(np.int32)
    if n > 2:
        ids[1], ids[n // 2], ids[n - 1] = -1, vocab, -2 ** 31
        ids[0] = vocab - 1
    codes = code_rows(torch, table, rng, 1)
    out = torch.full((n + 1, cols + slack), -7.0, device="cuda")
    mult = float(np.float32(np.sqrt(cols)))
    N.i8_lookup_dev(N.i8_lookup(n=n, cols=cols, n_rows=vocab, codes=codes, scales=dev(torch, scales),
                                ids=dev(torch, ids), mult=mult, out=out, out_stride=cols + slack))
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert (got[n] == -7).all() and (got[:, cols:] == -7).all()
    inside = (ids >= 0) & (ids < vocab)
    at = np.where(inside, ids, 0)
    want = np.where(inside[:, None], table[at].astype(np.float64) * (scales[at].astype(np.float64) * mult)[:, None], 0)
    assert (np.abs(got[:n, :cols] - want) <= 2.001 * H.U * np.abs(want)).all()  # two roundings


def test_rows_read_back_are_what_was_quantised(nncu, torch_cuda):
    """Every value within half a step of what went in."""
    torch, N = torch_cuda, nncu
    x = torch.randn(37, 1000, device="cuda")
    codes = torch.empty(37, 1008, dtype=torch.int8, device="cuda")
    scales, back = torch.empty(37, device="cuda"), torch.empty(37, 1000, device="cuda")
    N.i8_quantise_dev(N.i8_rows(n=37, cols=1000, x=x, codes=codes, scales=scales))
    N.i8_lookup_dev(N.i8_lookup(n=37, cols=1000, n_rows=37, codes=codes, scales=scales, out=back))
    off = (back.double() - x.double()).abs()
    assert bool((off <= (0.5 + 127 * 2 * H.U) * scales.double().unsqueeze(1)).all())


# ---- multiplied ----------------------------------------------------------------------------

LINEAR = [  # tokens, rows, cols, bias, add (2: y itself), values between rows of y
    (1, 1, 1, 0, 0, 0), (1, 128, 128, 0, 0, 0), (1, 6144, 4096, 0, 0, 0), (3, 5, 17, 1, 1, 3), (7, 130, 300, 1, 0, 1),
    (16, 2560, 2048, 0, 2, 0), (17, 257, 129, 1, 2, 5), (31, 1000, 4096, 0, 1, 0), (33, 4096, 2560, 1, 1, 0),
    (64, 640, 8192, 0, 0, 0), (65, 129, 127, 0, 1, 2), (100, 6144, 640, 1, 0, 0), (128, 256, 16384, 0, 0, 0),
    (129, 512, 512, 1, 1, 0), (255, 2561, 1000, 0, 0, 7), (256, 256, 256, 0, 2, 0), (257, 300, 2048, 1, 0, 0),
    (300, 4096, 2560, 0, 1, 0), (777, 2560, 2048, 1, 0, 0), (1000, 100, 96, 0, 0, 0), (1025, 1537, 130, 1, 1, 1),
    (200, 2560, 10240, 0, 1, 0), (520, 2000, 20000, 1, 0, 1), (333, 515, 9000, 1, 2, 1), (1500, 300, 16384, 0, 0, 0),
    (200, 20480, 300, 0, 0, 0), (4099, 6200, 300, 1, 0, 3),
    (53, 6961, 10665, 1, 1, 0), (1, 5940, 7068, 0, 2, 0), (1, 10436, 9584, 1, 1, 1), (2793, 17, 7489, 0, 1, 0),
    (1, 2912, 4032, 1, 2, 0), (2538, 20, 6169, 1, 1, 2), (1367, 16, 6873, 0, 0, 0), (1187, 18, 7366, 1, 1, 0),
    (363, 6513, 2729, 0, 1, 1), (155, 9877, 3828, 1, 2, 0), (383, 1993, 14475, 1, 1, 1), (50, 7333, 14773, 0, 2, 0),
    (2498, 147, 14681, 1, 1, 0), (49, 4725, 21378, 1, 0, 2), (1910, 165, 14429, 0, 2, 1), (57, 2895, 27905, 1, 1, 0),
    (600, 5000, 130, 1, 1, 3), (270, 9000, 64, 0, 2, 0), (2050, 1300, 3000, 1, 1, 2), (2050, 1300, 3000, 0, 2, 0), (900, 700, 640, 0, 1, 0),
    (2500, 40, 700, 0, 0, 0), (2048, 2048, 1024, 0, 0, 0), (5, 40000, 200, 0, 0, 0), (2, 3, 131071, 0, 0, 0),
    (40, 16, 100000, 0, 0, 0), (4100, 130, 16, 1, 2, 2),
]


def multiplied(N, torch, x, xs, w, ws, bias, add, slack, rng, stream=None):
    n, r = x.shape[0], w.shape[0]
    y = torch.full((n + 1, r + slack), -7.0, device="cuda")
    a = None
    if add is not None and add[1]:  # in place
        y[:n, :r] = dev(torch, add[0])
        a = y
    elif add is not None:
        a = rows(torch, add[0], 2, float("nan"))
    call = N.i8_linear(n_tok=n, rows=r, cols=x.shape[1], x=code_rows(torch, x, rng), x_scales=dev(torch, xs),
                       w=code_rows(torch, w, rng, 1), w_scales=dev(torch, ws),
                       bias=None if bias is None else dev(torch, bias), add=a, y=y, y_stride=r + slack,
                       x_stride=pitch(x.shape[1]), w_stride=pitch(x.shape[1]) + 16,
                       add_stride=r + slack if add is not None and add[1] else r + 2)
    N.i8_linear_dev(call, stream)
    torch.cuda.synchronize()
    N.i8_check()
    got = y.cpu().numpy()
    assert (got[n] == -7).all() and (got[:, r:] == -7).all()
    return got[:n, :r]


@pytest.mark.parametrize("case", LINEAR)
def test_linear(nncu, torch_cuda, case):
    n, r, c, has_bias, has_add, slack = case
    rng = np.random.default_rng(n + r + c)
    x, w = rng.integers(-128, 128, (n, c), dtype=np.int8), rng.integers(-128, 128, (r, c), dtype=np.int8)
    xs, ws = rng.uniform(1e-3, 1, n).astype(np.float32), rng.uniform(1e-4, 1e-3, r).astype(np.float32)
    bias = rng.standard_normal(r).astype(np.float32) * 50 if has_bias else None
    add = rng.standard_normal((n, r)).astype(np.float32) * 50 if has_add else None
    got = multiplied(nncu, torch_cuda, x, xs, w, ws, bias, None if add is None else (add, has_add == 2), slack, rng)
    want, tol = H.linear(x.astype(np.float64), xs, w.astype(np.float64), ws, bias, add) if n * r * c < 1 << 22 else \
        exact_linear(torch_cuda, x, xs, w, ws, bias, add)
    assert (np.abs(got - want) <= tol).all()


def exact_linear(torch, x, xs, w, ws, bias, add):
    """H.linear with its product on the GPU: float64 sums of whole numbers below 2^53 are exact."""
    p = (dev(torch, x).double() @ dev(torch, w).double().T).cpu().numpy() * xs.astype(np.float64)[:, None] * ws.astype(np.float64)
    tol = 3 * H.U * np.abs(p)
    for more in (bias, add):
        if more is not None:
            p = p + more.astype(np.float64)
            tol = tol + H.U * np.abs(p)
    return p, 1.001 * tol + 1e-43


@pytest.mark.parametrize("n,r", [(1, 3), (20, 130), (300, 257)])
def test_linear_largest_sums(nncu, torch_cuda, n, r):
    """Codes of -128 over the longest rows: the sum is 2^31 - 2^14."""
    c = 131071
    x, w = np.full((n, c), -128, np.int8), np.full((r, c), -128, np.int8)
    one = np.ones(max(n, r), np.float32)
    got = multiplied(nncu, torch_cuda, x, one[:n], w, one[:r], None, None, 0, np.random.default_rng(0))
    assert (got == np.float32(2 ** 31 - 2 ** 14)).all()


def test_linear_rows_with_nan_scales(nncu, torch_cuda):
    """A token or a channel whose scale is NaN (a row that had a NaN) leaves the others alone."""
    rng = np.random.default_rng(3)
    x, w = rng.integers(-9, 9, (40, 64), dtype=np.int8), rng.integers(-9, 9, (200, 64), dtype=np.int8)
    xs, ws = np.ones(40, np.float32), np.ones(200, np.float32)
    xs[7], ws[130] = np.nan, np.inf
    got = multiplied(nncu, torch_cuda, x, xs, w, ws, None, None, 0, rng)
    want = x.astype(np.float64) @ w.astype(np.float64).T
    fine = np.ones((40, 200), bool)
    fine[7], fine[:, 130] = False, False
    assert np.isnan(got[7]).all() and not np.isfinite(got[:, 130]).any()
    np.testing.assert_array_equal(got[fine], want[fine])


def test_a_token_does_not_go_by_its_batch(nncu, torch_cuda):
    """The same token alone and among others (other kernels, other tiles): the same bits."""
    rng = np.random.default_rng(9)
    x, w = rng.integers(-127, 128, (600, 2048), dtype=np.int8), rng.integers(-127, 128, (700, 2048), dtype=np.int8)
    xs, ws = rng.uniform(0.01, 1, 600).astype(np.float32), rng.uniform(0.01, 1, 700).astype(np.float32)
    b = rng.standard_normal(700).astype(np.float32)
    whole = multiplied(nncu, torch_cuda, x, xs, w, ws, b, None, 0, rng)
    for lo, hi in ((0, 1), (5, 21), (100, 164), (300, 500)):
        np.testing.assert_array_equal(multiplied(nncu, torch_cuda, x[lo:hi], xs[lo:hi], w, ws, b, None, 0, rng), whole[lo:hi])


# ---- places past 32 bits ---------------------------------------------------------------------

def test_tables_past_4_gb(nncu, torch_cuda):
    """A table of 4.5 GB: rows at its end looked up and multiplied, and quantised into."""
    torch, N = torch_cuda, nncu
    rows_, cols = 1_100_000, 4096
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randint(-127, 128, (rows_, cols), generator=g, dtype=torch.int8, device="cuda")
    ws = torch.rand(rows_, generator=g, device="cuda")
    ids = torch.tensor([rows_ - 1, 0, 1 << 20, 524_287, 524_288], dtype=torch.int32, device="cuda")
    out = torch.zeros(5, cols, device="cuda")
    N.i8_lookup_dev(N.i8_lookup(n=5, cols=cols, n_rows=rows_, codes=w, scales=ws, ids=ids, out=out))
    want = w[ids.long()].double() * ws[ids.long()].double()[:, None]
    assert bool(((out.double() - want).abs() <= 2.01 * H.U * want.abs()).all())
    x = torch.randint(-127, 128, (3, cols), generator=g, dtype=torch.int8, device="cuda")
    y = torch.zeros(3, rows_, device="cuda")
    N.i8_linear_dev(N.i8_linear(n_tok=3, rows=rows_, cols=cols, x=x, x_scales=torch.ones(3, device="cuda"), w=w, w_scales=ws, y=y))
    at = torch.cat([torch.arange(0, rows_, 997, device="cuda"), torch.arange(rows_ - 300, rows_, device="cuda")])
    want = (x.double() @ w[at].double().T) * ws[at].double()
    assert bool(((y[:, at].double() - want).abs() <= 3.01 * H.U * want.abs()).all())
    f = torch.randn(2, cols, generator=g, device="cuda")
    sc = torch.zeros(2, device="cuda")
    before = w[:2].clone()
    # two rows, from the table's third to last one on
    N.i8_quantise_dev(N.i8_rows(n=2, cols=cols, x=f, codes=w[rows_ - 3:], scales=sc))
    codes, scales = H.quantise(f.cpu().numpy(), None, 0, 0.0)
    np.testing.assert_array_equal(w[rows_ - 3:rows_ - 1].cpu().numpy(), codes)
    assert torch.equal(w[:2], before)
    N.i8_check()


def test_rows_past_8_gb_apart(nncu, torch_cuda):
    """Strides whose product with a row's number passes 2^32: x, y, add and the codes of the second row."""
    torch, N = torch_cuda, nncu
    far, cols = 1 << 31, 256
    flat = torch.zeros(far + cols, device="cuda")
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, cols)).astype(np.float32)
    flat[:cols], flat[far:] = dev(torch, x[0]), dev(torch, x[1])
    codes, sc = torch.zeros(2, cols, dtype=torch.int8, device="cuda"), torch.zeros(2, device="cuda")
    N.i8_quantise_dev(N.i8_rows(n=2, cols=cols, x=flat, x_stride=far, codes=codes, scales=sc))
    check_rows(x, (codes.cpu().numpy().astype(np.int64), sc.cpu().numpy()), None, 0)
    w = rng.integers(-127, 128, (cols, cols), dtype=np.int8)
    one = torch.ones(cols, device="cuda")
    N.i8_linear_dev(N.i8_linear(n_tok=2, rows=cols, cols=cols, x=codes, x_scales=one, w=dev(torch, w), w_scales=one,
                                add=flat, add_stride=far, y=flat, y_stride=far))
    p = codes.cpu().numpy().astype(np.float64) @ w.astype(np.float64).T
    for r, got in enumerate((flat[:cols], flat[far:])):
        assert (np.abs(got.cpu().numpy() - (p[r] + x[r])) <= 1.01 * H.U * (3 * np.abs(p[r]) + np.abs(p[r] + x[r]))).all()
    N.i8_lookup_dev(N.i8_lookup(n=2, cols=cols, n_rows=2, codes=codes, scales=one, out=flat, out_stride=far))
    np.testing.assert_array_equal(flat[far:].cpu().numpy(), codes[1].cpu().numpy().astype(np.float32))
    logits = flat
    ent, ids = torch.zeros(2, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    N.logprobs_dev(N.logprobs(n=2, n_vocab=cols, logits=logits, stride=far, entropy=ent, top=3, top_ids=ids))
    for r in range(2):
        row = codes[r].cpu().numpy().astype(np.float32)
        want, off = H.logprobs(row, 1.0, -1, 3)
        np.testing.assert_array_equal(ids[r].cpu().numpy(), want["top_ids"])
        assert abs(float(ent[r]) - want["entropy"]) <= off["entropy"]
