"""The paged serving operators against plain implementations in 64 bits:
tables, rotation, the 4-bit write and read, the attention, and one step of a
layer with all of them."""
from __future__ import annotations

import numpy as np
import pytest

import paged_helpers as P

pytestmark = pytest.mark.gpu


def dev(torch, x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=dtype, device="cuda")


# ---- a step's tables: whole numbers, equal -------------------------------------------------

STEP_CASES = [
    # n_req, page, longest past, most new tokens, ended, free pages, padding of the token buffer
    (1, 16, 0, 1, 0, 1, 0),
    (1, 64, 5000, 1, 0, 0, 3),       # nothing free: served only where the last page has room
    (7, 16, 40, 5, 2, 6, 0),
    (33, 32, 300, 70, 5, 4, 9),      # runs out of pages in the middle
    (256, 64, 2000, 1, 30, 300, 0),
    (700, 128, 900, 3, 0, 900, 1),   # more requests than threads
    (513, 16, 100, 9, 513, 0, 0),    # all end
    (3, 256, 0, 0, 0, 4, 5),         # no tokens at all
    (5000, 16, 64, 2, 100, 2000, 17),  # sums in more than 48 KB of shared memory
]


def step_inputs(case, seed):
    n, page, past_hi, new_hi, ended, free, pad = case
    rng = np.random.default_rng(seed)
    past = rng.integers(0, past_hi + 1, n)
    new = rng.integers(0, new_hi + 1, n)
    new[rng.permutation(n)[:ended]] = -1
    held = -(-past // page)
    held[rng.permutation(n)[:n // 4]] += 1  # some hold a page more than their length asks for
    max_blocks = max(1, int(held.max()), int((-(-(past + np.maximum(new, 0)) // page)).max()) - (1 if n > 3 else 0))
    held = np.minimum(held, max_blocks)
    n_pages = int(held.sum()) + free + 1
    ids = rng.permutation(n_pages)
    table = np.full((n, max_blocks), -7)
    at = 0
    for r in range(n):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    head = int(rng.integers(0, n_pages))
    ring = np.full(n_pages, -9)
    for i in range(free):
        ring[(head + i) % n_pages] = ids[at + i]
    total = int(np.maximum(new, 0).sum())
    return dict(past=past, new=new, held=held, table=table, ring=ring, queue=[head, free], n_pages=n_pages,
                max_blocks=max_blocks, max_tok=max(0, total + pad - (3 if n == 7 else 0)), page=page)


@pytest.mark.parametrize("case", STEP_CASES)
def test_step_tables(nncu, torch_cuda, case):
    torch, N = torch_cuda, nncu
    s = step_inputs(case, sum(case))
    want = P.step(s["past"], s["new"], s["held"], s["queue"], s["ring"], s["table"], s["page"], s["n_pages"],
                  s["max_blocks"], s["max_tok"])
    n, i32 = case[0], torch.int32
    wide = np.full((n, s["max_blocks"] + 3), -7)  # rows further apart than they are long
    wide[:, :s["max_blocks"]] = s["table"]
    table, ring = dev(torch, wide, i32), dev(torch, s["ring"], i32)
    z = lambda k: torch.full((k + 2,), -99, dtype=i32, device="cuda")  # noqa: E731
    out = {k: z(m) for k, m in dict(held_out=n, queue_out=4, seq_len=n, q_start=n + 1, positions=s["max_tok"],
                                    slots=s["max_tok"], token_req=s["max_tok"]).items()}
    call = N.paged_step(n_req=n, page_size=s["page"], n_pages=s["n_pages"], max_blocks=s["max_blocks"],
                        max_tok=s["max_tok"], past=dev(torch, s["past"], i32), n_new=dev(torch, s["new"], i32),
                        held=dev(torch, s["held"], i32), queue=dev(torch, s["queue"], i32), ring=ring,
                        block_table=table, **out)
    N.paged_step_dev(call)
    torch.cuda.synchronize()
    got = {k: v.cpu().numpy() for k, v in out.items()}
    for name, key in (("held_out", "held"), ("queue_out", "queue"), ("seq_len",) * 2, ("q_start",) * 2,
                      ("positions",) * 2, ("slots",) * 2, ("token_req",) * 2):
        np.testing.assert_array_equal(got[name][:-2], np.asarray(want[key], np.int64), err_msg=name)
        assert (got[name][-2:] == -99).all(), name  # nothing past the end
    np.testing.assert_array_equal(table.cpu().numpy()[:, :s["max_blocks"]], np.asarray(want["table"]))
    assert (table.cpu().numpy()[:, s["max_blocks"]:] == -7).all()
    np.testing.assert_array_equal(ring.cpu().numpy(), np.asarray(want["ring"]))


def test_steps_follow_one_another(nncu, torch_cuda):
    """Pages go round: requests grow, end and come back over 40 steps, and no
    page is ever held twice or lost."""
    torch, N, i32 = torch_cuda, nncu, torch_cuda.int32
    n, page, n_pages, max_blocks, max_tok = 6, 16, 40, 12, 64
    rng = np.random.default_rng(5)
    table = torch.full((n, max_blocks), -1, dtype=i32, device="cuda")
    ring = torch.arange(n_pages, dtype=i32, device="cuda")
    a = {k: torch.zeros(m, dtype=i32, device="cuda") for k, m in
         dict(held0=n, held1=n, queue0=4, queue1=4, seq=n, start=n + 1, pos=max_tok, slot=max_tok, req=max_tok,
              past=n, new=n).items()}
    a["queue0"][1] = n_pages
    calls = [N.paged_step(n_req=n, page_size=page, n_pages=n_pages, max_blocks=max_blocks, max_tok=max_tok,
                          past=a["past"], n_new=a["new"], held=a[f"held{i}"], queue=a[f"queue{i}"], ring=ring,
                          block_table=table, held_out=a[f"held{1 - i}"], queue_out=a[f"queue{1 - i}"],
                          seq_len=a["seq"], q_start=a["start"], positions=a["pos"], slots=a["slot"],
                          token_req=a["req"]) for i in (0, 1)]
    length = np.zeros(n, np.int64)
    for it in range(40):
        new = rng.integers(0, 20, n)
        new[rng.random(n) < 0.15] = -1
        a["past"].copy_(torch.as_tensor(length, dtype=i32))
        a["new"].copy_(torch.as_tensor(new, dtype=i32))
        N.paged_step_dev(calls[it & 1])
        torch.cuda.synchronize()
        length = a["seq"].cpu().numpy().astype(np.int64)
        held = a[f"held{1 - (it & 1)}"].cpu().numpy()
        head, count = a[f"queue{1 - (it & 1)}"].cpu().numpy()[:2]
        t, r = table.cpu().numpy(), ring.cpu().numpy()
        pages = [p for i in range(n) for p in t[i, :held[i]]] + [r[(head + i) % n_pages] for i in range(count)]
        assert sorted(pages) == list(range(n_pages)), it
        assert (held * page >= length).all()
        slots = a["slot"].cpu().numpy()
        live = slots[slots >= 0]
        assert len(set(live)) == len(live)


# ---- rotation ---------------------------------------------------------------------------------

ROPE_CASES = [
    # tokens, heads, kv heads, head_dim, n_rot, mode, sections, interleaved, norm, row slack (floats)
    (1, 4, 1, 64, 64, 0, [32], 0, 1, 0),
    (5, 32, 8, 128, 128, 0, [24, 20, 20], 1, 1, 0),
    (7, 3, 3, 128, 128, 0, [16, 24, 24], 0, 0, 4),
    (3, 16, 4, 256, 64, 0, [11, 11, 10], 1, 1, 8),
    (2, 8, 4, 256, 256, 1, [64, 64], 0, 1, 0),
    (9, 5, 1, 64, 16, 1, [8], 0, 0, 0),
    (4, 2, 2, 96, 40, 0, [8, 6, 4, 2], 0, 1, 0),
    (3, 3, 1, 80, 20, 0, [10], 0, 1, 1),      # rows off the 16-byte grid, half not a multiple of 4
    (2, 1, 1, 6, 2, 1, [1], 0, 1, 0),
    (2, 2, 1, 512, 512, 0, [256], 0, 1, 0),
    (2, 2, 1, 510, 510, 1, [100, 155], 0, 1, 0),
    (3, 2, 1, 128, 0, 0, [0], 0, 1, 0),       # norm alone
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", ROPE_CASES)
def test_rope_axes(nncu, torch_cuda, case, in_place):
    torch, N = torch_cuda, nncu
    n, nh, nk, d, n_rot, mode, sections, inter, norm, slack = case
    rng = np.random.default_rng(d + n_rot + n)
    axes, half = len(sections), n_rot // 2
    pos = rng.integers(-3, 100000, (axes, n + 2))  # columns past the tokens: a row longer than n_tok
    inv = (1e4 ** (-np.arange(half) / max(half, 1))).astype(np.float32)
    axis = [i % axes if i // axes < sections[i % axes] else 0 for i in range(half)] if inter else \
        [a for a in range(axes) for _ in range(sections[a])]
    # the angle is the float32 product, by definition; the rest in 64 bits
    ang = np.stack([pos[axis[i], :n].astype(np.float32) * inv[i] for i in range(half)], 1).astype(np.float64) \
        if half else np.zeros((n, 0))
    first = np.arange(half) * (1 if mode == 0 else 2)
    second = first + (half if mode == 0 else 1)
    posd, invd = dev(torch, pos, torch.int32), dev(torch, inv if half else np.zeros(1, np.float32))
    bufs, wants, gammas = [], [], []
    for heads in (nh, nk):
        x = rng.standard_normal((n, heads * d + slack)).astype(np.float32) * 3
        g = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32)
        y = x[:, :heads * d].astype(np.float64).reshape(n, heads, d)
        if norm:
            y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + 1e-6) * g
        z = y.copy()
        a, b, c, s = y[..., first], y[..., second], np.cos(ang)[:, None], np.sin(ang)[:, None]
        z[..., first], z[..., second] = a * c - b * s, a * s + b * c
        # per value: the norm (a sum of d squares, a root, two products), sine and cosine to two units, two
        # products and a sum: under 24 half-units of the pair's size
        tol = np.abs(y) * 24 * 2.0 ** -24
        tol[..., first] = tol[..., second] = (np.abs(a) + np.abs(b)) * 24 * 2.0 ** -24
        bufs.append(dev(torch, x))
        gammas.append(dev(torch, g) if norm else None)
        wants.append((z, tol + 1e-30))
    outs = bufs if in_place else [torch.full((n, b.shape[1] + 4), 7.0, device="cuda") for b in bufs]
    call = N.rope_axes(n_tok=n, n_head=nh, n_kv=nk, head_dim=d, positions=posd, inv_freq=invd, q=bufs[0], k=bufs[1],
                       q_out=outs[0], k_out=outs[1], n_rot=n_rot, rope_mode=mode, sections=sections,
                       interleaved=inter, q_gamma=gammas[0], k_gamma=gammas[1], eps=1e-6)
    N.rope_axes_dev(call)
    torch.cuda.synchronize()
    for out, heads, (want, tol) in zip(outs, (nh, nk), wants):
        got = out.cpu().numpy()
        if not in_place:
            assert (got[:, heads * d:] == 7.0).all()
        err = np.abs(got[:, :heads * d].reshape(n, heads, d) - want)
        assert (err <= tol).all(), float((err / tol).max())


def test_rope_axes_of_one_axis_is_rope_dev(nncu, torch_cuda):
    """Consecutive positions on one axis: the framework's own rotation."""
    torch, N = torch_cuda, nncu
    n, heads, d, base = 6, 4, 128, 1e6
    x = torch.randn(n, heads * d, device="cuda")
    y = x.clone()
    N.rope_dev(y, n, heads, d, d, 17, 1.0, base)
    # float32 recurrence of the reference: inv[i] = inv[i - 1] * base^(-2 / n_rot); compared through its values
    inv = dev(torch, (base ** (-np.arange(d // 2, dtype=np.float64) * 2 / d)).astype(np.float32))
    z = torch.empty_like(x)
    N.rope_axes_dev(N.rope_axes(n_tok=n, n_head=heads, n_kv=0, head_dim=d,
                                positions=dev(torch, np.arange(17, 17 + n), torch.int32), inv_freq=inv, q=x, q_out=z))
    torch.cuda.synchronize()
    # the recurrence is up to 64 roundings off (64 * 2^-24), times positions up to 22
    assert float((y - z).abs().max()) <= 64 * 2.0 ** -24 * 22 * float(x.abs().max()) * 1.5


# ---- the 4-bit write and read: equal ------------------------------------------------------------

APPEND_CASES = [(1, 1, 64, 16), (3, 2, 128, 32), (17, 1, 256, 64), (65, 3, 64, 128), (33, 8, 128, 256), (130, 2, 256, 16)]


@pytest.mark.parametrize("slack", [0, 12])
@pytest.mark.parametrize("case", APPEND_CASES)
def test_append_and_read(nncu, torch_cuda, case, slack):
    torch, N = torch_cuda, nncu
    n, n_kv, d, page = case
    rng = np.random.default_rng(n * d + page)
    n_pages = -(-n // page) + 2
    pool = P.Pool(n_pages, page, n_kv, d, rng)
    slots = rng.permutation(n_pages * page)[:n].astype(np.int64)
    if n > 3:
        slots[1], slots[2] = -1, n_pages * page + 5  # skipped: none, and outside the pool
    rows = [rng.standard_normal((n, n_kv * d + slack)).astype(np.float32) for _ in range(2)]
    x = rows[0]
    if n > 16:  # the form's edges, each in a group of its own
        x[3, :32] = 0.0
        x[4, :32] = np.nan
        x[5, 1], x[5, 40] = np.inf, -np.inf
        x[6, :32] *= 1e30                                  # saturates
        x[7, :32] *= 1e-30                                 # below the smallest scale
        x[8, :32] = np.where(np.arange(32) % 2, 1.5, -1.5)  # the largest magnitude with both signs
        x[9, :32] = np.arange(32) - 16                     # ties between codes
        x[10, :32] = -0.0
    pages = dev(torch, pool.bytes)
    p = N.kv4_pool(pages, n_pages, page, n_kv, d)
    sd = dev(torch, slots, torch.int32)
    N.kv4_append_dev(N.kv4_rows(p, slots=sd, n_tok=n, k=dev(torch, rows[0]), v=dev(torch, rows[1])))
    back = [torch.full((n, n_kv * d + slack), 3.0, device="cuda") for _ in range(2)]
    N.kv4_read_dev(N.kv4_rows(p, slots=sd, n_tok=n, k=back[0], v=back[1]))
    torch.cuda.synchronize()
    for which in range(2):
        c, s = P.quantise(rows[which][:, :n_kv * d].reshape(n, n_kv, d))
        want = P.value(c, s)
        for t in range(n):
            if not 0 <= slots[t] < n_pages * page:
                want[t] = 0.0
                continue
            for h in range(n_kv):
                pool.put(int(slots[t]), h, which, c[t, h], s[t, h])
        got = back[which].cpu().numpy()
        np.testing.assert_array_equal(got[:, :n_kv * d].reshape(n, n_kv, d), want.astype(np.float32))
        assert (got[:, n_kv * d:] == 3.0).all()
    got = pages.cpu().numpy()
    np.testing.assert_array_equal(got, pool.bytes)  # the layout itself, and nothing else touched


def test_append_of_one_side(nncu, torch_cuda):
    torch, N = torch_cuda, nncu
    pool = P.Pool(2, 16, 2, 64, np.random.default_rng(1))
    pages = dev(torch, pool.bytes)
    p = N.kv4_pool(pages, 2, 16, 2, 64)
    sd = dev(torch, [5, 20], torch.int32)
    x = torch.randn(2, 128, device="cuda")
    N.kv4_append_dev(N.kv4_rows(p, slots=sd, n_tok=2, v=x))
    y = torch.empty_like(x)
    N.kv4_read_dev(N.kv4_rows(p, slots=sd, n_tok=2, v=y))
    torch.cuda.synchronize()
    c, s = P.quantise(x.cpu().numpy().reshape(2, 2, 64))
    np.testing.assert_array_equal(y.cpu().numpy().reshape(2, 2, 64), P.value(c, s).astype(np.float32))
    half = 16 * 64 // 2
    np.testing.assert_array_equal(pages.cpu().numpy()[..., :half], pool.bytes[..., :half])  # K untouched


# ---- attention ---------------------------------------------------------------------------------

ATTN_CASES = [
    # (keys, new tokens) of each request; KV heads, group, head_dim, page, window, softcap
    ([(1, 1)], 1, 1, 64, 16, 0, 0.0),
    ([(1, 1), (2, 1), (63, 1), (64, 1), (65, 1)], 2, 4, 128, 64, 0, 0.0),
    ([(300, 1), (17, 1), (0, 0), (129, 1), (5, 0)], 8, 4, 128, 16, 0, 0.0),  # requests without tokens, without keys
    ([(1000, 4)], 4, 2, 256, 128, 0, 0.0),
    ([(777, 5), (33, 5), (5, 5), (200, 3)], 2, 4, 64, 16, 100, 30.0),
    ([(2500, 1), (90, 1)], 1, 8, 128, 32, 0, 0.0),
    ([(600, 7)], 2, 7, 64, 256, 0, 0.0),
    ([(700, 2), (256, 1)], 1, 4, 256, 64, 256, 0.0),
    ([(513, 3)], 1, 12, 128, 64, 1, 0.0),      # each query sees itself alone
    ([(100, 33), (64, 64), (257, 40)], 2, 4, 128, 64, 0, 0.0),
    ([(500, 200), (130, 130)], 2, 4, 128, 16, 77, 0.0),
    ([(300, 150)], 1, 2, 256, 32, 0, 20.0),
    ([(333, 222), (10, 1)], 2, 4, 64, 64, 0, 0.0),
    ([(140, 140)], 1, 16, 64, 128, 0, 0.0),
    ([(130, 129)], 3, 1, 128, 64, 0, 0.0),
    ([(4000, 1)] + [(40 + 3 * i, 1) for i in range(30)], 1, 4, 64, 16, 0, 0.0),
    ([(3, 5), (0, 2), (40, 41)], 2, 2, 128, 64, 0, 0.0),  # more tokens than keys: the first see none
    ([(3, 70), (150, 60)], 2, 2, 128, 64, 0, 0.0),        # the same among many rows
    ([(200, 24), (200, 25), (90, 1)], 1, 4, 128, 64, 0, 0.0),
    ([(200, 48), (200, 49), (90, 1)], 1, 4, 128, 64, 0, 0.0),  # 192 and 196 rows a KV head: one kernel and the other
    ([(200, 64), (200, 65)], 1, 4, 64, 32, 0, 0.0),
    ([(200, 32), (200, 33)], 1, 4, 256, 64, 0, 0.0),
]
# enough key tiles for several row tiles a segment: 8, 16, 24, 32 rows and more
ATTN_MANY = [([(60 + 7 * (i % 9), n) for i in range(300)], 8, g, d, 64, 0, 0.0)
             for n, g, d in ((2, 2, 64), (3, 4, 64), (4, 4, 64), (5, 4, 64), (9, 4, 64), (4, 4, 128), (5, 4, 128))]


class Attn:
    """One case on the device: a pool in use, its requests' tables, q rows and the wanted output."""

    def __init__(self, torch, N, case, seed=3, slack=0, k_scale=1.0, spoil=None):
        reqs, self.n_kv, self.group, self.d, self.page, window, softcap = case
        rng = np.random.default_rng(seed)
        d, page, n_kv = self.d, self.page, self.n_kv
        blocks = [-(-k // page) for k, _ in reqs]
        self.n_pages = sum(blocks) + 2
        pool = P.Pool(self.n_pages, page, n_kv, d, rng)
        ids = rng.permutation(self.n_pages)
        mb = max(max(blocks), 1)
        table = np.full((len(reqs), mb + 1), -1)
        start = np.concatenate([[0], np.cumsum([n for _, n in reqs])])
        n_tok, nh = int(start[-1]), n_kv * self.group
        q = (rng.standard_normal((n_tok, nh * d + slack)) * 2).astype(np.float32)
        want = np.zeros((n_tok, nh * d))
        self.vmax, at = 0.0, 0
        for r, (keys, new) in enumerate(reqs):
            table[r, :blocks[r]] = ids[at:at + blocks[r]]
            at += blocks[r]
            x = rng.standard_normal((2, keys, n_kv, d)).astype(np.float32)
            x[0] *= k_scale
            if spoil:
                spoil(x, r)
            c, s = P.quantise(x)
            kv = P.value(c, s)
            for k in range(keys):
                for h in range(n_kv):
                    for w in range(2):
                        pool.put(int(table[r, k // page]) * page + k % page, h, w, c[w, k, h], s[w, k, h])
            self.vmax = max(self.vmax, float(np.nanmax(np.abs(kv[1]), initial=0.0)))
            for t in range(new):
                for h in range(nh):
                    row = q[start[r] + t, h * d:(h + 1) * d]
                    want[start[r] + t, h * d:(h + 1) * d] = P.attention(
                        row, kv[0][:, h // self.group], kv[1][:, h // self.group], keys - new + t, window,
                        d ** -0.5, softcap)
        self.want, self.n_tok, self.q = want, n_tok, q
        i32 = torch.int32
        self.out = torch.full((max(n_tok, 1) + 1, nh * d + slack), 5.0, device="cuda")
        self.pages = dev(torch, pool.bytes)
        self.call = N.kv4_attn(N.kv4_pool(self.pages, self.n_pages, page, n_kv, d), n_req=len(reqs), n_tok=n_tok,
                               n_head=nh, max_new=max(n for _, n in reqs), max_blocks=mb,
                               block_table=dev(torch, table, i32), seq_len=dev(torch, [k for k, _ in reqs], i32),
                               q_start=dev(torch, start, i32), q=dev(torch, q), out=self.out, softcap=softcap,
                               window=window)
        self.ws = torch.zeros(N.kv4_workspace_bytes(self.call), dtype=torch.uint8, device="cuda")
        self.call.workspace, self.call.workspace_bytes = self.ws.data_ptr(), self.ws.numel()

    # Scores of size up to 40 in base 2 carry 40 * 2^-24 from their rounding and as much from the products' sums, the
    # exponential 2^-22, the two 16-bit halves of q and of the weights 2^-21: weights are good to 6e-6, and an output
    # is a mean of values no larger than vmax.
    def check(self, got, tol=1e-5):
        nhd = self.want.shape[1]
        got = got.cpu().numpy()
        assert (got[self.n_tok:] == 5.0).all() and (got[:, nhd:] == 5.0).all()
        err = np.abs(got[:self.n_tok, :nhd].astype(np.float64) - self.want)
        assert err.max(initial=0.0) <= tol * max(self.vmax, 1e-30), (float(err.max()), self.vmax)


@pytest.mark.parametrize("slack", [0, 8])
@pytest.mark.parametrize("case", ATTN_CASES, ids=lambda c: f"{len(c[0])}req-{c[0][0]}-kv{c[1]}x{c[2]}-d{c[3]}-p{c[4]}-w{c[5]}")
def test_attention(nncu, torch_cuda, case, slack):
    a = Attn(torch_cuda, nncu, case, slack=slack)
    nncu.kv4_attention_dev(a.call)
    nncu.kv4_check(a.call)
    a.check(a.out)


@pytest.mark.parametrize("case", ATTN_MANY, ids=lambda c: f"{c[0][0][1]}x{c[2]}-d{c[3]}")
def test_attention_of_many_requests(nncu, torch_cuda, case):
    """A few of many requests checked (the table and lengths of all are live; the pool holds what the few see)."""
    torch = torch_cuda
    reqs, n_kv, g, d, page, _, _ = case
    few = Attn(torch, nncu, (reqs[:3],) + case[1:])
    keep = few.call._keep
    n, new, mb = len(reqs), reqs[0][1], few.call.max_blocks
    table = keep["block_table"][:, :mb].repeat(n // 3, 1).contiguous()
    seq = keep["seq_len"].repeat(n // 3)
    q = few.call._keep["q"].repeat(n // 3, 1).contiguous()
    out = torch.zeros_like(q)
    start = torch.arange(0, n * new + 1, new, dtype=torch.int32, device="cuda")
    wide = 16 * mb  # a table with room: what the call can know of the lengths
    roomy = torch.full((n, wide), -1, dtype=torch.int32, device="cuda")
    roomy[:, :mb] = table
    call = nncu.kv4_attn(few.call.pool, n_req=n, n_tok=n * new, n_head=n_kv * g, max_new=new, max_blocks=wide,
                         block_table=roomy, seq_len=seq, q_start=start, q=q, out=out)
    ws = torch.zeros(nncu.kv4_workspace_bytes(call), dtype=torch.uint8, device="cuda")
    call.workspace, call.workspace_bytes = ws.data_ptr(), ws.numel()
    nncu.kv4_attention_dev(call)
    nncu.kv4_check(call)
    got = out.view(n // 3, 3 * new, -1)
    want = torch.as_tensor(few.want, device="cuda")
    assert float((got.double() - want).abs().max()) <= 1e-5 * few.vmax


@pytest.mark.parametrize("case", [ATTN_CASES[1], ATTN_CASES[4], ATTN_CASES[9], ATTN_CASES[15]])
def test_attention_again_is_the_same(nncu, torch_cuda, case):
    """The workspace is left ready, and no sum depends on the order in which
    blocks finish: ten calls, on a stream of their own, bit for bit."""
    torch = torch_cuda
    a = Attn(torch, nncu, case)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    outs = []
    with torch.cuda.stream(st):
        for _ in range(10):
            nncu.kv4_attention_dev(a.call, st)
            outs.append(a.out.clone())
    torch.cuda.synchronize()
    a.check(outs[0])
    assert all(torch.equal(o, outs[0]) for o in outs[1:])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_one_workspace_for_all_row_counts(nncu, torch_cuda, d):
    """Decode, verify and prompt calls share a workspace in turn."""
    torch = torch_cuda
    cases = [Attn(torch, nncu, ([(900, n), (333, n)], 2, 4, d, 64, 0, 0.0), seed=n) for n in (1, 3, 60, 8)]
    ws = max((a.ws for a in cases), key=lambda w: w.numel())
    for a in cases + cases[::-1] + cases:
        a.call.workspace, a.call.workspace_bytes = ws.data_ptr(), ws.numel()
        a.out.fill_(5.0)
        nncu.kv4_attention_dev(a.call)
        a.check(a.out)


@pytest.mark.parametrize("case", [([(2100, 70), (1500, 45)], 1, 4, 128, 64, 0, 0.0), ([(1400, 40)], 2, 2, 256, 16, 0, 0.0),
                                  ([(2600, 90), (40, 33)], 1, 4, 64, 32, 1100, 0.0)])
def test_prompts_over_long_spans(nncu, torch_cuda, case):
    """Spans of many tiles: sums that start anew on their way, and pieces that meet."""
    a = Attn(torch_cuda, nncu, case)
    nncu.kv4_attention_dev(a.call)
    nncu.kv4_check(a.call)
    a.check(a.out)


@pytest.mark.parametrize("k_scale", [1e-4, 30.0])
def test_attention_of_flat_and_sharp_scores(nncu, torch_cuda, k_scale):
    """Near-equal weights, and one key that outweighs all others. Scores reach
    30 * 60 / ln 2: 2600 * 2^-23 of a weight."""
    a = Attn(torch_cuda, nncu, ([(900, 1), (130, 40)], 2, 4, 128, 64, 0, 0.0), k_scale=k_scale)
    nncu.kv4_attention_dev(a.call)
    torch_cuda.cuda.synchronize()
    a.check(a.out, tol=1e-5 if k_scale < 1 else 4e-4)


def test_attention_weights_far_below_the_largest(nncu, torch_cuda):
    """One key holds half the weight, 3000 others e^-8.3 of it each: weights
    near 2^-12 carry as many digits as the large one."""
    def spoil(x, r):
        x[0] *= 0.02
        x[0, 7] = np.sign(x[0, 7]) * 2.0
        x[1] = 1.0 + 0.05 * x[1]

    torch = torch_cuda
    a = Attn(torch, nncu, ([(3000, 1)], 1, 1, 128, 64, 0, 0.0), spoil=spoil)
    nncu.kv4_attention_dev(a.call)
    torch.cuda.synchronize()
    a.check(a.out)


@pytest.mark.parametrize("n_new", [1, 60])
def test_a_bad_key_spoils_only_who_sees_it(nncu, torch_cuda, n_new):
    """A key with a NaN: queries before it, and those whose window has passed
    it, are untouched; V's NaN stays in its group of 32 values."""
    def spoil(x, r):
        if x.shape[1] > 50:
            x[0, 50, 0, 3] = np.nan
        x[1, 10, 0, 40] = np.inf

    torch = torch_cuda
    for keys in (40 + n_new, 140 + n_new):
        a = Attn(torch, nncu, ([(keys, n_new)], 1, 4, 128, 16, 64, 0.0), spoil=spoil)
        nncu.kv4_attention_dev(a.call)
        torch.cuda.synchronize()
        got = a.out.cpu().numpy()[:n_new]
        assert (np.isnan(got) == np.isnan(a.want)).all()
        fine = ~np.isnan(a.want)
        assert np.abs(got - a.want)[fine].max(initial=0.0) <= 1e-5 * a.vmax


def test_keys_on_no_page_are_not_seen(nncu, torch_cuda):
    """A table entry outside the pool hides its page's keys."""
    torch = torch_cuda
    case = ([(200, 1), (90, 50)], 2, 4, 64, 16, 0, 0.0)
    a = Attn(torch, nncu, case)
    nncu.kv4_attention_dev(a.call)
    ref = a.out.clone()
    t = a.call._keep["block_table"]
    keep = t.clone()
    t[0, :] = torch.tensor([-1, 10 ** 6], dtype=torch.int32, device="cuda")[torch.arange(t.shape[1], device="cuda") % 2]
    nncu.kv4_attention_dev(a.call)
    torch.cuda.synchronize()
    assert float(a.out[0, :a.want.shape[1]].abs().max()) == 0.0  # request 0 sees nothing
    assert torch.equal(a.out[1:], ref[1:])
    t.copy_(keep)
    nncu.kv4_attention_dev(a.call)
    torch.cuda.synchronize()
    assert torch.equal(a.out, ref)


def test_attention_leaves_out_what_passes_its_bounds(nncu, torch_cuda):
    """max_new and n_tok bound what is computed; nothing else is written."""
    torch = torch_cuda
    a = Attn(torch, nncu, ([(100, 6), (70, 3)], 1, 4, 128, 64, 0, 0.0))
    a.call.max_new = 4
    nncu.kv4_attention_dev(a.call)
    torch.cuda.synchronize()
    got = a.out.cpu().numpy()
    rows = [0, 1, 2, 3, 6, 7, 8]
    assert np.abs(got[rows] - a.want[rows]).max() <= 1e-5 * a.vmax
    assert (got[[4, 5, 9]] == 5.0).all()
    a.out.fill_(5.0)
    a.call.max_new, a.call.n_tok = 6, 7
    nncu.kv4_attention_dev(a.call)
    torch.cuda.synchronize()
    got = a.out.cpu().numpy()
    assert np.abs(got[:7] - a.want[:7]).max() <= 1e-5 * a.vmax and (got[7:] == 5.0).all()


@pytest.mark.parametrize("seq,rows", [(2 ** 31 - 1, 64 * 2), (-5, 0), (1000, 64 * 2)])
def test_lengths_no_table_can_hold(nncu, torch_cuda, seq, rows):
    """A seq_len past the table row counts as the row's end, a negative one as none: nothing is read beyond."""
    torch = torch_cuda
    for new in (1, 50):
        a = Attn(torch, nncu, ([(128, new)], 1, 4, 128, 64, 100, 0.0))
        a.call._keep["seq_len"].fill_(seq)
        nncu.kv4_attention_dev(a.call)
        nncu.kv4_check(a.call)
        if rows:
            a.check(a.out)
        else:
            assert float(a.out[:new].abs().max()) == 0.0


def test_attention_in_a_graph_follows_new_lengths(nncu, torch_cuda):
    """Lengths are read on the device: a captured call replays with others."""
    torch = torch_cuda
    a = Attn(torch, nncu, ([(700, 1), (300, 1)], 2, 4, 128, 64, 0, 0.0))
    nncu.kv4_attention_dev(a.call)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        nncu.kv4_attention_dev(a.call, torch.cuda.current_stream())
    seq = a.call._keep["seq_len"]
    seq.copy_(torch.tensor([123, 300], dtype=torch.int32))
    a.out.fill_(5.0)
    g.replay()
    torch.cuda.synchronize()
    short = a.out.clone()
    assert torch.isfinite(short).all()
    nncu.kv4_attention_dev(a.call)
    torch.cuda.synchronize()
    assert torch.equal(short, a.out)
    seq.copy_(torch.tensor([700, 300], dtype=torch.int32))
    g.replay()
    torch.cuda.synchronize()
    a.check(a.out)


# ---- a step of a layer: tables, rotation, write, attention ------------------------------------------


@pytest.mark.parametrize("d", [64, 128, 256])
def test_serving_steps(nncu, torch_cuda, d):
    """Three requests prompted and decoded through the four operators, against
    the same steps written out: rotated rows quantised, attended in 64 bits."""
    torch, N, i32 = torch_cuda, nncu, torch_cuda.int32
    n_req, n_kv, group, page, n_pages, max_blocks, max_tok = 3, 2, 2, 16, 40, 12, 160
    rng = np.random.default_rng(d)
    nh = n_kv * group
    z = lambda *k: torch.zeros(*k, dtype=i32, device="cuda")  # noqa: E731
    pages = torch.randint(0, 256, (N.kv4_bytes(n_pages, page, n_kv, d),), dtype=torch.uint8, device="cuda")
    pool = N.kv4_pool(pages, n_pages, page, n_kv, d)
    t = dict(past=z(n_req), new=z(n_req), held0=z(n_req), held1=z(n_req), queue0=z(4), queue1=z(4), seq=z(n_req),
             start=z(n_req + 1), pos=z(max_tok), slot=z(max_tok), req=z(max_tok), table=z(n_req, max_blocks),
             ring=torch.arange(n_pages, dtype=i32, device="cuda"))
    t["queue0"][1] = n_pages
    q, k, v = (torch.zeros(max_tok, h * d, device="cuda") for h in (nh, n_kv, n_kv))
    out = torch.zeros_like(q)
    half = d // 2
    inv = (1e4 ** (-np.arange(half) / half)).astype(np.float32)
    steps = [N.paged_step(n_req=n_req, page_size=page, n_pages=n_pages, max_blocks=max_blocks, max_tok=max_tok,
                          past=t["past"], n_new=t["new"], held=t[f"held{i}"], queue=t[f"queue{i}"], ring=t["ring"],
                          block_table=t["table"], held_out=t[f"held{1 - i}"], queue_out=t[f"queue{1 - i}"],
                          seq_len=t["seq"], q_start=t["start"], positions=t["pos"], slots=t["slot"],
                          token_req=t["req"]) for i in (0, 1)]
    rope = N.rope_axes(n_tok=max_tok, n_head=nh, n_kv=n_kv, head_dim=d, positions=t["pos"], inv_freq=dev(torch, inv),
                       q=q, k=k)
    rows = N.kv4_rows(pool, slots=t["slot"], n_tok=max_tok, k=k, v=v)
    attn = N.kv4_attn(pool, n_req=n_req, n_tok=max_tok, n_head=nh, max_new=max_tok, max_blocks=max_blocks,
                      block_table=t["table"], seq_len=t["seq"], q_start=t["start"], q=q, out=out)
    ws = torch.zeros(N.kv4_workspace_bytes(attn), dtype=torch.uint8, device="cuda")
    attn.workspace, attn.workspace_bytes = ws.data_ptr(), ws.numel()
    cache = [[np.zeros((0, n_kv, d)) for _ in range(2)] for _ in range(n_req)]
    for it, new in enumerate([[37, 1, 90], [1, 1, 1], [1, 20, 1], [3, 1, -1], [1, 1, 50]]):
        lens = np.array([c[0].shape[0] for c in cache])
        t["past"].copy_(torch.as_tensor(lens, dtype=i32))
        t["new"].copy_(torch.as_tensor(new, dtype=i32))
        host = [rng.standard_normal((max_tok, h * d)).astype(np.float32) for h in (nh, n_kv, n_kv)]
        for x, y in zip((q, k, v), host):
            x.copy_(torch.as_tensor(y))
        N.paged_step_dev(steps[it & 1])
        N.rope_axes_dev(rope)
        N.kv4_append_dev(rows)
        N.kv4_attention_dev(attn)
        torch.cuda.synchronize()
        at = 0
        # rotated rows as the device has them (float32): the codes of a value at a tie follow them
        kr, qr, got = k.cpu().numpy(), q.cpu().numpy(), out.cpu().numpy()
        for r, n in enumerate(new):
            if n < 0:
                cache[r] = [np.zeros((0, n_kv, d)) for _ in range(2)]
                continue
            ang = ((lens[r] + np.arange(n)).astype(np.float32)[:, None] * inv).astype(np.float64)
            for x, y, h in ((kr, host[1], n_kv), (qr, host[0], nh)):
                y = y[at:at + n].astype(np.float64).reshape(n, h, d)
                c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
                turned = np.concatenate([y[..., :half] * c - y[..., half:] * s, y[..., :half] * s + y[..., half:] * c], -1)
                assert np.abs(x[at:at + n].reshape(n, h, d) - turned).max() <= 24 * 2.0 ** -24 * 2 * np.abs(y).max()
            for w, x in enumerate((kr, host[2])):
                rowsq = P.value(*P.quantise(x[at:at + n].reshape(n, n_kv, d)))
                cache[r][w] = np.concatenate([cache[r][w], rowsq])
            vmax = np.abs(cache[r][1]).max()
            for i in range(n):
                for h in range(nh):
                    want = P.attention(qr[at + i, h * d:(h + 1) * d], cache[r][0][:, h // group],
                                       cache[r][1][:, h // group], int(lens[r]) + i, 0, d ** -0.5, 0.0)
                    assert np.abs(got[at + i, h * d:(h + 1) * d] - want).max() <= 1e-5 * vmax, (it, r, i, h)
            at += n


def test_the_serving_command(nncu, torch_cuda, capsys):
    import json

    from libllmcpu_b200 import paged_bench

    assert paged_bench.main(["--model", "llama3.2-1b", "--requests", "5", "--context", "300", "--page", "16",
                             "--steps", "7", "--tokens", "2"]) == 0
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert set(line["operators_us"]) == {"tables", "rope", "append", "attention"} and line["step_us"] > 0
