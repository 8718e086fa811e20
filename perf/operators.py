"""The paged serving operators, measured: block tables and slot maps, rotary
positions with several axes, the 4-bit cache's write and read-back, and the
attention over that cache.

``listed()`` names the cases, ``draw(rng)`` makes more of the same ranges,
``prepare(case, seed)`` the inputs, ``run(state)`` one pass: with ``own`` the
framework's calls, otherwise the operators' plain form in elementary torch
operations (32 bits). ``exact(case, seed)`` is the definition in 64 bits.

The cache, one uint8 array ``[n_pages][n_kv][chunk]`` per layer: a chunk holds
a page's keys of one KV head as K codes, V codes (``page x head_dim / 2``
bytes each), K scales, V scales (bf16, one per 32 values). A key's row of
codes is ``U = head_dim / 32`` units of 16 bytes, one per group of 32 values;
unit g of key k sits at place ``g ^ ((k * head_dim / 2 / 128) % U)``. The 32-bit
word w of a unit holds values 8w .. 8w + 7, nibble n the value ``8w + 2 (n % 4)
+ n / 4``, as code + 8.
"""
from __future__ import annotations

import math
import random

import torch

own = False

GROUP = 32
NIBBLE = [0, 2, 4, 6, 1, 3, 5, 7]  # the value (of its eight) that nibble n of a word holds


# ---- the cases -----------------------------------------------------------------------------


def listed():
    # heads: Qwen3-8B 32/8 x 128, Gemma-3-4B 8/4 x 256, Llama-3.2-1B 32/8 x 64, Qwen3.5-4B 16/4 x 256
    return [
        # one decode step's tables for a full serving batch: the small call, latency counts
        dict(name="step decode 256", op="step", n_req=256, page=64, past_lo=1, past_hi=8192, new_lo=1, new_hi=1,
             ended=8, spare=64, pad=0),
        # prompts admitted together with running requests, small pages, a padded token buffer
        dict(name="step prompts 60", op="step", n_req=60, page=16, past_lo=1, past_hi=2000, new_lo=1, new_hi=4096,
             ended=3, spare=8192, pad=500),
        # a decode batch's q and k: per-head norms and one position axis
        dict(name="rope decode 64x32/8x128", op="rope", n_tok=64, n_head=32, n_kv=8, head_dim=128, n_rot=128, axes=1,
             interleaved=0, norm=1, neox=1, pos_hi=32768),
        # a prompt with an image in it: time, height and width, interleaved
        dict(name="rope image 8192x16/4x256", op="rope", n_tok=8192, n_head=16, n_kv=4, head_dim=256, n_rot=64,
             axes=3, interleaved=1, norm=1, neox=1, pos_hi=32768),
        # a decode batch's new rows into the cache (and read back)
        dict(name="append 64x8x128", op="append", n_tok=64, n_kv=8, head_dim=128, page=64, skipped=2),
        # a prompt's rows, small pages, an odd number of tokens
        dict(name="append 8191x4x256", op="append", n_tok=8191, n_kv=4, head_dim=256, page=16, skipped=5),
        # one user decoding: latency
        dict(name="decode 1x4096 32/8x128", op="attention", n_req=1, n_head=32, n_kv=8, head_dim=128, page=64,
             len_lo=4096, len_hi=4096, new_lo=1, new_hi=1, window=0, softcap=0.0),
        # a serving batch of ragged requests decoding
        dict(name="decode 64x512-8192 32/8x128", op="attention", n_req=64, n_head=32, n_kv=8, head_dim=128, page=64,
             len_lo=512, len_hi=8192, new_lo=1, new_hi=1, window=0, softcap=0.0),
        # one long context, four speculated tokens verified
        dict(name="verify 1x131072 8/4x256", op="attention", n_req=1, n_head=8, n_kv=4, head_dim=256, page=128,
             len_lo=131072, len_hi=131072, new_lo=4, new_hi=4, window=0, softcap=0.0),
        # a batch verifying five tokens through a sliding window, small pages, odd lengths, a score soft-cap
        dict(name="window 33x700-5000 32/8x64", op="attention", n_req=33, n_head=32, n_kv=8, head_dim=64, page=16,
             len_lo=700, len_hi=5000, new_lo=5, new_hi=5, window=1024, softcap=30.0),
        # prompts of several users packed together, some with a cached prefix
        dict(name="prompts 6x200-2048 32/8x128", op="attention", n_req=6, n_head=32, n_kv=8, head_dim=128, page=64,
             len_lo=777, len_hi=4096, new_lo=200, new_hi=2048, window=0, softcap=0.0),
        # one long prompt's chunk over what is cached already
        dict(name="chunk 1x1000+15000 8/4x256", op="attention", n_req=1, n_head=8, n_kv=4, head_dim=256, page=64,
             len_lo=16000, len_hi=16000, new_lo=1000, new_hi=1000, window=0, softcap=0.0),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "rope", "append", "attention", "attention", "attention"])
    if op == "step":
        n_req = _spread(rng, 1, 512)
        new_hi = rng.choice([1, 8, max(1, min(4096, 65536 // n_req))])
        return dict(op=op, n_req=n_req, page=rng.choice([16, 32, 64, 128]), past_lo=1, past_hi=_spread(rng, 64, 8192),
                    new_lo=1, new_hi=new_hi, ended=rng.randint(0, n_req // 4), spare=_spread(rng, 1, 8192),
                    pad=rng.choice([0, 0, _spread(rng, 1, 512)]))
    n_kv, group, head_dim = rng.choice([(8, 4, 128), (4, 2, 256), (8, 4, 64), (4, 4, 256), (1, 4, 256), (2, 7, 64),
                                        (8, 8, 128), (3, 1, 128)])
    if op == "rope":
        half = rng.choice([head_dim // 2, head_dim // 8])
        return dict(op=op, n_tok=_spread(rng, 1, 8192), n_head=n_kv * group, n_kv=n_kv, head_dim=head_dim,
                    n_rot=2 * half, axes=rng.choice([1, 2, 3]), interleaved=rng.randint(0, 1), norm=rng.randint(0, 1),
                    neox=rng.randint(0, 1), pos_hi=_spread(rng, 16, 131072))
    if op == "append":
        n_tok = _spread(rng, 1, 8192)
        return dict(op=op, n_tok=n_tok, n_kv=n_kv, head_dim=head_dim, page=rng.choice([16, 32, 64, 128]),
                    skipped=rng.randint(0, min(8, n_tok - 1)))
    kind = rng.choice(["decode", "decode", "verify", "prompt"])
    if kind == "prompt":
        n_req = _spread(rng, 1, 8)
        new_hi = _spread(rng, 33, 2048 // n_req + 100)
        len_hi = _spread(rng, new_hi, 8192)
    else:
        n_req = _spread(rng, 1, 64)
        new_hi = 1 if kind == "decode" else rng.randint(2, 8)
        len_hi = _spread(rng, 16, 131072 // n_req)
    return dict(op=op, n_req=n_req, n_head=n_kv * group, n_kv=n_kv, head_dim=head_dim,
                page=rng.choice([16, 32, 64, 128]), len_lo=max(1, len_hi // rng.choice([1, 3, 16])), len_hi=len_hi,
                new_lo=max(1, new_hi // rng.choice([1, 4])), new_hi=new_hi,
                window=rng.choice([0, 0, _spread(rng, 16, 4096)]), softcap=rng.choice([0.0, 0.0, 50.0]))


def _sizes(lo, hi, n, step):
    """n whole numbers over [lo, hi], even over the logarithm, in a fixed mixed order: the lengths are the case's, not
    the seed's."""
    if n == 1:
        return [hi]
    s = [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    while math.gcd(step, n) != 1:
        step += 1
    return [s[(i * step) % n] for i in range(n)]


def _requests(case):
    """(keys, new tokens) of each request of an attention case."""
    new = _sizes(case["new_lo"], case["new_hi"], case["n_req"], 5)
    keys = _sizes(case["len_lo"], case["len_hi"], case["n_req"], 7)
    return [(max(k, n), n) for k, n in zip(keys, new)]


def _visible(first, last, window):
    """Keys seen by the queries at positions first .. last together."""
    n, w = last - first + 1, window
    if not w or last < w:
        return n * (first + 1 + last + 1) // 2
    full = min(n, last - w + 2 if last >= w else 0)  # queries at w - 1 and after see w keys
    rest = n - full
    return full * w + rest * (first + 1 + first + rest) // 2


def work(case):
    if case["op"] == "step":
        n, new = case["n_req"], sum(_step_lengths(case)[1])
        total = sum(max(x, 0) for x in _step_lengths(case)[1]) + case["pad"]
        return {"bytes": 4 * (n * 5 + 3 * total + 2 * (new // case["page"] + 1)), "flops": total + n}
    if case["op"] == "rope":
        rows = case["n_tok"] * (case["n_head"] + case["n_kv"])
        return {"bytes": 8 * rows * case["head_dim"] + 4 * case["axes"] * case["n_tok"],
                "flops": rows * (3 * case["n_rot"] + 4 * case["head_dim"] * case["norm"])}
    d, kv = case["head_dim"], case["n_kv"]
    row = d // 2 + d // GROUP * 2
    if case["op"] == "append":
        n = case["n_tok"]
        return {"bytes": 2 * n * kv * (4 * d + row + row + 4 * d) + 8 * n, "flops": 2 * n * kv * d * 4}
    cached = pairs = tokens = 0
    for keys, new in _requests(case):
        first, last = keys - new, keys - 1
        cached += last + 1 - (max(0, first + 1 - case["window"]) if case["window"] else 0)
        pairs += _visible(first, last, case["window"])
        tokens += new
    return {"bytes": 2 * cached * kv * row + 8 * tokens * case["n_head"] * d, "flops": 4 * d * case["n_head"] * pairs}


# ---- the 4-bit form --------------------------------------------------------------------------


def _quantise(x):
    """Codes (-8 .. 7, int32) and bf16 scales of x [..., head_dim] (float32), per group of 32: the value of largest
    magnitude, with its sign (the positive one on a tie), over -8, rounded to bf16 and held between 2^-17 and 2^11."""
    g = x.unflatten(-1, (-1, GROUP))
    hi, lo = g.amax(-1), g.amin(-1)
    s = (torch.where(hi >= -lo, hi, lo) * -0.125).to(torch.bfloat16).float()
    s = torch.copysign(s.abs().clamp(2.0 ** -17, 2.0 ** 11), s)
    c = torch.round(g * torch.reciprocal(s).unsqueeze(-1)).clamp(-8, 7)
    bad = ~torch.isfinite(g).all(-1)
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    c = torch.where(bad.unsqueeze(-1), torch.zeros_like(c), c)
    return c.to(torch.int32).flatten(-2), s.to(torch.bfloat16)


def _pack(c):
    """The 16-byte units [..., U, 16] of codes [..., head_dim]."""
    n = (c + 8).unflatten(-1, (-1, 8))[..., torch.tensor(NIBBLE, device=c.device)]
    return (n[..., 0::2] | (n[..., 1::2] << 4)).to(torch.uint8).flatten(-2).unflatten(-1, (-1, 16))


def _unpack(units):
    """Codes [..., head_dim] (float32) of units [..., U, 16]."""
    b = units.flatten(-2).unflatten(-1, (-1, 4)).to(torch.int32)
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2)  # nibbles 0 .. 7 of each word
    place = torch.tensor([NIBBLE.index(v) for v in range(8)], device=b.device)
    return (n[..., place] - 8).float().flatten(-2)


def _place(off, d):
    """Where the units of the keys at offsets `off` of their page sit: [..., U]."""
    u = d // GROUP
    return torch.arange(u, device=off.device) ^ ((off * (d // 2) // 128) % u).unsqueeze(-1)


def _parts(pages, page, d):
    """Views of the pool [n_pages][n_kv][chunk]: K units, V units [.., page, U, 16], K scales, V scales [.., page, U]."""
    u, codes = d // GROUP, page * d // 2
    k = pages[..., :codes].unflatten(-1, (page, u, 16))
    v = pages[..., codes:2 * codes].unflatten(-1, (page, u, 16))
    s = pages[..., 2 * codes:].view(torch.bfloat16)
    return k, v, s[..., :page * u].unflatten(-1, (page, u)), s[..., page * u:].unflatten(-1, (page, u))


def _chunk(page, d):
    return page * d + 2 * page * (d // GROUP) * 2


# ---- inputs ------------------------------------------------------------------------------------


def _step_lengths(case):
    n = case["n_req"]
    past = _sizes(case["past_lo"], case["past_hi"], n, 7)
    new = _sizes(case["new_lo"], case["new_hi"], n, 3)
    for i in range(case["ended"]):
        new[(i * 5 + 1) % n] = -1
    return past, new


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _prepare_step(case, seed):
    rng = random.Random(seed)
    past, new = _step_lengths(case)
    order = list(range(case["n_req"]))
    rng.shuffle(order)
    past, new = [past[i] for i in order], [new[i] for i in order]
    page = case["page"]
    held = [-(-p // page) for p in past]
    max_blocks = max(-(-(p + max(n, 0)) // page) for p, n in zip(past, new))
    n_pages = sum(held) + case["spare"]
    ids = list(range(n_pages))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (max_blocks - h))
        at += h
    head = rng.randrange(n_pages)
    ring = [-1] * n_pages
    for i, p in enumerate(ids[at:]):
        ring[(head + i) % n_pages] = p
    total = sum(max(n, 0) for n in new)
    z = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(case=case, past=_ints(past), new=_ints(new), held=_ints(held), ring=_ints(ring),
                queue=_ints([head, case["spare"]]), table=_ints(table), max_blocks=max_blocks, n_pages=n_pages,
                max_tok=total + case["pad"], held_out=z(case["n_req"]), queue_out=z(4), seq_len=z(case["n_req"]),
                q_start=z(case["n_req"] + 1), positions=z(total + case["pad"]), slots=z(total + case["pad"]),
                token_req=z(total + case["pad"]))


def _sections(half, axes, interleaved):
    if interleaved:
        s = [(half - a - 1) // axes + 1 for a in range(axes)]  # as many pairs as an axis's places hold ...
        s[-1] -= (half // axes) // 5  # ... and a few less for the last, which the first axis takes
        s[0] = half - sum(s[1:])
        return s
    s = [half * (axes + 1 - a) // (axes * (axes + 3) // 2) for a in range(axes)]
    s[0] = half - sum(s[1:])
    return s


def _prepare_rope(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, d = case["n_tok"], case["head_dim"]
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    t = torch.randint(0, case["pos_hi"], (1,), generator=g, device="cuda") + torch.arange(n, device="cuda") // 4
    if case["axes"] == 1:  # a decode batch: every token at a position of its own
        t = torch.randint(0, case["pos_hi"], (n,), generator=g, device="cuda")
    axes = [t, t + torch.arange(n, device="cuda") % 61, t + torch.arange(n, device="cuda") // 61 % 47]
    half = case["n_rot"] // 2
    inv = 1e6 ** (-torch.arange(half, dtype=torch.float64) / half)
    s = dict(case=case, q=rnd(n, case["n_head"] * d) * 2, k=rnd(n, case["n_kv"] * d) + rnd(case["n_kv"] * d),
             positions=torch.stack(axes[:case["axes"]]).to(torch.int32), inv_freq=inv.float().cuda(),
             sections=_sections(half, case["axes"], case["interleaved"]))
    s["q_gamma"] = 1 + 0.2 * rnd(d) if case["norm"] else None
    s["k_gamma"] = 1 + 0.2 * rnd(d) if case["norm"] else None
    s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
    return s


def _prepare_append(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, kv, d, page = case["n_tok"], case["n_kv"], case["head_dim"], case["page"]
    n_pages = -(-n // page) * 2 + 1
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:n]
    if n > 256:  # a prompt: runs of whole pages, in any order
        slots = (torch.randperm(n_pages, generator=g, device="cuda").unsqueeze(1) * page +
                 torch.arange(page, device="cuda")).flatten()[:n]
    slots[n - case["skipped"]:] = -1  # a padded buffer's tail
    k = rnd(n, kv * d) * (1 + 4 * (torch.rand(kv * d, generator=g, device="cuda") < 0.03))  # a few large channels
    pages = torch.randint(0, 256, (n_pages, kv, _chunk(page, d)), generator=g, dtype=torch.uint8, device="cuda")
    return dict(case=case, k=k, v=rnd(n, kv * d) * 0.5, slots=slots.to(torch.int32), pages=pages, n_pages=n_pages,
                k_back=torch.empty(n, kv * d, device="cuda"), v_back=torch.empty(n, kv * d, device="cuda"))


def _prepare_attention(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv, d, page = case["n_kv"], case["head_dim"], case["page"]
    reqs = _requests(case)
    blocks = [-(-k // page) for k, _ in reqs]
    n_pages = sum(blocks) + 3
    # a pool in use: what no request holds (and the rest of a last page) is whatever was there before
    pages = torch.randint(0, 256, (n_pages, kv, _chunk(page, d)), generator=g, dtype=torch.uint8, device="cuda")
    ids = torch.randperm(n_pages, generator=g, device="cuda")
    table = torch.full((len(reqs), max(blocks)), -1, dtype=torch.int32, device="cuda")
    offset = torch.randn(kv, 1, d, generator=g, device="cuda")  # K has channels off zero
    place = _place(torch.arange(page, device="cuda"), d).expand(kv, page, d // GROUP)
    at = 0
    for r, ((keys, _), nb) in enumerate(zip(reqs, blocks)):
        table[r, :nb] = ids[at:at + nb]
        at += nb
        for b0 in range(0, nb, 256):  # K and V rows, quantised into the request's pages
            n = min(256, nb - b0)
            rows = torch.randn(2, n, kv, page, d, generator=g, device="cuda")
            rows[0] += offset
            c, s = _quantise(rows)
            u = _pack(c).gather(-2, place.unsqueeze(-1).expand(2, n, kv, page, d // GROUP, 16))
            whole = table[r, b0:b0 + n].long()
            new = torch.cat([u[0].flatten(2), u[1].flatten(2), s[0].flatten(2).view(torch.uint8),
                             s[1].flatten(2).view(torch.uint8)], -1)
            if b0 + n == nb and keys % page:  # the last page: only its first keys
                last = pages[whole[-1]].clone()
                for part, have in zip(_parts(last, page, d), _parts(new[-1], page, d)):
                    part[:, :keys % page] = have[:, :keys % page]
                new[-1] = last
            pages[whole] = new
    new = [n for _, n in reqs]
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    q = torch.randn(starts[-1], case["n_head"] * d, generator=g, device="cuda") * 1.5
    return dict(case=case, pages=pages, n_pages=n_pages, table=table, q=q, seq_len=_ints([k for k, _ in reqs]),
                q_start=_ints(starts), max_new=max(new), max_keys=max(k for k, _ in reqs), out=torch.zeros_like(q))


def prepare(case, seed):
    return globals()["_prepare_" + case["op"]](case, seed)


# ---- the plain forms ---------------------------------------------------------------------------------


def _plain_step(s):
    c, page = s["case"], s["case"]["page"]
    past, new, held, ring, table = (s[k].long() for k in ("past", "new", "held", "ring", "table"))
    head, count = s["queue"][0].long(), s["queue"][1].long()
    ends, n = new < 0, new.clamp(min=0)
    q_end = n.cumsum(0)
    q_start = q_end - n
    fits = ~ends & (past + n <= s["max_blocks"] * page) & (q_end <= s["max_tok"])
    need = torch.where(fits, ((past + n + page - 1) // page - held).clamp(min=0), torch.zeros_like(n))
    cum = need.cumsum(0)
    served = fits & ((need == 0) | (cum <= count))
    got = torch.where(served, need, torch.zeros_like(need))
    taken = got.sum()
    freed = torch.where(ends, held, torch.zeros_like(held))
    held_out = torch.where(ends, torch.zeros_like(held), held + got)
    col = torch.arange(s["max_blocks"], device=past.device)
    fresh = (col >= held.unsqueeze(1)) & (col < held_out.unsqueeze(1))
    take = ring[(head + (cum - need).unsqueeze(1) + col - held.unsqueeze(1)) % s["n_pages"]]
    table = torch.where(fresh, take, table)
    give = (col < freed.unsqueeze(1))
    to = (head + count + (freed.cumsum(0) - freed).unsqueeze(1) + col) % s["n_pages"]
    ring = ring.index_put((to[give],), table[give])
    tok = torch.arange(s["max_tok"], device=past.device)
    req = torch.searchsorted(q_end, tok, right=True)
    real = req < c["n_req"]
    r = req.clamp(max=c["n_req"] - 1)
    pos = past[r] + tok - q_start[r]
    slot = table[r, (pos // page).clamp(max=s["max_blocks"] - 1)] * page + pos % page
    none = torch.full_like(tok, -1)
    i32 = torch.int32
    return dict(table=table.to(i32), ring=ring.to(i32), held=held_out.to(i32),
                queue=torch.stack([(head + taken) % s["n_pages"], count - taken + freed.sum(), cum[-1] - taken,
                                   q_end[-1]]).to(i32),
                seq_len=torch.where(ends, torch.zeros_like(past), torch.where(served, past + n, past)).to(i32),
                q_start=torch.cat([q_start, q_end[-1:]]).to(i32),
                positions=torch.where(real, pos, torch.zeros_like(pos)).to(i32),
                slots=torch.where(real & served[r], slot, none).to(i32), token_req=torch.where(real, req, none).to(i32))


def _axis_of(s):
    """The axis of each pair."""
    half, axes = s["case"]["n_rot"] // 2, s["case"]["axes"]
    if s["case"]["interleaved"]:
        return [i % axes if i // axes < s["sections"][i % axes] else 0 for i in range(half)]
    return [a for a in range(axes) for _ in range(s["sections"][a])]


def _plain_rope(s):
    c, d, half = s["case"], s["case"]["head_dim"], s["case"]["n_rot"] // 2
    if "axis" not in s:
        s["axis"] = torch.tensor(_axis_of(s), device="cuda")
    angle = s["positions"].float()[s["axis"]].T * s["inv_freq"]
    cos, sin = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)

    def turned(x, gamma):
        x = x.unflatten(-1, (-1, d))
        if gamma is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gamma
        a, b = (x[..., :half], x[..., half:2 * half]) if c["neox"] else (x[..., 0:2 * half:2], x[..., 1:2 * half:2])
        u, w = a * cos - b * sin, a * sin + b * cos
        r = torch.cat([u, w], -1) if c["neox"] else torch.stack([u, w], -1).flatten(-2)
        return torch.cat([r, x[..., 2 * half:]], -1).flatten(-2)

    return turned(s["q"], s["q_gamma"]), turned(s["k"], s["k_gamma"])


def _plain_append(s):
    c, d, page = s["case"], s["case"]["head_dim"], s["case"]["page"]
    slots = s["slots"].long()
    keep = (slots >= 0).nonzero().squeeze(1)
    at, off = slots[keep] // page, slots[keep] % page
    place = _place(off, d).unsqueeze(1).expand(-1, c["n_kv"], -1)  # [n][kv][U]
    ku, vu, ks, vs = _parts(s["pages"], page, d)

    def put(units, scales, x):
        q, sc = _quantise(x[keep].unflatten(-1, (c["n_kv"], d)))
        units[at, :, off] = _pack(q).gather(2, place.unsqueeze(-1).expand(-1, -1, -1, 16))
        scales[at, :, off] = sc

    def get(units, scales, x):
        u = units[at, :, off].gather(2, place.unsqueeze(-1).expand(-1, -1, -1, 16))
        value = _unpack(u).unflatten(-1, (-1, GROUP)) * scales[at, :, off].float().unsqueeze(-1)
        return torch.zeros_like(x).index_copy(0, keep, value.flatten(1))

    put(ku, ks, s["k"])
    put(vu, vs, s["v"])
    return get(ku, ks, s["k"]), get(vu, vs, s["v"])


def _plain_attention(s):
    c, d, page, kv = s["case"], s["case"]["head_dim"], s["case"]["page"], s["case"]["n_kv"]
    group = c["n_head"] // kv
    table, seq_len, q_start = s["table"].long().clamp(min=0), s["seq_len"].long(), s["q_start"].long()
    n_req, n_key = table.shape[0], table.shape[1] * page
    dev = table.device
    place = _place(torch.arange(page, device=dev), d)
    key = torch.arange(n_key, device=dev)
    live = (key < seq_len.unsqueeze(1))[:, None, :, None]
    ku, vu, ks, vs = _parts(s["pages"], page, d)

    def values(units, scales):  # [n_req][kv][n_key][d], nothing where no key is
        u = units[table].gather(-2, place.unsqueeze(-1).expand(n_req, table.shape[1], kv, page, d // GROUP, 16))
        x = (_unpack(u).unflatten(-1, (-1, GROUP)) * scales[table].float().unsqueeze(-1)).flatten(-2)
        return torch.where(live, x.transpose(1, 2).flatten(2, 3), torch.zeros((), device=dev))

    new = q_start[1:] - q_start[:-1]
    t = torch.arange(s["max_new"], device=dev)
    real = t < new.unsqueeze(1)
    row = (q_start[:-1].unsqueeze(1) + t).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].unflatten(-1, (kv, group, d))
    score = torch.einsum("rtkgd,rknd->rkgtn", q, values(ku, ks)) * (1.0 / math.sqrt(d))
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    pos = (seq_len - new).unsqueeze(1) + t
    sees = (key <= pos.unsqueeze(-1)) & (key < seq_len[:, None, None])
    if c["window"]:
        sees &= key > pos.unsqueeze(-1) - c["window"]
    score = torch.where(sees[:, None, None], score, torch.full((), -math.inf, device=dev))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.einsum("rkgtn,rknd->rtkgd", p, values(vu, vs)).flatten(2)
    return torch.zeros_like(s["q"]).index_put((row[real],), out[real])


# ---- the framework's calls ------------------------------------------------------------------------------


def _own_step(s, N):
    if "call" not in s:
        c = s["case"]
        s["call"] = N.paged_step(n_req=c["n_req"], page_size=c["page"], n_pages=s["n_pages"],
                                 max_blocks=s["max_blocks"], max_tok=s["max_tok"], past=s["past"], n_new=s["new"],
                                 held=s["held"], queue=s["queue"], ring=s["ring"], block_table=s["table"],
                                 held_out=s["held_out"], queue_out=s["queue_out"], seq_len=s["seq_len"],
                                 q_start=s["q_start"], positions=s["positions"], slots=s["slots"],
                                 token_req=s["token_req"])
        s["result"] = dict(table=s["table"], ring=s["ring"], held=s["held_out"], queue=s["queue_out"],
                           seq_len=s["seq_len"], q_start=s["q_start"], positions=s["positions"], slots=s["slots"],
                           token_req=s["token_req"])
    N.paged_step_dev(s["call"], torch.cuda.current_stream())
    return s["result"]


def _own_rope(s, N):
    if "call" not in s:
        c = s["case"]
        s["call"] = N.rope_axes(n_tok=c["n_tok"], n_head=c["n_head"], n_kv=c["n_kv"], head_dim=c["head_dim"],
                                n_rot=c["n_rot"], rope_mode=N.ROPE_NEOX if c["neox"] else N.ROPE_NORM,
                                sections=s["sections"], interleaved=c["interleaved"], positions=s["positions"],
                                inv_freq=s["inv_freq"], q_gamma=s["q_gamma"], k_gamma=s["k_gamma"], eps=1e-6,
                                q=s["q"], k=s["k"], q_out=s["q_out"], k_out=s["k_out"])
    N.rope_axes_dev(s["call"], torch.cuda.current_stream())
    return s["q_out"], s["k_out"]


def _pool(s, N):
    c = s["case"]
    return N.kv4_pool(s["pages"], n_pages=s["n_pages"], page_size=c["page"], n_kv=c["n_kv"], head_dim=c["head_dim"])


def _own_append(s, N):
    if "call" not in s:
        pool, n = _pool(s, N), s["case"]["n_tok"]
        s["call"] = N.kv4_rows(pool, slots=s["slots"], n_tok=n, k=s["k"], v=s["v"])
        s["back"] = N.kv4_rows(pool, slots=s["slots"], n_tok=n, k=s["k_back"], v=s["v_back"])
    stream = torch.cuda.current_stream()
    N.kv4_append_dev(s["call"], stream)
    N.kv4_read_dev(s["back"], stream)
    return s["k_back"], s["v_back"]


def _own_attention(s, N):
    if "call" not in s:
        c = s["case"]
        s["call"] = N.kv4_attn(_pool(s, N), n_req=c["n_req"], n_tok=s["q"].shape[0], n_head=c["n_head"],
                               max_new=s["max_new"], scale=1.0 / math.sqrt(c["head_dim"]), softcap=c["softcap"],
                               window=c["window"], block_table=s["table"], max_blocks=s["table"].shape[1],
                               seq_len=s["seq_len"], q_start=s["q_start"], q=s["q"], out=s["out"])
        s["ws"] = torch.zeros(N.kv4_workspace_bytes(s["call"]), dtype=torch.uint8, device="cuda")
        s["call"].workspace, s["call"].workspace_bytes = s["ws"].data_ptr(), s["ws"].numel()
    N.kv4_attention_dev(s["call"], torch.cuda.current_stream())
    return s["out"]


def run(state):
    op = state["case"]["op"]
    if own:
        import libllmcpu_b200 as N

        return globals()["_own_" + op](state, N)
    return globals()["_plain_" + op](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------


def _exact_rope(case, seed):
    s = _prepare_rope(case, seed)
    d, half = case["head_dim"], case["n_rot"] // 2
    axis = _axis_of(s)
    pos, inv = s["positions"].double().cpu(), s["inv_freq"].double().cpu()
    angle = torch.stack([pos[axis[i]] * inv[i] for i in range(half)], 1).cuda()
    first = [i if case["neox"] else 2 * i for i in range(half)]
    second = [i + half if case["neox"] else 2 * i + 1 for i in range(half)]
    outs = []
    for x, gamma in ((s["q"], s["q_gamma"]), (s["k"], s["k_gamma"])):
        x = x.double().view(case["n_tok"], -1, d)
        if gamma is not None:
            x = x / ((x ** 2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * gamma.double()
        y = x.clone()
        a, b, co, si = x[..., first], x[..., second], torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        y[..., first] = a * co - b * si
        y[..., second] = b * co + a * si
        outs.append(y.view(case["n_tok"], -1))
    return tuple(outs)


def _exact_append(case, seed):
    s = _prepare_append(case, seed)

    def rows(x):  # what each value reads as
        x = x.double().view(-1, case["head_dim"] // GROUP, GROUP)
        most = x.abs().amax(-1, keepdim=True)
        top = torch.where((x == most).any(-1, keepdim=True), most, -most)
        step = (top / -8).float().to(torch.bfloat16).double()
        step = torch.where(torch.signbit(step), -1.0, 1.0) * step.abs().clamp(2.0 ** -17, 2.0 ** 11)
        y = (step * torch.round(x / step).clamp(-8, 7)).view(case["n_tok"], -1)
        y[s["slots"] < 0] = 0
        return y

    return rows(s["k"]), rows(s["v"])


def _exact_attention(case, seed):
    s = _prepare_attention(case, seed)
    d, page, kv, u = case["head_dim"], case["page"], case["n_kv"], case["head_dim"] // GROUP
    group, half = case["n_head"] // kv, page * d // 2
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for r, (keys, new) in enumerate(_requests(case)):
        ids = s["table"][r, :-(-keys // page)].long()
        raw = s["pages"][ids]  # [blocks][kv][chunk]

        def values(codes0, scales0):
            x = torch.empty(len(ids), kv, page, d, dtype=torch.float64, device="cuda")
            sc = raw[..., scales0:scales0 + 2 * page * u].contiguous().view(torch.bfloat16).double()
            sc = sc.view(len(ids), kv, page, u)
            for g in range(u):
                for k in range(page):
                    b0 = codes0 + k * (d // 2) + 16 * (g ^ (k * d // 256 % u))
                    b = raw[..., b0:b0 + 16].to(torch.int64)
                    for i in range(32):
                        n = (i % 8) // 2 + 4 * (i % 2)
                        x[:, :, k, 32 * g + i] = ((b[..., i // 8 * 4 + n // 2] >> (4 * (n % 2))) % 16 - 8) * sc[..., k, g]
            return x.transpose(0, 1).reshape(kv, -1, d)[:, :keys]

        K, V = values(0, 2 * half), values(half, 2 * half + 2 * page * u)
        q = s["q"][at:at + new].double().view(new, kv, group, d)
        pos = torch.arange(keys - new, keys, device="cuda")
        key = torch.arange(keys, device="cuda")
        hidden = key > pos[:, None]
        if case["window"]:
            hidden |= key <= pos[:, None] - case["window"]
        for h in range(kv):
            score = q[:, h].transpose(0, 1) @ K[h].T / math.sqrt(d)
            if case["softcap"]:
                score = case["softcap"] * torch.tanh(score / case["softcap"])
            p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            out[at:at + new].view(new, kv, group, d)[:, h] = (p @ V[h]).transpose(0, 1)
        at += new
    return out


def exact(case, seed):
    return None if case["op"] == "step" else globals()["_exact_" + case["op"]](case, seed)
