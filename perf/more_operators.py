"""The projections of a serving batch in 8-bit integers and what is reported of
its logits, measured: rows quantised (with their norm), rows looked up, the
product of 8-bit rows, and log probabilities.

``listed()`` names the cases, ``draw(rng)`` makes more of the same ranges,
``prepare(case, seed)`` the inputs, ``run(state)`` one pass: with ``own`` the
framework's calls, otherwise the operators' plain form in elementary torch
operations (32 bits; codes at their borders in 64). ``exact(case, seed)`` is the
definition in 64 bits.

A row in 8 bits is codes (int8) and one float32 scale. Of a row x with a gain g:
z = x * g (a float32 product), s = max(max |z| / 127, 2^-126) (float32), code =
z / s rounded to the nearest whole number, ties to even; the row's scale is s,
with an RMS norm s / sqrt(mean(x^2) + eps): the norm is a factor of the whole row
and leaves the codes alone.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
TINY = 2.0 ** -126


# ---- the cases -----------------------------------------------------------------------------


def listed():
    # widths: Qwen3-8B 4096 (q, k, v together 6144 rows), Gemma-3-4B 2560 (4096), Llama-3.2-1B 2048
    return [
        # a decode batch's hidden states, normed and quantised before a projection (and read back): the small call
        dict(name="quantise 64x4096", op="quantise", n=64, cols=4096, type="float32", gain=1, norm=1),
        # a packed prompt batch's, an odd number of tokens
        dict(name="quantise 8191x2560", op="quantise", n=8191, cols=2560, type="float32", gain=1, norm=1),
        # a step's tokens into hidden states, from the tied embedding table
        dict(name="lookup 64 of 262144x2560", op="lookup", n=64, vocab=262144, cols=2560, scaled=1, pad=0),
        # a prompt batch's tokens, the buffer padded at its end
        dict(name="lookup 8191 of 128256x2048", op="lookup", n=8191, vocab=128256, cols=2048, scaled=0, pad=500),
        # one user decoding, q, k and v in one product: latency
        dict(name="linear 1x4096 to 6144", op="linear", n=1, cols=4096, rows=6144, bias=0, add=0),
        # a serving batch's output projection, added to the residual stream
        dict(name="linear 64x4096 to 4096", op="linear", n=64, cols=4096, rows=4096, bias=0, add=1),
        # the logits of 16 requests: the weights' bytes
        dict(name="linear 16x2560 to 262144", op="linear", n=16, cols=2560, rows=262144, bias=0, add=0),
        # an odd chunk of a prompt, with the projections' biases
        dict(name="linear 777x2048 to 2560", op="linear", n=777, cols=2048, rows=2560, bias=1, add=0),
        # a prompt batch: the tensor cores
        dict(name="linear 8192x4096 to 6144", op="linear", n=8192, cols=4096, rows=6144, bias=0, add=0),
        # one user's sampled token with its alternatives: latency
        dict(name="logprobs 1x262144 top 20", op="logprobs", n=1, vocab=262144, top=20, scale=1.0, masked=0.0, steps=0),
        # a serving batch whose output is held to a grammar: most of the vocabulary is masked; logits of 16 bits tie
        dict(name="logprobs 64x151936 top 5", op="logprobs", n=64, vocab=151936, top=5, scale=1.25, masked=0.9, steps=1),
        # a prompt scored: the log probability of every next token and the entropy there
        dict(name="logprobs 2047x128256", op="logprobs", n=2047, vocab=128256, top=0, scale=1.0, masked=0.0, steps=0),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantise", "lookup", "linear", "linear", "linear", "logprobs", "logprobs"])
    width = rng.choice([2048, 2560, 4096, _spread(rng, 64, 16384)])
    if op == "quantise":
        return dict(op=op, n=_spread(rng, 1, min(8192, 20_000_000 // width)), cols=width,
                    type=rng.choice(["float32", "float32", "bfloat16", "float16"]), gain=rng.randint(0, 1),
                    norm=rng.randint(0, 1))
    if op == "lookup":
        return dict(op=op, n=_spread(rng, 1, min(8192, 16_000_000 // width)),
                    vocab=_spread(rng, 1000, min(262144, 600_000_000 // width)), cols=width, scaled=rng.randint(0, 1),
                    pad=rng.choice([0, _spread(rng, 1, 500)]))
    if op == "linear":
        rows = rng.choice([1024, 2560, 4096, 6144, _spread(rng, 16, 16384), _spread(rng, 16384, 262144)])
        most = min(8192, 8192 * 4096 * 6144 // (rows * width), 64 if rows > 16384 else 8192)
        rows = min(rows, 671_000_000 // width)
        return dict(op=op, n=_spread(rng, 1, max(1, most)), cols=width, rows=rows, bias=rng.randint(0, 1),
                    add=rng.randint(0, 1))
    vocab = _spread(rng, 1000, 262144)
    return dict(op=op, n=_spread(rng, 1, min(2048, 260_000_000 // vocab)), vocab=vocab,
                top=rng.choice([0, 1, 5, 20, rng.randint(2, 32)]), scale=rng.choice([1.0, 1.0, 0.5, 1.43]),
                masked=rng.choice([0.0, 0.0, 0.5, 0.99]), steps=rng.randint(0, 1))


def work(case):
    n = case["n"]
    if case["op"] == "quantise":
        size = 4 if case["type"] == "float32" else 2
        return {"bytes": n * case["cols"] * (size + 1 + 1 + 4) + 8 * n, "flops": 8 * n * case["cols"]}
    if case["op"] == "lookup":
        return {"bytes": n * case["cols"] * 5 + 8 * n, "flops": n * case["cols"]}
    if case["op"] == "linear":
        r, c = case["rows"], case["cols"]
        return {"bytes": r * c + n * c + n * r * (8 if case["add"] else 4) + 4 * (r + n), "flops": 2 * n * r * c}
    return {"bytes": 4 * n * case["vocab"] + n * (16 + 8 * case["top"]), "flops": 6 * n * case["vocab"]}


# ---- inputs ------------------------------------------------------------------------------------


def _pitch(cols):
    """Bytes from one row of codes to the next: rows start on 16 bytes."""
    return -(-cols // 16) * 16


def _codes(g, n, cols):
    """Codes as a quantised row of normal values has them: a bell within -127 .. 127, in rows of 16-byte steps. What lies
    between two rows is whatever was there before."""
    c = torch.empty(n, _pitch(cols), dtype=torch.int8, device="cuda")
    for a in range(0, n, 16384):
        part = c[a:a + 16384]
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 33).clamp_(-127, 127).round_())
    return c


def _prepare_quantise(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, cols = case["n"], case["cols"]
    x = torch.randn(n, cols, generator=g, device="cuda")
    x *= 1 + 15 * (torch.rand(cols, generator=g, device="cuda") < 0.004)  # hidden states have a few large channels
    x = x.to(getattr(torch, case["type"]))
    gain = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda") if case["gain"] else None
    return dict(case=case, x=x, gain=gain, codes=torch.zeros(n, _pitch(cols), dtype=torch.int8, device="cuda"),
                scales=torch.zeros(n, device="cuda"), back=torch.zeros(n, cols, device="cuda"))


def _prepare_lookup(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, case["vocab"], (case["n"],), generator=g, device="cuda", dtype=torch.int32)
    ids[case["n"] - min(case["pad"], case["n"] - 1):] = -1
    return dict(case=case, codes=_codes(g, case["vocab"], case["cols"]), ids=ids,
                scales=(0.5 + torch.rand(case["vocab"], generator=g, device="cuda")) * 4e-4,
                mult=math.sqrt(case["cols"]) if case["scaled"] else 1.0,
                out=torch.zeros(case["n"], case["cols"], device="cuda"))


def _prepare_linear(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, cols, rows = case["n"], case["cols"], case["rows"]
    return dict(case=case, x=_codes(g, n, cols), w=_codes(g, rows, cols),
                x_scales=(0.5 + torch.rand(n, generator=g, device="cuda")) * 0.03,
                w_scales=(0.5 + torch.rand(rows, generator=g, device="cuda")) * 4e-4,
                bias=torch.randn(rows, generator=g, device="cuda") if case["bias"] else None,
                add=torch.randn(n, rows, generator=g, device="cuda") * 3 if case["add"] else None,
                y=torch.zeros(n, rows, device="cuda"))


def _prepare_logprobs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, vocab, top = case["n"], case["vocab"], case["top"]
    x = torch.randn(n, vocab, generator=g, device="cuda") * 2.5
    peak = torch.randint(0, vocab, (n, 8), generator=g, device="cuda")
    x.scatter_add_(1, peak, torch.rand(n, 8, generator=g, device="cuda") * 18)  # a few likely tokens
    if case["steps"]:
        x = x.to(torch.bfloat16).float()
    token = torch.where(torch.rand(n, generator=g, device="cuda") < 0.7, peak[:, 0],
                        torch.randint(0, vocab, (n,), generator=g, device="cuda"))
    if case["masked"]:
        x.masked_fill_(torch.rand(n, vocab, generator=g, device="cuda") < case["masked"], -math.inf)
    return dict(case=case, logits=x, tokens=token.to(torch.int32), logprob=torch.zeros(n, device="cuda"),
                entropy=torch.zeros(n, device="cuda"), rank=torch.zeros(n, dtype=torch.int32, device="cuda"),
                top_ids=torch.zeros(n, max(top, 1), dtype=torch.int32, device="cuda"),
                top_logprobs=torch.zeros(n, max(top, 1), device="cuda"))


def prepare(case, seed):
    return globals()["_prepare_" + case["op"]](case, seed)


# ---- the plain forms ---------------------------------------------------------------------------------


def _plain_quantise(s):
    x = s["x"].float()
    z = x if s["gain"] is None else x * s["gain"]
    step = (z.abs().amax(-1) / 127).clamp(min=TINY)
    code = torch.round(z.double() / step.double().unsqueeze(-1)).float()
    scale = step * torch.rsqrt((x * x).mean(-1) + EPS) if s["case"]["norm"] else step
    return scale, code * scale.unsqueeze(-1)


def _plain_lookup(s):
    ids = s["ids"].long()
    real = ids >= 0
    at = ids.clamp(min=0)
    scale = torch.where(real, s["scales"][at] * s["mult"], torch.zeros((), device="cuda"))
    return s["codes"][at, :s["case"]["cols"]].float() * scale.unsqueeze(-1)


def _plain_linear(s):
    cols = s["case"]["cols"]
    y = (s["x"][:, :cols].float() @ s["w"][:, :cols].float().T) * s["x_scales"].unsqueeze(-1) * s["w_scales"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y if s["add"] is None else y + s["add"]


def _order(x):
    """int64 keys that rank float32 values downwards and, where they are equal, indices upwards."""
    b = (x + 0.0).view(torch.int32)  # both zeros alike
    b = torch.where(b < 0, b ^ 0x7FFFFFFF, b).long()
    return b * 2 ** 32 + (2 ** 31 - torch.arange(x.shape[-1], device=x.device))


def _plain_logprobs(s):
    c, x, token = s["case"], s["logits"], s["tokens"].long().unsqueeze(-1)
    t = (x - x.amax(-1, keepdim=True)) * c["scale"]
    e = torch.exp(t)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, e * t, torch.zeros((), device="cuda")).sum(-1, keepdim=True) / total
    mine = x.gather(-1, token)
    before = (x > mine) | ((x == mine) & (torch.arange(x.shape[-1], device="cuda") < token))
    out = dict(logprob=(t.gather(-1, token) - log_total).squeeze(-1), entropy=entropy.squeeze(-1),
               rank=before.sum(-1).to(torch.int32))
    if c["top"]:
        ids = torch.topk(_order(x), c["top"], -1).indices
        lp = t.gather(-1, ids) - log_total
        out["top_ids"] = torch.where(torch.isinf(lp), torch.full_like(ids, -1), ids).to(torch.int32)
        out["top_logprobs"] = lp
    return out


# ---- the framework's calls ------------------------------------------------------------------------------


def _own_quantise(s, N):
    if "call" not in s:
        c = s["case"]
        s["call"] = N.i8_rows(n=c["n"], cols=c["cols"], x=s["x"], gamma=s["gain"], norm=c["norm"], eps=EPS,
                              codes=s["codes"], scales=s["scales"])
        s["read"] = N.i8_lookup(n=c["n"], cols=c["cols"], n_rows=c["n"], codes=s["codes"], scales=s["scales"],
                                out=s["back"])
    stream = torch.cuda.current_stream()
    N.i8_quantise_dev(s["call"], stream)
    N.i8_lookup_dev(s["read"], stream)
    return s["scales"], s["back"]


def _own_lookup(s, N):
    if "call" not in s:
        c = s["case"]
        s["call"] = N.i8_lookup(n=c["n"], cols=c["cols"], n_rows=c["vocab"], codes=s["codes"], scales=s["scales"],
                                ids=s["ids"], mult=s["mult"], out=s["out"])
    N.i8_lookup_dev(s["call"], torch.cuda.current_stream())
    return s["out"]


def _own_linear(s, N):
    if "call" not in s:
        c = s["case"]
        s["call"] = N.i8_linear(n_tok=c["n"], rows=c["rows"], cols=c["cols"], x=s["x"], x_scales=s["x_scales"],
                                w=s["w"], w_scales=s["w_scales"], bias=s["bias"], add=s["add"], y=s["y"])
    N.i8_linear_dev(s["call"], torch.cuda.current_stream())
    return s["y"]


def _own_logprobs(s, N):
    if "call" not in s:
        c = s["case"]
        more = dict(top_ids=s["top_ids"], top_logprobs=s["top_logprobs"]) if c["top"] else {}
        s["call"] = N.logprobs(n=c["n"], n_vocab=c["vocab"], logits=s["logits"], scale=c["scale"], tokens=s["tokens"],
                               logprob=s["logprob"], rank=s["rank"], entropy=s["entropy"], top=c["top"], **more)
        s["result"] = dict(logprob=s["logprob"], entropy=s["entropy"], rank=s["rank"], **more)
    N.logprobs_dev(s["call"], torch.cuda.current_stream())
    return s["result"]


def run(state):
    op = state["case"]["op"]
    if own:
        import libllmcpu_b200 as N

        return globals()["_own_" + op](state, N)
    return globals()["_plain_" + op](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------


def _exact_quantise(case, seed):
    s = _prepare_quantise(case, seed)
    z = s["x"].float()
    if case["gain"]:
        z = torch.mul(z, s["gain"])  # the definition's 32-bit product
    top = torch.maximum(z.max(-1).values, -z.min(-1).values)
    step = torch.maximum(torch.div(top, 127.0), torch.full_like(top, TINY)).double()
    code = (z.double() / step[:, None]).round()
    if case["norm"]:
        step = step / ((s["x"].double() ** 2).sum(-1) / case["cols"] + EPS).sqrt()
    return step, code * step[:, None]


def _exact_lookup(case, seed):
    s = _prepare_lookup(case, seed)
    out = torch.zeros(case["n"], case["cols"], dtype=torch.float64, device="cuda")
    at = torch.nonzero(s["ids"] >= 0).squeeze(1)
    ids = s["ids"][at].long()
    out[at] = s["codes"].index_select(0, ids)[:, :case["cols"]].double() * (s["scales"].double()[ids] * s["mult"])[:, None]
    return out


def _exact_linear(case, seed):
    s = _prepare_linear(case, seed)
    n, rows, cols = case["n"], case["rows"], case["cols"]
    out = torch.empty(n, rows, dtype=torch.float64, device="cuda")
    xt = s["x"].double()[:, :cols].T.contiguous()
    for a in range(0, rows, 8192):
        b = min(rows, a + 8192)
        part = (s["w"][a:b, :cols].double() @ xt).T
        out[:, a:b] = part * s["x_scales"].double()[:, None] * s["w_scales"][a:b].double()[None]
    if case["bias"]:
        out += s["bias"].double()[None]
    if case["add"]:
        out += s["add"].double()
    return out


def _exact_logprobs(case, seed):
    s = _prepare_logprobs(case, seed)
    n, top = case["n"], case["top"]
    f64 = dict(dtype=torch.float64, device="cuda")
    out = dict(logprob=torch.empty(n, **f64), entropy=torch.empty(n, **f64), rank=None)
    if top:
        out |= dict(top_ids=None, top_logprobs=torch.empty(n, top, **f64))
    for a in range(0, n, 64):
        x = s["logits"][a:a + 64].double() * case["scale"]
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        out["logprob"][a:a + 64] = lp[torch.arange(len(x), device="cuda"), s["tokens"][a:a + 64].long()]
        out["entropy"][a:a + 64] = torch.special.entr(lp.exp()).sum(-1)
        if top:
            out["top_logprobs"][a:a + 64] = lp.sort(-1, descending=True).values[:, :top]
    return out


def exact(case, seed):
    return globals()["_exact_" + case["op"]](case, seed)
