"""The 8-bit operators and the log probabilities by their definitions, in
64 bits, with how far a float32 result may be off: what the GPU tests compare
the kernels with."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24  # half a step of float32, relative


def quantise(x, gamma, norm, eps):
    """(codes int64, scales float64, both of x [n][cols] float32): z and the step are float32 by the definition."""
    with np.errstate(all="ignore"):
        z = x if gamma is None else x * gamma.astype(np.float32)
        bad = ~np.isfinite(z).all(-1)
        step = np.maximum(np.where(bad, np.float32(1), np.abs(z).max(-1)) * (np.float32(1) / np.float32(127)),
                          np.float32(2.0 ** -126))
        step = step.astype(np.float32)
        codes = np.rint(np.where(bad[:, None], 0, z).astype(np.float64) / step.astype(np.float64)[:, None])
        scale = step.astype(np.float64)
        if norm:
            mean = (x.astype(np.float64) ** 2).mean(-1) + np.float64(np.float32(eps))
            scale = np.where(mean > 0, scale / np.sqrt(np.where(mean > 0, mean, 1)), scale)
        scale[bad] = np.nan
    return codes.astype(np.int64), scale


def linear(x, xs, w, ws, bias=None, add=None):
    """(y, how far a float32 result may be off). The sum is exact; it is rounded once, each scale rounds once, and so
    do the sums with bias and add: half a step of what is rounded, each."""
    p = (x.astype(np.int64) @ w.astype(np.int64).T).astype(np.float64)
    p = p * xs.astype(np.float64)[:, None] * ws.astype(np.float64)
    tol = 3 * U * np.abs(p)
    for more in (bias, add):
        if more is not None:
            p = p + more.astype(np.float64)
            tol = tol + U * np.abs(p)
    return p, 1.001 * tol + 1e-43


def order(x):
    """The row's tokens as they come: by logit downwards (a NaN as -infinity), equal ones by index."""
    v = np.where(np.isnan(x), -np.inf, x).astype(np.float64) + 0.0
    return np.argsort(-v, kind="stable")


# float32 sums of a row's terms are formed of at most this many roundings one after another (a term's way through the
# group, the thread's groups, the threads)
CHAIN = 64


def logprobs(x, scale, token, top):
    """A row's values in 64 bits, and how far float32 ones may be off:
    t = (x - max) * scale rounds twice and the exponent's conversion to base 2 once more, 3 U |t| together; e = exp(t) is
    then off by that and the exponential's own 4 U, its sum by CHAIN U more."""
    v = x.astype(np.float64)
    s = np.float64(np.float32(scale))
    ids = order(x)
    rank = int(np.nonzero(ids == token)[0][0]) if 0 <= token < len(x) else -1
    alive = [int(i) for i in ids[:top] if x[i] > -np.inf]
    tops = np.array(alive + [-1] * (top - len(alive)), np.int64)
    inside = 0 <= token < len(x)
    if np.isnan(v).any() or (v == np.inf).any():
        lp = np.nan if inside else 0.0
        return dict(logprob=lp, entropy=np.nan, rank=rank, top_ids=tops,
                    top_logprobs=np.where(tops >= 0, np.nan, -np.inf)), dict(logprob=0, entropy=0, top_logprobs=0)
    if not (v > -np.inf).any():
        return dict(logprob=-np.inf if inside else 0.0, entropy=0.0, rank=rank, top_ids=tops,
                    top_logprobs=np.full(top, -np.inf)), dict(logprob=0, entropy=0, top_logprobs=0)
    t = (v - v.max()) * s
    e = np.exp(t)
    z = e.sum()
    far = np.where(e > 0, np.abs(np.where(e > 0, t, 0)), 0)
    mean_t = (e * far).sum() / z
    mean_tt = (e * far * far).sum() / z
    lp = t - np.log(z)
    # two finite logits lie up to 6.8e38 apart, twice the largest float32 (3.4e38): such a log probability rounds to -inf
    lp = np.where(lp < -np.float64(np.finfo(np.float32).max), -np.inf, lp)
    entropy = np.log(z) + mean_t
    z_off = 3 * mean_t + 4 + CHAIN  # of U, relative to z
    with np.errstate(invalid="ignore"):
        tl = np.where(tops >= 0, lp[np.maximum(tops, 0)], -np.inf)
        off = lambda q: U * (3 * np.abs(t[q]) + z_off + np.abs(lp[q])) * 1.01 if np.isfinite(lp[q]) else 0.0  # noqa: E731
        return dict(logprob=lp[token] if inside else 0.0, entropy=entropy, rank=rank, top_ids=tops, top_logprobs=tl), \
            dict(logprob=off(token) if inside else 0.0,
                 # h = sum e t: its terms are off by 3 |t| more than e's, relatively
                 entropy=1.01 * U * (z_off + 3 * mean_tt + (4 + CHAIN + 2 + z_off) * mean_t + entropy),
                 top_logprobs=np.array([off(i) if i >= 0 else 0.0 for i in tops]))
