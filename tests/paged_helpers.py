"""The paged operators written out in plain numpy, one value or one request at
a time, in 64 bits: what the GPU tests compare the kernels with."""
from __future__ import annotations

import numpy as np

GROUP = 32


def bf16(x):
    """float32 values rounded to bf16 (nearest, ties to even), as float32."""
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16) << 16
    return r.astype(np.uint32).view(np.float32)


def quantise(x):
    """(codes, scales) of float32 x [..., D], by the definition: per group of
    32 the value of largest magnitude over -8 in bf16, codes by the float32
    product with the scale's reciprocal."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    with np.errstate(all="ignore"):
        hi, lo = np.fmax.reduce(g, -1), np.fmin.reduce(g, -1)
        s = bf16(np.where(hi >= -lo, hi, lo) * np.float32(-0.125))
        s = np.copysign(np.clip(np.abs(s), np.float32(2.0 ** -17), np.float32(2.0 ** 11)), s).astype(np.float32)
        c = np.clip(np.rint(g * (np.float32(1) / s)[..., None]), -8, 7)
    bad = ~np.isfinite(g).all(-1)
    s[bad] = np.nan
    c[bad] = 0
    return c.astype(np.int64).reshape(x.shape), s


def value(c, s):
    return (c.reshape(*s.shape, GROUP) * s[..., None].astype(np.float64)).reshape(c.shape)


class Pool:
    """A layer's pool on the host: codes and scales per (page, head, offset), packed on request."""

    def __init__(self, n_pages, page, n_kv, d, rng, junk=True):
        self.n_pages, self.page, self.n_kv, self.d, self.u = n_pages, page, n_kv, d, d // GROUP
        self.chunk = page * d + 4 * page * self.u
        # what was there before: random bytes, among them NaN and infinite scales
        self.bytes = rng.integers(0, 256, (n_pages, n_kv, self.chunk), dtype=np.uint8) if junk else \
            np.zeros((n_pages, n_kv, self.chunk), np.uint8)
        if junk:
            self.bytes[..., page * d:].view(np.uint16)[..., ::3] = 0x7FC0
            self.bytes[..., page * d:].view(np.uint16)[..., 1::5] = 0xFF80

    def put(self, slot, h, which, c, s):
        """One row's codes (D, -8..7) and scales (U, float32) at a slot."""
        pg, off, half = slot // self.page, slot % self.page, self.page * self.d // 2
        for g in range(self.u):
            unit = g ^ ((off * self.d // 256) % self.u)
            at = which * half + off * self.d // 2 + 16 * unit
            for w in range(4):
                word = 0
                for i in range(8):
                    word |= int(c[32 * g + 8 * w + i] + 8) << (4 * (i // 2 + 4 * (i % 2)))
                self.bytes[pg, h, at + 4 * w:at + 4 * w + 4] = np.frombuffer(np.uint32(word).tobytes(), np.uint8)
            at = 2 * half + which * 2 * self.page * self.u + 2 * (off * self.u + g)
            b = (np.float32(s[g]).view(np.uint32) >> 16).astype(np.uint16)
            self.bytes[pg, h, at:at + 2] = np.frombuffer(b.tobytes(), np.uint8)


def attention(q, K, V, pos, window, scale, softcap):
    """One query row [D] over K, V [keys, D] in 64 bits; a row without keys is zero."""
    first = max(0, pos - window + 1) if window else 0
    k, v = K[first:max(pos + 1, 0)], V[first:max(pos + 1, 0)]
    if k.shape[0] == 0:
        return np.zeros(q.shape[-1])
    s = k @ q.astype(np.float64) * scale
    if softcap:
        s = softcap * np.tanh(s / softcap)
    p = np.exp(s - s.max())
    return p @ v / p.sum()


def step(past, new, held, queue, ring, table, page, n_pages, max_blocks, max_tok):
    """A step's tables, one request after the other (nncu_paged_step_dev)."""
    ring, table, held = list(ring), [list(r) for r in table], list(held)
    head, count = queue
    n = len(past)
    seq, start, wanted, taken, freed, given = [0] * n, [0], 0, 0, [], {}
    for r in range(n):
        nn = max(new[r], 0)
        start.append(start[-1] + nn)
        if new[r] < 0:
            freed += table[r][:held[r]]
            held[r], seq[r] = 0, 0
            continue
        fits = past[r] + nn <= max_blocks * page and start[-1] <= max_tok
        need = max(0, -(-(past[r] + nn) // page) - held[r]) if fits else 0
        ok = fits and (need == 0 or wanted + need <= count)
        for j in range(need if ok else 0):
            table[r][held[r] + j] = ring[(head + wanted + j) % n_pages]
        wanted += need
        given[r] = ok
        held[r] += need if ok else 0
        taken += need if ok else 0
        seq[r] = past[r] + nn if ok else past[r]
    for i, p in enumerate(freed):
        ring[(head + count + i) % n_pages] = p
    pos, slots, req = [0] * max_tok, [-1] * max_tok, [-1] * max_tok
    for r in range(n):
        for t in range(start[r], min(start[r + 1], max_tok)):
            pos[t], req[t] = past[r] + t - start[r], r
            if given.get(r):
                slots[t] = table[r][pos[t] // page] * page + pos[t] % page
    return dict(seq_len=seq, q_start=start, held=held, table=table, positions=pos, slots=slots, token_req=req,
                ring=ring, queue=[(head + taken) % n_pages, count - taken + len(freed), wanted - taken, start[-1]])
