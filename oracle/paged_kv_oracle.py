"""CPU oracle of the paged fp8 cache: plain loops in 64 bits over host tensors, written from the definitions in
include/fa8_kv_cache.h.  Test infrastructure only."""
from __future__ import annotations

import math

import torch

FP8_MAX = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


def spans(seqlens, cu_seqlens, tokens):
    """(sequence, first row, new tokens, length) of every sequence, host numbers."""
    lens = [int(x) for x in seqlens]
    if cu_seqlens is None:
        n = tokens // max(1, len(lens))
        return [(b, b * n, n, s) for b, s in enumerate(lens)]
    cu = [int(x) for x in cu_seqlens]
    return [(b, cu[b], cu[b + 1] - cu[b], s) for b, s in enumerate(lens)]


def scale_for(amax: float, largest: float) -> float:
    """Smallest 2^e with amax <= largest * 2^e, -64 <= e <= 64."""
    e = -64
    while e < 64 and amax > largest * 2.0 ** e:
        e += 1
    return 2.0 ** e


def to_fp8(x: torch.Tensor, dtype) -> torch.Tensor:
    """x (64-bit) rounded to fp8, saturating; NaN stays NaN.  32 bits hold what the callers pass exactly."""
    return x.clamp(-FP8_MAX[dtype], FP8_MAX[dtype]).float().to(dtype)


def append(cache, k, v, page_table, seqlens, cu_seqlens=None):
    """The cache (host tensors k, v, k_descale, v_descale) after the append: new tensors."""
    out = [t.clone() for t in cache]
    P = cache[0].shape[2]
    for x8, d, x in ((out[0], out[2], k), (out[1], out[3], v)):
        largest = FP8_MAX[x8.dtype]
        for b, first, n, length in spans(seqlens, cu_seqlens, x.shape[0]):
            pos = length - n
            while pos < length:
                page, off = int(page_table[b, pos // P]), pos % P
                m = min(P - off, length - pos)
                rows = x[first + pos - (length - n):first + pos - (length - n) + m].double()
                for h in range(x8.shape[1]):
                    r = rows[:, h]
                    finite = r[torch.isfinite(r)].abs()
                    new = scale_for(float(finite.max()) if finite.numel() else 0.0, largest)
                    if off > 0:
                        old = float(d[page, h])
                        new = max(new, old)
                        if new > old:
                            x8[page, h, :off] = to_fp8(x8[page, h, :off].double() * (old / new), x8.dtype)
                    d[page, h] = new
                    x8[page, h, off:off + m] = to_fp8(r / new, x8.dtype)
                pos += m
    return out


def keys_values(cache, page_table, b, length):
    """Sequence b's keys and values in 64 bits: [length, heads_kv, head_dim] each."""
    P = cache[0].shape[2]
    ids = [int(page_table[b, p]) for p in range(-(-length // P))]
    if not ids:
        return [x8.double()[:0, :, 0] for x8 in cache[:2]]
    return [(x8[ids].double() * d[ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:length]
            for x8, d in ((cache[0], cache[2]), (cache[1], cache[3]))]


def read(cache, page_table, seqlens, tokens, cu_seqlens=None):
    """(k, v) [tokens, heads_kv, head_dim] in 64 bits; rows of no sequence are NaN."""
    shape = (tokens, cache[0].shape[1], cache[0].shape[3])
    out = [torch.full(shape, math.nan, dtype=torch.float64) for _ in range(2)]
    for b, first, n, length in spans(seqlens, cu_seqlens, tokens):
        for o, x in zip(out, keys_values(cache, page_table, b, length)):
            o[first:first + n] = x[length - n:]
    return out


def attention(q, cache, page_table, seqlens, causal, scale, cu_seqlens=None):
    """(O, lse, A): O and lse in 64 bits, A = softmax . |V| (what a relative error of the probabilities is relative to).
    Rows of no sequence are NaN."""
    T, H, D = q.shape
    G = H // cache[0].shape[1]
    o, a = (torch.full((T, H, D), math.nan, dtype=torch.float64) for _ in range(2))
    lse = torch.full((T, H), math.nan, dtype=torch.float64)
    for b, first, n, length in spans(seqlens, cu_seqlens, T):
        if n == 0:
            continue
        k, v = keys_values(cache, page_table, b, length)
        kq, vq = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)                     # [length, H, D]
        s = torch.einsum("ihd,jhd->hij", q[first:first + n].double(), kq) * scale
        if causal:
            s = s.masked_fill(torch.arange(length)[None, :] > (length - n + torch.arange(n))[:, None], -math.inf)
        m = s.amax(-1, keepdim=True) if length else torch.full((H, n, 1), -math.inf, dtype=torch.float64)
        p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
        l = p.sum(-1, keepdim=True)
        p = p / torch.where(l == 0, 1.0, l)
        # what a row does not see does not count, whatever is held there
        seen = (s > -math.inf) | torch.isnan(s)
        nan, up, down = (torch.einsum("hij,jhd->ihd", seen.double(), of.double()) > 0 for of in (torch.isnan(vq), vq == math.inf, vq == -math.inf))
        vq = torch.where(torch.isfinite(vq), vq, 0.0)
        special = torch.where(up, math.inf, 0.0) + torch.where(down, -math.inf, 0.0) + torch.where(nan, math.nan, 0.0)
        o[first:first + n] = torch.einsum("hij,jhd->ihd", p, vq) + special
        a[first:first + n] = torch.einsum("hij,jhd->ihd", p, vq.abs())
        lse[first:first + n] = (m + torch.log(l)).squeeze(-1).t()
    return o, lse, a
