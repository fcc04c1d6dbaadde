"""Attention over pages, and the step before it, in 64 bits from their definitions: what the
paged operators' tests compare with."""
import math

import torch

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make_pool(lengths, page, kv_heads, dim, dtype, g, slots=None, spare=2, fill=None):
    """k, v pools with every number set, tables [slots, table_len] of shuffled pages (unused
    entries -7) and lengths; sequence i of `lengths` in slot slots[i] (default i)."""
    slots = list(range(len(lengths))) if slots is None else slots
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    shape = (pages, kv_heads, page, dim)
    k = torch.randn(shape, generator=g).to(dtype)
    v = torch.randn(shape, generator=g).mul(2.0).to(dtype)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    count = max(slots) + 1 + 1
    tables = torch.full((count, max(1, max(need))), -7, dtype=torch.int32)
    held = torch.zeros(count, dtype=torch.int32)
    at = 0
    for s, n, length in zip(slots, need, lengths):
        tables[s, :n] = order[at:at + n]
        held[s] = length
        at += n
    if fill is not None:  # everything that is no sequence's token
        free = torch.ones(shape[0], page, dtype=torch.bool)
        for s, length in zip(slots, lengths):
            j = torch.arange(length)
            free[tables[s][j // page].long(), j % page] = False
        where = free[:, None, :, None].expand(shape)
        k[where] = fill
        v[where] = fill
    return k, v, tables, held


def rows_of(k, table, page, length):
    j = torch.arange(length)
    ids = table[j // page].long() if length else j
    return k[ids, :, j % page]  # [length, kv, dim]


def attention(q, k, v, tables, lengths, page, starts, slots, heads, scale, window, sinks):
    """(out, bound): 64 bits, and how far 32-bit arithmetic in any order may be from it.

    A score is a sum of dim products: in 32 bits, in any order and with the scale behind it, off
    by at most delta = (dim + 2) eps scale sum |q| |k| (dim roundings of the sum, one of a product
    or of an operand's pieces, one of the scale).  A probability is off by the score's and the
    maximum's delta, three eps of its exponential (2 ulp) and one of the difference, each sum over
    n keys by n eps more, its products and the division by one each, and the difference itself
    by eps of its size."""
    heads_per = heads // k.shape[1]
    dim = k.shape[3]
    out = torch.zeros(q.shape[0], heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    eps = 2.0 ** -24
    for i, s in enumerate(slots):
        length, first, n = int(lengths[s]), starts[i], starts[i + 1] - starts[i]
        keys = rows_of(k, tables[s], page, length).double()
        values = rows_of(v, tables[s], page, length).double()
        for t in range(n):
            p = length - n + t
            if p < 0:
                continue
            j = torch.arange(length)
            seen = j <= p
            if window > 0:
                seen &= (j > p - window) | (j < sinks)
            ks = keys[seen].repeat_interleave(heads_per, dim=1)    # [m, heads, dim]
            vs = values[seen].repeat_interleave(heads_per, dim=1)
            x = q[first + t].double().view(heads, dim)
            score = torch.einsum("hd,mhd->hm", x, ks) * scale
            delta = (dim + 2) * eps * abs(scale) * torch.einsum("hd,mhd->hm", x.abs(), ks.abs())
            prob = torch.softmax(score, -1)
            out[first + t] = torch.einsum("hm,mhd->hd", prob, vs)
            spread = score.amax(-1, keepdim=True) - score
            rel = 2 * delta.amax(-1, keepdim=True) + (spread + 6 + ks.shape[0]) * eps
            size = torch.einsum("hm,mhd->hd", prob * rel, vs.abs())
            size += torch.einsum("hm,mhd->hd", prob, vs.abs()) * (prob * rel).sum(-1, keepdim=True)
            bound[first + t] = size + 2.0 ** -140
    return out.view(q.shape), bound.view(q.shape)


def prepare(qkv, lengths, starts, slots, heads, kv_heads, dim, qw, kw, eps, cos, sin):
    """Rotated q [rows, heads, dim], and per sequence its new keys and values, in 64 bits."""
    def rotated(x, w, p):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        c, s = cos[p].double()[:, None], sin[p].double()[:, None]
        return torch.cat([a * c - b * s, a * s + b * c], -1)
    q = torch.zeros(qkv.shape[0], heads, dim, dtype=torch.float64)
    new = []
    for i, s in enumerate(slots):
        n = starts[i + 1] - starts[i]
        length = int(lengths[s])
        skip = max(0, n - length)
        rows = qkv[starts[i] + skip:starts[i + 1]].view(n - skip, heads + 2 * kv_heads, dim)
        p = torch.arange(length - n + skip, length)
        q[starts[i] + skip:starts[i + 1]] = rotated(rows[:, :heads], qw, p)
        new.append((p, rotated(rows[:, heads:heads + kv_heads], kw, p),
                    rows[:, heads + kv_heads:].double()))
    return q, new


def norm_error(got, want):
    return float((got.double() - want).norm() / want.norm().clamp_min(math.ulp(0.0)))
