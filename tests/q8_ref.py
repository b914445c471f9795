"""What the tests of the cache of 8 bits an element share: the formats in 64 bits on
the CPU, caches over shuffled pages, and how far a decode over them may be off."""
import math

import numpy as np
import torch

import ikv
from batch_ref import EPS, rows_of, tables_for

FORMATS = [torch.int8, torch.float8_e4m3fn]
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def bits(codes):
    """Codes as bytes."""
    return codes.view(torch.int8)


def quantised(x, dtype):
    """Codes and scales of rows x [..., dim] by the definition, in 64 bits on the CPU."""
    x = x.detach().cpu().double()
    top = x.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(x).all(-1, keepdim=True)
    unit = torch.where(fine & (top > 0), top, torch.ones_like(top))
    y = torch.where(fine, x, torch.zeros_like(x)) * TOP[dtype] / unit
    codes = torch.round(y).to(torch.int8) if dtype is torch.int8 else y.float().to(dtype)
    scales = torch.where(fine, top / TOP[dtype], torch.full_like(top, math.nan))[..., 0]
    return codes, scales.float()


def values(codes, scales):
    """What codes and scales stand for, in 64 bits."""
    return codes.detach().cpu().double() * scales.detach().cpu().double()[..., None]


def place(cache, tables, s, bt, tokens):
    """Block and place in it of tokens of sequence s, on the cache's device."""
    at = torch.tensor(rows_of(tables, s, bt, tokens), dtype=torch.long, device=cache[1].device)
    return at // bt, at % bt


def held(cache, tables, s, bt, n):
    """(K, V) [n, n_head_kv, dim] of sequence s's first n tokens, in 64 bits."""
    if n == 0:
        return [torch.zeros(0, cache[0].shape[1], cache[0].shape[3], dtype=torch.float64)] * 2
    blk, at = place(cache, tables, s, bt, range(n))
    out = []
    for codes, scales in ((cache[0], cache[1]), (cache[2], cache[3])):
        c = bits(codes).movedim(1, 2)[blk, at].cpu().view(codes.dtype)
        out.append(values(c, scales.movedim(1, 2)[blk, at]))
    return out


def filled_cache(dev, gen, lengths, bt, kv, dim, dtype, seed, stale=True):
    """A cache that holds normal rows of the given lengths, and its tables. Places of
    no token hold codes of the largest size and NaN scales, which must not be read."""
    tables, blocks = tables_for(lengths, bt, seed)
    cache = ikv.cache_q8(blocks, bt, kv, dim, dtype, device=dev)
    if stale:
        for codes, scales in ((cache[0], cache[1]), (cache[2], cache[3])):
            bits(codes).fill_(127)  # (e4m3: NaN)
            scales.fill_(math.nan)
    for s, n in enumerate(lengths):
        if n == 0:
            continue
        blk, at = place(cache, tables, s, bt, range(n))
        for codes, scales in ((cache[0], cache[1]), (cache[2], cache[3])):
            c, sc = quantised(torch.randn(n, kv, dim, generator=gen, device=dev), dtype)
            bits(codes).movedim(1, 2)[blk, at] = bits(c).to(dev)
            scales.movedim(1, 2)[blk, at] = sc.to(dev)
    return cache, tables


def decode_bound(q, k, v, scale=None):
    """The most that an element of the decode may be off. A score is a sum of 3 D
    products of a code and a bf16 piece of the query, each exact, every addition
    rounded once at most, times a scale; with the query's own rounding to its scaled
    value, the key's scale and the exponent's argument (3 D + 12) EPS of the sum of its
    terms' sizes. That moves the weight, and its sum, by as much (2 x). A weight times
    the value's scale is rounded once, three pieces of it are added to a sum of 3 K
    terms; the parts' join and the division: (6 K + 16) EPS of the largest value."""
    D, K = q.shape[-1], k.shape[0]
    scale = scale or 1.0 / math.sqrt(D)
    terms = float(q.abs().amax()) * float(k.abs().sum(-1).amax()) * scale
    return ((2 * (3 * D + 12) * terms) + 6 * K + 16) * EPS * float(v.abs().amax())


def dev32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(dev)
