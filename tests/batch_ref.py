"""What the tests of a step over several sequences share: block tables, packed
sizes, attention in 64 bits, and how far F32 results may be from it."""
import math

import numpy as np
import torch

EPS = 2.0 ** -24  # the largest relative error of one F32 rounding


def tables_for(lengths, bt, seed, spare=3):
    """int32 block tables [n_seq, width] over a shuffled pool (-1 behind a
    sequence's last block), and the pool's blocks."""
    need = [-(-n // bt) for n in lengths]
    total = sum(need) + spare
    order = np.random.default_rng(seed).permutation(total)
    tables = np.full((len(lengths), max(1, max(need))), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        tables[s, :n] = order[at:at + n]
        at += n
    return tables, total


def rows_of(tables, s, bt, tokens):
    """Pool rows of tokens of sequence s."""
    return [int(tables[s, t // bt]) * bt + t % bt for t in tokens]


def starts(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


def attention64(q, k, v, past, scale=None):
    """Causal attention in 64 bits: q [L, H, D] behind `past` keys of k, v
    [K, KV, D]; query t sees keys 0 .. past + t."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    L, H, D = q.shape
    G = H // k.shape[1]
    scale = scale or 1.0 / math.sqrt(D)
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    x = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) * scale
    hidden = torch.arange(k.shape[0])[None, :] > past + torch.arange(L)[:, None]
    p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
    return torch.matmul(p, v.transpose(0, 1).contiguous()).transpose(0, 1)


def attention_bound(q, k, v, scale=None):
    """The most that an element of an F32 attention over these rows may be off,
    whatever the order of its sums. A score is a sum of D products, each
    operand or product rounded (or split into pieces) once, times the scale,
    and its exponent is rounded once more: at most (D + 8) EPS of the sum of
    its terms' sizes. That moves a weight by as much, relatively, and both the
    weighted sum and its divisor (2 x); the sums over K keys and the last
    division add (2 K + 8) EPS. All relative to the largest value."""
    D, K = q.shape[-1], k.shape[0]
    scale = scale or 1.0 / math.sqrt(D)
    terms = float(q.abs().amax()) * float(k.abs().sum(-1).amax()) * scale
    return ((2 * (D + 8) * terms) + 2 * K + 8) * EPS * float(v.abs().amax())


# The 2-norm of the error over that of the result, for normal data and scores
# of size 1. The roundings are independent: of a score, a sum of D products, by
# about EPS sqrt(D) of a term's size over sqrt(D), and as much for the exponent
# (its argument reaches 5, in units of which it is rounded) and the weight;
# together some 8 EPS, which averages over the keys as the values do. Four times
# that.
NORMAL_REL = 32 * EPS


def assert_near(got, want, bound, rel=NORMAL_REL):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all()
    off = (got - want).abs().max().item()
    assert off <= bound, f"off by {off:.3g}, at most {bound:.3g}"
    norm = want.norm().item()
    if rel is not None and norm > 0:
        far = (got - want).norm().item() / norm
        assert far <= rel, f"2-norm off by {far:.3g}, at most {rel:.3g}"
