"""The operators of a step over several sequences, as cases to be timed and
checked: each in a plain form (elementary torch operations) and as the calls
that a user makes of `ikv`.

  append   K and V rows of several sequences' new tokens, packed one sequence
           behind the other, into the sequences' pages
  prefill  causal attention with grouped heads over several packed prompts, or
           chunks of prompts behind what is already in a paged cache
  decode   one new token of each of several sequences over a paged cache of
           different lengths, with the append of the token's K and V row
  sample   the next token of each row of logits: temperature, top-k, top-p and
           min-p, from given uniform numbers

Head layouts are those of the library's presets (16 and 32 query heads over 8
KV heads of 128), of its tests' 12 heads of 64 over 4, and, drawn, a few other
sizes; vocabularies are the presets' and the tests' small one. All data is F32,
as the library's.
"""
import math
import os
import random
import sys

import torch

own = False


def listed():
    return [
        # the new rows of a few chats' prompts: launch latency
        dict(name="append_chats", kind="append", kv=8, dim=128, seqs=5, rows=211, past=700, block=64),
        # the prompts of a full batch
        dict(name="append_prompts", kind="append", kv=8, dim=128, seqs=24, rows=8190, past=0, block=256),
        # the first step of a few short chats
        dict(name="prefill_chats", kind="prefill", heads=16, kv=8, dim=128, seqs=6, rows=160, past=0,
             block=64),
        # an ordinary batch of prompts of very different lengths, no cache involved
        dict(name="prefill_prompts", kind="prefill", heads=16, kv=8, dim=128, seqs=16, rows=7001, past=0,
             block=0),
        # prompts that continue cached histories, in the head layout of the tests' other model
        dict(name="prefill_h64_chunks", kind="prefill", heads=12, kv=4, dim=64, seqs=9, rows=1999,
             past=1500, block=64),
        # the largest: long prompts of the large preset, some of them behind a history
        dict(name="prefill_8b_long", kind="prefill", heads=32, kv=8, dim=128, seqs=5, rows=8192,
             past=2000, block=256),
        # a decode step of three young chats and an idle slot: latency
        dict(name="decode_chats", kind="decode", heads=16, kv=8, dim=128, seqs=4, ctx=150, idle=1,
             block=64),
        # an ordinary decode step: contexts of very different lengths
        dict(name="decode_h64_batch", kind="decode", heads=12, kv=4, dim=64, seqs=37, ctx=5003, idle=2,
             block=64),
        # the largest: many long contexts of the large preset
        dict(name="decode_8b_long", kind="decode", heads=32, kv=8, dim=128, seqs=48, ctx=16384, idle=0,
             block=256),
        # one chat's next token
        dict(name="sample_one", kind="sample", rows=1, vocab=151936, std=3.0, coarse=False),
        # a batch of requests with settings of their own
        dict(name="sample_batch", kind="sample", rows=48, vocab=151936, std=2.5, coarse=True),
        # a large batch over the small vocabulary, the distribution nearly flat
        dict(name="sample_small_vocab", kind="sample", rows=200, vocab=8191, std=0.5, coarse=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "prefill", "prefill", "decode", "decode", "sample"])
    if kind == "sample":
        vocab = rng.choice([151936, _log_int(rng, 100, 151936)])
        return dict(kind=kind, rows=_log_int(rng, 1, 48), vocab=vocab, std=rng.uniform(0.5, 5.0),
                    coarse=rng.random() < 0.5)
    heads, kv, dim = rng.choice([(16, 8, 128), (32, 8, 128), (12, 4, 64), (8, 8, 96), (16, 1, 80)])
    seqs, block = _log_int(rng, 1, 48), rng.choice([64, 128, 256])
    if kind == "decode":
        return dict(kind=kind, heads=heads, kv=kv, dim=dim, seqs=seqs, ctx=_log_int(rng, 1, 16384),
                    idle=rng.randrange(min(seqs, 3)), block=block)
    past = rng.choice([0, _log_int(rng, 1, 2000)])
    if kind == "append":
        return dict(kind=kind, kv=kv, dim=dim, seqs=seqs, rows=_log_int(rng, seqs, 8192), past=past,
                    block=block)
    return dict(kind=kind, heads=heads, kv=kv, dim=dim, seqs=seqs, rows=_log_int(rng, seqs, 4000),
                past=past, block=rng.choice([0, block]) if past == 0 else block)


# ---------------------------------------------------------------------------
# sizes that follow from a case alone
# ---------------------------------------------------------------------------

def _rng_of(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    """Rows of each sequence (they add up to `rows`, each at least one) and the
    tokens cached before them."""
    rng = _rng_of(case)
    n, total = case["seqs"], case["rows"]
    share = [math.exp(rng.uniform(0.0, math.log(24.0))) for _ in range(n)]
    rows = [1 + int((total - n) * s / sum(share)) for s in share]
    rows[rng.randrange(n)] += total - sum(rows)
    past = [rng.randint(0, case["past"]) for _ in range(n)]
    return rows, past


def _contexts(case):
    """Keys of each sequence, the new token's among them; idle slots have none."""
    rng = _rng_of(case)
    n, ctx = case["seqs"], case["ctx"]
    got = [ctx] + [_log_int(rng, max(1, ctx // 16), ctx) for _ in range(n - 1)]
    rng.shuffle(got)
    for at in rng.sample(range(n), case["idle"]):
        got[at] = 0
    return got


def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4.0 * n + 28.0 * case["rows"], "flops": 0.0}
    row = 4.0 * case["kv"] * case["dim"]  # bytes of a token's K or V row
    if kind == "append":
        return {"bytes": 4.0 * row * case["rows"], "flops": 0.0}
    q_row = 4.0 * case["heads"] * case["dim"]
    if kind == "decode":
        keys, live = sum(_contexts(case)), sum(c > 0 for c in _contexts(case))
        return {"bytes": 2 * row * keys + 2 * row * live + 2 * q_row * case["seqs"], "flops": q_row * keys}
    rows, past = _lengths(case)
    seen = sum(r * p + r * (r + 1) / 2 for r, p in zip(rows, past))
    keys = sum(rows) + (sum(past) if case["block"] else 0)
    return {"bytes": 2 * row * keys + 2 * q_row * sum(rows), "flops": q_row * seen}


# ---------------------------------------------------------------------------
# inputs, made from the seed alone
# ---------------------------------------------------------------------------

class _Source:
    """Seeded device tensors, in the order they are asked for."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.gen, device="cuda").mul_(std)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def pages(self, tokens, block):
        """Block tables [sequences, blocks] over a shuffled pool, and the pool's
        blocks. Entries behind a sequence's last block are never to be read."""
        need = [-(-t // block) for t in tokens]
        width, total = max(1, max(need)), sum(need) + 3
        order = torch.randperm(total, generator=self.gen, device="cuda").to(torch.int32)
        tables = torch.full((len(tokens), width), -1, dtype=torch.int32, device="cuda")
        held = torch.arange(width, device="cuda")[None, :] < _device(need)[:, None]
        tables[held] = order[:sum(need)]
        return tables, total


def _device(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _prepare_sample(case, src):
    n, vocab = case["rows"], case["vocab"]
    logits = src.normal(n, vocab, std=case["std"])
    if case["coarse"]:  # as a head with 8-bit mantissas leaves them: many ties
        logits = logits.to(torch.bfloat16).to(torch.float32)
    # a quarter of the rows may use half of the vocabulary only
    masked = (src.uniform(n, 1) < 0.25) & (src.uniform(n, vocab) < 0.5)
    masked[:, vocab // 2] = False
    logits.masked_fill_(masked, -math.inf)
    u, pick = src.uniform(n), src.uniform(4, n)
    temperature = torch.where(pick[0] < 0.1, 0.0, 0.6 + 0.7 * src.uniform(n))
    top_k = torch.where(pick[1] < 0.5, 0.0, 1 + 199 * src.uniform(n)).to(torch.int32)
    top_p = torch.where(pick[2] < 0.3, 1.0, 0.7 + 0.29 * src.uniform(n))
    min_p = torch.where(pick[3] < 0.6, 0.0, 0.01 + 0.1 * src.uniform(n))
    return dict(logits=logits, u=u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


def prepare(case, seed):
    src = _Source(seed)
    kind = case["kind"]
    if kind == "sample":
        return dict(_prepare_sample(case, src), kind=kind)
    kv, dim, block = case["kv"], case["dim"], case["block"]
    s = dict(kind=kind, block=block)
    if kind == "decode":
        contexts = _contexts(case)
        s["n_kv"], s["longest"] = _device(contexts), max(contexts)
        s["live"] = _device([i for i, c in enumerate(contexts) if c], torch.int64)
        s["tables"], blocks = src.pages(contexts, block)
        s["q"] = src.normal(case["seqs"], case["heads"], dim)
        s["k_new"] = src.normal(case["seqs"], kv, dim)
        s["v_new"] = src.normal(case["seqs"], kv, dim, std=0.6)
    else:
        rows, past = _lengths(case)
        s["row_start"] = _device([0] + [sum(rows[:i + 1]) for i in range(len(rows))])
        s["longest"] = max(rows), max(r + (p if block else 0) for r, p in zip(rows, past))
        if kind == "prefill":
            s["q"] = src.normal(case["rows"], case["heads"], dim)
        if not block:
            s["k"], s["v"] = src.normal(case["rows"], kv, dim), src.normal(case["rows"], kv, dim, std=0.6)
            return s
        s["past"] = _device(past)
        s["tables"], blocks = src.pages([r + p for r, p in zip(rows, past)], block)
        if kind == "append":
            s["k_rows"] = src.normal(case["rows"], kv, dim)
            s["v_rows"] = src.normal(case["rows"], kv, dim, std=0.6)
    # rows that no table names hold whatever was there
    s["k_pool"] = src.normal(blocks * block, kv, dim)
    s["v_pool"] = src.normal(blocks * block, kv, dim, std=0.6)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _pool_rows(tables, block, seq, token):
    """Pool row of a token of a sequence (elementwise over index tensors)."""
    return tables[seq, token // block].long() * block + token % block


def _packed_places(row_start, n):
    """Sequence of each packed row and its place in it."""
    i = torch.arange(n, device="cuda")
    seq = torch.searchsorted(row_start[1:].long(), i, right=True)
    return seq, i - row_start.long()[seq]


def _plain_append(s):
    seq, t = _packed_places(s["row_start"], s["k_rows"].shape[0])
    rows = _pool_rows(s["tables"], s["block"], seq, s["past"].long()[seq] + t)
    s["k_pool"][rows] = s["k_rows"]
    s["v_pool"][rows] = s["v_rows"]
    return [s["k_pool"], s["v_pool"]]


def _padded_keys(s, lengths, width):
    """Keys and values of every sequence from its pages, padded to the longest:
    [sequences, width, KV heads, dim]."""
    n = lengths.shape[0]
    token = torch.arange(width, device="cuda")[None, :].expand(n, width)
    token = torch.minimum(token, (lengths - 1).clamp(min=0)[:, None])
    seq = torch.arange(n, device="cuda")[:, None].expand(n, width)
    rows = _pool_rows(s["tables"], s["block"], seq, token).clamp_(min=0)
    return s["k_pool"][rows], s["v_pool"][rows]


def _attention(q, k, v, sees):
    """softmax(q k / sqrt(dim)) v for q [S, L, H, D], k and v [S, K, KV, D];
    sees [S, L, K]: the keys that a query sees. A query that sees none gets 0."""
    S, L, H, D = q.shape
    KV = k.shape[2]
    G = H // KV
    q = q.reshape(S, L, KV, G, D).permute(0, 2, 3, 1, 4).reshape(S, KV, G * L, D)
    k = k.permute(0, 2, 3, 1).contiguous()
    v = v.permute(0, 2, 1, 3).contiguous()
    x = torch.matmul(q, k).mul_(1.0 / math.sqrt(D)).view(S, KV, G, L, -1)
    x.masked_fill_(~sees[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    x.div_(torch.where(total == 0, torch.ones_like(total), total))
    o = torch.matmul(x.view(S, KV, G * L, -1), v)
    return o.view(S, KV, G, L, D).permute(0, 3, 1, 2, 4).reshape(S, L, H, D)


def _plain_prefill(s):
    q = s["q"]
    start = s["row_start"].long()
    rows = start[1:] - start[:-1]
    past = s["past"].long() if "past" in s else torch.zeros_like(rows)
    lengths = past + rows
    width_q, width = s["longest"]
    seq, t = _packed_places(s["row_start"], q.shape[0])
    padded = torch.zeros(rows.shape[0], width_q, *q.shape[1:], device="cuda")
    padded[seq, t] = q
    if "past" in s:
        k, v = _padded_keys(s, lengths, width)
    else:
        k = torch.zeros(rows.shape[0], width, *s["k"].shape[1:], device="cuda")
        v = torch.zeros_like(k)
        k[seq, t], v[seq, t] = s["k"], s["v"]
    last = past[:, None] + torch.arange(width_q, device="cuda")[None, :]
    sees = torch.arange(width, device="cuda")[None, None, :] <= last[:, :, None]
    return _attention(padded, k, v, sees)[seq, t]


def _plain_decode(s):
    n_kv = s["n_kv"].long()
    live = s["live"]
    rows = _pool_rows(s["tables"], s["block"], live, n_kv[live] - 1)
    s["k_pool"][rows] = s["k_new"][live]
    s["v_pool"][rows] = s["v_new"][live]
    width = s["longest"]
    k, v = _padded_keys(s, n_kv, width)
    sees = torch.arange(width, device="cuda")[None, None, :] < n_kv[:, None, None]
    return [_attention(s["q"][:, None], k, v, sees)[:, 0], s["k_pool"], s["v_pool"]]


def _plain_sample(s):
    # in 64 bits: a running sum next to a border decides the token
    x, order = torch.sort(s["logits"], dim=-1, descending=True, stable=True)
    n, vocab = x.shape
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    y = (x.double() - x[:, :1].double()) / t
    w = torch.exp(y)
    run = torch.cumsum(w, -1)
    at = torch.arange(vocab, device="cuda")[None, :]
    top_k = torch.where((s["top_k"] <= 0) | (s["top_k"] > vocab), vocab, s["top_k"]).long()[:, None]
    mass_k = run.gather(1, top_k - 1)
    before = run - w
    p = s["top_p"].double()[:, None]
    kept = (at < top_k) & ((before < p * mass_k) | (p >= 1)) & (y >= torch.log(s["min_p"].double())[:, None])
    kept[:, 0] = True
    count = kept.sum(-1, keepdim=True)
    mass = run.gather(1, count - 1)
    target = s["u"].double()[:, None] * mass
    pick = torch.minimum((run <= target).sum(-1, keepdim=True), count - 1)
    pick = torch.where(greedy[:, None], torch.zeros_like(pick), pick)
    token = order.gather(1, pick)[:, 0].to(torch.int32)
    logprob = (y.gather(1, pick) - torch.log(mass))[:, 0]
    return [token, torch.where(greedy, torch.zeros_like(logprob), logprob).float()]


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------

def _library():
    if "ikv" not in sys.modules:
        sys.path.insert(1, os.path.join(os.getcwd(), "infer-llm_amd"))
    import ikv
    return ikv


def _own(s):
    ikv = _library()
    kind = s["kind"]
    if kind == "append":
        ikv.append_packed(s["k_pool"], s["v_pool"], s["k_rows"], s["v_rows"], s["tables"], s["block"],
                          s["row_start"], s["past"])
        return [s["k_pool"], s["v_pool"]]
    if kind == "prefill":
        if "past" not in s:
            return ikv.attn_prefill_packed(s["q"], s["k"], s["v"], s["row_start"])
        return ikv.attn_prefill_packed_paged(s["q"], s["k_pool"], s["v_pool"], s["tables"], s["block"],
                                             s["row_start"], s["past"])
    if kind == "decode":
        if "workspace" not in s:  # one for all steps of a program
            s["workspace"] = ikv.decode_batch_workspace(s["q"].shape[1], s["k_pool"].shape[1],
                                                        s["q"].shape[2])
        out = ikv.attn_decode_batch(s["q"], s["k_pool"], s["v_pool"], s["tables"], s["block"], s["n_kv"],
                                    k_new=s["k_new"], v_new=s["v_new"], workspace=s["workspace"])
        return [out, s["k_pool"], s["v_pool"]]
    if "workspace" not in s:
        s["workspace"] = ikv.sample_workspace(*s["logits"].shape)
    return list(ikv.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                           top_p=s["top_p"], min_p=s["min_p"], workspace=s["workspace"]))


def run(state):
    if own:
        return _own(state)
    plain = {"append": _plain_append, "prefill": _plain_prefill, "decode": _plain_decode,
             "sample": _plain_sample}
    return plain[state["kind"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits, a sequence and a row at a time
# ---------------------------------------------------------------------------

def _exact_heads(q, k, v, past):
    """q [L, H, D] over k, v [K, KV, D], in 64 bits; query t sees past + t + 1 keys."""
    L, H, D = q.shape
    out = torch.empty(L, H, D, dtype=torch.float64, device="cuda")
    key = torch.arange(k.shape[0], device="cuda")
    for h in range(H):
        kk, vv = k[:, h * k.shape[1] // H].double(), v[:, h * k.shape[1] // H].double()
        for a in range(0, L, 1024):
            b = min(L, a + 1024)
            x = q[a:b, h].double() @ kk.T / math.sqrt(D)
            sees = key[None, :] <= past + torch.arange(a, b, device="cuda")[:, None]
            out[a:b, h] = torch.softmax(x.masked_fill(~sees, -math.inf), -1) @ vv
    return out


def _places(s, i, tokens):
    """Pool rows of one sequence's tokens."""
    block, blocks = s["block"], s["tables"][i].tolist()
    return torch.tensor([blocks[t // block] * block + t % block for t in tokens], device="cuda")


def _sequence(s, i, length):
    """K and V of one sequence's first `length` tokens, from its pages."""
    at = _places(s, i, range(length))
    return s["k_pool"][at], s["v_pool"][at]


def _exact_sample(s):
    logprob = torch.zeros(s["logits"].shape[0], dtype=torch.float64, device="cuda")
    for r in range(logprob.shape[0]):
        t = float(s["temperature"][r])
        if t <= 0:
            continue
        x = torch.sort(s["logits"][r].double(), descending=True)[0]
        y = (x - x[0]) / t
        keep = int(s["top_k"][r])
        y = y[:keep] if 0 < keep < y.shape[0] else y
        mass = torch.exp(y)
        if float(s["top_p"][r]) < 1.0:
            need = float(s["top_p"][r]) * float(mass.sum())
            y = y[:max(1, int((mass.cumsum(0) - mass < need).sum()))]
        low = float(s["min_p"][r])
        if low > 0.0:
            y = y[:max(1, int((y >= math.log(low)).sum()))]
        run_ = torch.exp(y).cumsum(0)
        pick = min(int((run_ <= float(s["u"][r]) * float(run_[-1])).sum()), y.shape[0] - 1)
        logprob[r] = y[pick] - math.log(float(run_[-1]))
    return [None, logprob]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "append":
        pools, start = [s["k_pool"].double(), s["v_pool"].double()], 0
        for i, (rows, past) in enumerate(zip(*_lengths(case))):
            at = _places(s, i, range(past, past + rows))
            for pool, new in zip(pools, (s["k_rows"], s["v_rows"])):
                pool[at] = new[start:start + rows].double()
            start += rows
        return pools
    if kind == "sample":
        return _exact_sample(s)
    if kind == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for i, n in enumerate(_contexts(case)):
            if n:
                k, v = _sequence(s, i, n)
                k[-1], v[-1] = s["k_new"][i], s["v_new"][i]
                out[i:i + 1] = _exact_heads(s["q"][i:i + 1], k, v, n - 1)
        return [out, None, None]
    out, at = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (rows, past) in enumerate(zip(*_lengths(case))):
        if case["block"]:
            k, v = _sequence(s, i, past + rows)
        else:
            past, k, v = 0, s["k"][at:at + rows], s["v"][at:at + rows]
        out[at:at + rows] = _exact_heads(s["q"][at:at + rows], k, v, past)
        at += rows
    return out
