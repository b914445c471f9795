"""Steps of a small model over several sequences, as a server runs them: packed
prompts, packed append, batched decode and sampling on one paged cache, with
sequences that join and leave. Against the same model run one sequence at a time
through the library's single-sequence calls."""
import numpy as np
import pytest
import torch

import ikv
from batch_ref import rows_of, starts, tables_for
from test_gpu_sample import reference

pytestmark = pytest.mark.gpu

E, H, KV, D, VOCAB, LAYERS, BT, CTX = 256, 8, 4, 64, 700, 2, 64, 512
EPS = 1e-6
# Logits of 256-term sums over two layers, each rounded some 20 times on the way,
# values of size 1: both sides are off by at most 20 sqrt(256) 2^-24 = 2e-5 of
# them, and sums in another order by as much.
LOGITS = 1e-4


class Model:
    def __init__(self, dev):
        g = torch.Generator(device=dev)
        g.manual_seed(123)
        rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
        self.embed = rnd(VOCAB, E)
        self.layers = [dict(norm=1 + 0.1 * rnd(E), q=rnd(H * D, E) / 16, k=rnd(KV * D, E) / 16,
                            v=rnd(KV * D, E) / 16, o=rnd(E, H * D) / 23, qn=1 + 0.1 * rnd(D),
                            kn=1 + 0.1 * rnd(D)) for _ in range(LAYERS)]
        self.norm, self.head = 1 + 0.1 * rnd(E), rnd(VOCAB, E) / 16
        s, c = ikv.rope_sincos_table(ikv.rope_theta_table(1e4, D, CTX))
        self.sin, self.cos = torch.from_numpy(s).to(dev), torch.from_numpy(c).to(dev)

    def qkv(self, w, x, pos):
        h = ikv.rms_norm(x, w["norm"], EPS)
        n = x.shape[0]
        q = ikv.qk_norm_rope(ikv.mul_mat(w["q"], h).view(n, H, D), w["qn"], pos, EPS, self.sin, self.cos)
        k = ikv.qk_norm_rope(ikv.mul_mat(w["k"], h).view(n, KV, D), w["kn"], pos, EPS, self.sin, self.cos)
        return q, k, ikv.mul_mat(w["v"], h).view(n, KV, D)

    def logits(self, x):
        return ikv.mul_mat(self.head, ikv.rms_norm(x, self.norm, EPS))


def _i32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).to(dev)


class Server:
    """The batch: pools, tables and lengths of a fixed number of slots."""

    def __init__(self, model, dev, slots):
        self.m, self.dev = model, dev
        tables, blocks = tables_for([CTX] * slots, BT, seed=5)
        self.host_tables, self.tables = tables, _i32(tables, dev)
        self.pools = [[torch.zeros(blocks * BT, KV, D, device=dev) for _ in range(2)] for _ in range(LAYERS)]
        self.length = [0] * slots
        self.workspace = ikv.decode_batch_workspace(H, KV, D)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)

    def prompts(self, rows):
        """rows: {slot: token ids} packed in slot order; the logits of each one's
        last token."""
        dev, sizes = self.dev, [len(rows.get(s, [])) for s in range(len(self.length))]
        start, past = _i32(starts(sizes), dev), _i32(self.length, dev)
        ids = _i32([t for s in sorted(rows) for t in rows[s]], dev)
        pos = _i32([self.length[s] + i for s in sorted(rows) for i in range(len(rows[s]))], dev)
        x = ikv.get_rows(self.m.embed, ids)
        for w, pools in zip(self.m.layers, self.pools):
            q, k, v = self.m.qkv(w, x, pos)
            ikv.append_packed(*pools, k, v, self.tables, BT, start, past, status=self.status)
            a = ikv.attn_prefill_packed_paged(q, *pools, self.tables, BT, start, past, status=self.status)
            x = ikv.mul_mat(w["o"], a.view(-1, H * D), residual=x)
        for s in rows:
            self.length[s] += len(rows[s])
        last = _i32([e - 1 for e, n in zip(starts(sizes)[1:], sizes) if n], dev)
        return self.m.logits(ikv.get_rows(x, last))

    def decode(self, tokens):
        """tokens: {slot: the token that comes next}; other slots idle. Logits of
        every slot (an idle one's mean nothing)."""
        dev, slots = self.dev, len(self.length)
        for s in tokens:
            self.length[s] += 1
        n_kv = _i32([self.length[s] if s in tokens else 0 for s in range(slots)], dev)
        pos = _i32([self.length[s] - 1 if s in tokens else 0 for s in range(slots)], dev)
        x = ikv.get_rows(self.m.embed, _i32([tokens.get(s, 0) for s in range(slots)], dev))
        for w, pools in zip(self.m.layers, self.pools):
            q, k, v = self.m.qkv(w, x, pos)
            a = ikv.attn_decode_batch(q, *pools, self.tables, BT, n_kv, k_new=k, v_new=v,
                                      workspace=self.workspace, status=self.status)
            x = ikv.mul_mat(w["o"], a.view(-1, H * D), residual=x)
        return self.m.logits(x)


class Alone:
    """One sequence through the single-sequence calls, on contiguous caches."""

    def __init__(self, model, dev):
        self.m, self.dev, self.n = model, dev, 0
        self.caches = [[torch.zeros(CTX, KV, D, device=dev) for _ in range(2)] for _ in range(LAYERS)]

    def feed(self, ids):
        pos = torch.arange(self.n, self.n + len(ids), dtype=torch.int32, device=self.dev)
        x = ikv.get_rows(self.m.embed, _i32(ids, self.dev))
        for w, (kc, vc) in zip(self.m.layers, self.caches):
            q, k, v = self.m.qkv(w, x, pos)
            kc[self.n:self.n + len(ids)], vc[self.n:self.n + len(ids)] = k, v
            if len(ids) == 1:
                a = ikv.attn_decode(q[0], kc, vc, self.n + 1)[None]
            else:
                a = ikv.attn_prefill(q, kc, vc, self.n)
            x = ikv.mul_mat(w["o"], a.reshape(-1, H * D), residual=x)
        self.n += len(ids)
        return self.m.logits(x[-1:].contiguous())[0]


def test_steps_of_a_batch_equal_its_sequences_alone(dev):
    rng = np.random.default_rng(3)
    model, slots = Model(dev), 6
    server, alone = Server(model, dev, slots), {}
    temperature, top_k, top_p, min_p = [0.0, 0.8, 1.0, 1.3, 0.7, 1.0], [0, 20, 0, 50, 0, 1], [1.0, 0.9, 0.8, 1.0, 0.95, 1.0], [0, 0, 0.05, 0, 0.1, 0]
    texts = {}

    def near(got, want, what):
        off = (got - want).abs().max().item()
        assert off <= LOGITS * max(1.0, want.abs().max().item()), f"{what}: logits off by {off:.3g}"

    def draw(logits, which):
        u = rng.random(len(which)).astype(np.float32)
        pick = lambda v, dt=torch.float32: torch.tensor([v[s] for s in which], dtype=dt, device=dev)  # noqa: E731
        token, logprob = ikv.sample(logits, torch.from_numpy(u).to(dev), temperature=pick(temperature),
                                    top_k=pick(top_k, torch.int32), top_p=pick(top_p), min_p=pick(min_p))
        rows = logits.cpu().numpy()
        for i, s in enumerate(which):
            as32 = lambda v: float(np.float32(v[s]))  # noqa: E731
            want, lp = reference(rows[i], float(u[i]), as32(temperature), top_k[s], as32(top_p), as32(min_p))
            assert token[i].item() == want
            assert abs(logprob[i].item() - lp) <= abs(lp) * 2.0 ** -23 + 1e-6
        return dict(zip(which, token.tolist()))

    def prompt(lengths):
        rows = {s: rng.integers(0, VOCAB, n).tolist() for s, n in lengths.items()}
        for s, ids in rows.items():
            texts.setdefault(s, []).extend(ids)
            alone.setdefault(s, Alone(model, dev))
        got = server.prompts(rows)
        for i, s in enumerate(sorted(rows)):
            near(got[i], alone[s].feed(rows[s]), f"prompt of slot {s}")
        return draw(got, sorted(rows))

    def step(tokens):
        got = server.decode(tokens)
        which = sorted(tokens)
        for s in which:
            near(got[s], alone[s].feed([tokens[s]]), f"step of slot {s}")
        return draw(got[which].contiguous(), which)

    # four requests, decoded together; then one leaves, two join (one with a prompt
    # in two chunks); then all that are there
    tokens = prompt({0: 70, 1: 1, 3: 130, 4: 7})
    for _ in range(4):
        tokens = step(tokens)
    del tokens[1]
    prompt({2: 64})
    joined = prompt({2: 40, 5: 200})
    tokens.update(joined)
    for _ in range(4):
        tokens = step(tokens)
    assert server.status.item() == 0
    # the caches hold what each sequence's own hold
    for layer in range(LAYERS):
        for s, a in alone.items():
            at = torch.tensor(rows_of(server.host_tables, s, BT, range(a.n)), device=dev)
            for pool, cache in zip(server.pools[layer], a.caches[layer]):
                assert (pool[at] - cache[:a.n]).abs().max().item() <= LOGITS * 4


def test_a_decode_step_captured_and_replayed(dev):
    """The step of a batch, sampling with it, as one graph: lengths, positions,
    tokens and uniform numbers are read anew, and the pools grow."""
    model, slots = Model(dev), 3
    eager, graphed = Server(model, dev, slots), Server(model, dev, slots)
    rng = np.random.default_rng(4)
    rows = {s: rng.integers(0, VOCAB, n).tolist() for s, n in enumerate((20, 90, 5))}
    for server in (eager, graphed):
        server.prompts(rows)
    n_kv, pos = _i32(graphed.length, dev), _i32(graphed.length, dev)
    ids, u = torch.zeros(slots, dtype=torch.int32, device=dev), torch.zeros(slots, device=dev)
    top_p = torch.full((slots,), 0.9, device=dev)
    space = ikv.sample_workspace(slots, VOCAB)

    def step():
        x = ikv.get_rows(model.embed, ids)
        for w, pools in zip(model.layers, graphed.pools):
            q, k, v = model.qkv(w, x, pos)
            a = ikv.attn_decode_batch(q, *pools, graphed.tables, BT, n_kv, k_new=k, v_new=v,
                                      workspace=graphed.workspace)
            x = ikv.mul_mat(w["o"], a.view(-1, H * D), residual=x)
        logits = model.logits(x)
        return logits, *ikv.sample(logits, u, top_p=top_p, workspace=space)

    # a first run outside the capture, on its stream (mul_mat allocates there),
    # that appends nothing
    n_kv.zero_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        logits, token, logprob = step()
    tokens = {s: s for s in range(slots)}
    for i in range(5):
        lengths = [len(rows[s]) + i + 1 for s in range(slots)]
        n_kv.copy_(torch.tensor(lengths, dtype=torch.int32))
        pos.copy_(torch.tensor([n - 1 for n in lengths], dtype=torch.int32))
        ids.copy_(torch.tensor([tokens[s] for s in range(slots)], dtype=torch.int32))
        u.copy_(torch.rand(slots))
        graph.replay()
        torch.cuda.synchronize()
        want = eager.decode(tokens)
        assert torch.equal(logits, want)
        again = ikv.sample(want, u, top_p=top_p)
        assert torch.equal(token, again[0]) and torch.equal(logprob, again[1])
        tokens = dict(enumerate(token.tolist()))
    for a, b in zip(eager.pools, graphed.pools):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("width", [0, 5])
def test_a_step_without_sequences(dev, width):
    """Nobody is active: nothing is written, nothing is refused."""
    kv, D = 2, 64
    pools = [torch.full((256, kv, D), 7.0, device=dev) for _ in range(2)]
    tables = torch.zeros((0, width), dtype=torch.int32, device=dev)
    none, start = torch.zeros(0, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev)
    for rows in (0, 3):  # (rows of no sequence)
        q, k = torch.randn(rows, 4, D, device=dev), torch.randn(rows, kv, D, device=dev)
        out = torch.full_like(q, 3.0)
        ikv.append_packed(*pools, k, k, tables, 64, start, none)
        assert ikv.attn_prefill_packed(q, k, k, start, out=out) is out
        for past in (none, None):
            assert ikv.attn_prefill_packed_paged(q, *pools, tables, 64, start, past, out=out) is out
        assert (out == 3.0).all()
    q, k = torch.randn(0, 4, D, device=dev), torch.randn(0, kv, D, device=dev)
    assert ikv.attn_decode_batch(q, *pools, tables, 64, none, k_new=k, v_new=k).shape == (0, 4, D)
    assert all((p == 7.0).all() for p in pools)
