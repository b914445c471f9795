"""Several sequences where element counts pass 32 bits: the ends of large pools,
of long packs of rows and of many rows of logits, against small calls."""
import pytest
import torch

import ikv
from batch_ref import assert_near, attention64, attention_bound, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _return_memory():
    yield
    torch.cuda.empty_cache()


def _dev32(x, dev):
    return torch.as_tensor(x, dtype=torch.int32).to(dev)


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (4, 2, 200)])
def test_the_end_of_a_large_pool(dev, heads, kv, dim):
    """Append, prompts and decode in blocks behind 2^31 floats: the bits of the
    same calls in a pool of those blocks alone."""
    bt, used, rows = 64, 6, [70, 3, 130]
    first = 2 ** 31 // (kv * dim) // bt + 1
    g = torch.Generator(device=dev)
    g.manual_seed(dim)
    rnd = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    n = sum(rows)
    k, v, q = rnd(n, kv, dim), rnd(n, kv, dim), rnd(n, heads, dim)
    one_q, one_k, one_v = rnd(3, heads, dim), rnd(3, kv, dim), rnd(3, kv, dim)
    start, n_kv = _dev32(starts(rows), dev), _dev32([r + 1 for r in rows], dev)
    table = torch.tensor([[1, 4, 0], [3, 0, 0], [0, 2, 5]], dtype=torch.int32, device=dev)
    results = []
    for ahead in (0, first):
        pools = [torch.empty((ahead + used) * bt, kv, dim, device=dev) for _ in range(2)]
        for p in pools:
            p[ahead * bt:] = 0
        tab = table + ahead
        ikv.append_packed(*pools, k, v, tab, bt, start)
        out = ikv.attn_prefill_packed_paged(q, *pools, tab, bt, start)
        one = ikv.attn_decode_batch(one_q, *pools, tab, bt, n_kv, k_new=one_k, v_new=one_v)
        results.append([out, one] + [p[ahead * bt:].clone() for p in pools])
        del pools
    for small, large in zip(*results):
        assert torch.equal(small, large)


def test_the_end_of_a_long_pack(dev):
    """Rows of q and out behind 2^31 floats."""
    n_seq, each, heads, dim = 4200, 63, 64, 128
    n = n_seq * each
    assert n * heads * dim > 2 ** 31
    q, out = (torch.zeros(n, heads, dim, device=dev) for _ in range(2))
    g = torch.Generator(device=dev)
    g.manual_seed(9)
    k, v = (torch.randn(n, 1, dim, generator=g, device=dev) for _ in range(2))
    q[-2 * each:] = torch.randn(2 * each, heads, dim, generator=g, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ikv.attn_prefill_packed(q, k, v, _dev32(starts([each] * n_seq), dev), out=out, status=status)
    assert status.item() == 0
    for s in (n_seq - 2, n_seq - 1):
        at = slice(s * each, (s + 1) * each)
        assert_near(out[at], attention64(q[at], k[at], v[at], 0), attention_bound(q[at], k[at], v[at]))


def test_many_rows_of_logits(dev):
    """Rows behind 2^31 logits give the tokens that they give alone."""
    n, vocab = 14200, 151936
    assert n * vocab > 2 ** 31
    g = torch.Generator(device=dev)
    g.manual_seed(4)
    x = torch.empty(n, vocab, device=dev).normal_(generator=g).mul_(3)
    u, p = torch.rand(n, generator=g, device=dev), torch.full((n,), 0.9, device=dev)
    token, logprob = ikv.sample(x, u, top_p=p)
    for rows in (slice(0, 2), slice(n - 3, n)):
        some, some_logprob = ikv.sample(x[rows], u[rows], top_p=p[rows])
        assert torch.equal(token[rows], some) and torch.equal(logprob[rows], some_logprob)
    assert (token >= 0).all() and (token < vocab).all() and torch.isfinite(logprob).all()
