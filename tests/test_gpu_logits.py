"""Penalties, biases and masks on rows of logits, against 64 bits."""
import math

import pytest
import torch

import ikv
from batch_ref import EPS
from q8_ref import dev32

pytestmark = pytest.mark.gpu


def _want(logits, history, n_history, n_prompt, rep, pres, freq, bias_tokens, bias_values, n_bias, masks, mask_of):
    """In 64 bits, a row and a token at a time, and the size of what was added up."""
    out = logits.detach().cpu().double().clone()
    size = out.abs()
    for r in range(out.shape[0]):
        count = {}
        for i in range(n_history[r]):
            t = int(history[r, i])
            count[t] = count.get(t, 0) + (1 if i >= n_prompt[r] else 0)
        for t, c in count.items():
            x = out[r, t]
            x = x / float(rep[r]) if x > 0 else x * float(rep[r])
            size[r, t] = max(float(size[r, t]), abs(float(x)))
            if c:
                x = x - float(freq[r]) * c - float(pres[r])
                size[r, t] += abs(float(freq[r])) * c + abs(float(pres[r]))
            out[r, t] = x
        last = {int(bias_tokens[r, i]): float(bias_values[r, i]) for i in range(n_bias[r])}
        for t, b in last.items():
            out[r, t] += b
            size[r, t] += abs(b)
        if masks is not None and mask_of[r] >= 0:
            words = masks[mask_of[r]].long()
            t = torch.arange(out.shape[1])
            out[r, (words[t // 32] >> (t % 32)) % 2 == 0] = -math.inf
    return out, size


def _near(got, want, size):
    """Each of the quotient or product, the two differences and the sum is rounded
    once, and so is frequency times the count: 5 roundings of at most EPS times what
    was added up so far."""
    got = got.detach().cpu().double()
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    fine = ~torch.isinf(want)
    assert ((got - want).abs()[fine] <= (5 * EPS * size)[fine]).all()


def _inputs(dev, seed, rows, vocab, history, biases, masks):
    g = torch.Generator()
    g.manual_seed(seed)
    small = max(2, vocab // 7)  # tokens come again and again
    d = dict(logits=torch.randn(rows, vocab, generator=g) * 3,
             history=torch.randint(0, small, (rows, history), generator=g, dtype=torch.int32),
             rep=1 + torch.rand(rows, generator=g), pres=torch.randn(rows, generator=g),
             freq=torch.rand(rows, generator=g) - 0.2,
             bias_tokens=torch.randint(0, vocab, (rows, biases), generator=g, dtype=torch.int32),
             bias_values=torch.randn(rows, biases, generator=g) * 5)
    d["n_history"] = torch.randint(0, history + 1, (rows,), generator=g).tolist()
    d["n_prompt"] = [int(torch.randint(0, n + 1, (1,), generator=g)) for n in d["n_history"]]
    d["n_bias"] = torch.randint(0, biases + 1, (rows,), generator=g).tolist()
    if masks:
        d["masks"] = torch.randint(-2 ** 31, 2 ** 31, (masks, (vocab + 31) // 32), generator=g).to(torch.int32)
        d["mask_of"] = (torch.randint(0, masks + 1, (rows,), generator=g) - 1).tolist()
    else:
        d["masks"], d["mask_of"] = None, None
    return d


def _call(dev, d, **more):
    args = dict(history=d["history"].to(dev), n_history=dev32(d["n_history"], dev), n_prompt=dev32(d["n_prompt"], dev),
                repetition=d["rep"].to(dev), presence=d["pres"].to(dev), frequency=d["freq"].to(dev),
                bias_tokens=d["bias_tokens"].to(dev), bias_values=d["bias_values"].to(dev),
                n_bias=dev32(d["n_bias"], dev))
    if d["masks"] is not None:
        args.update(masks=d["masks"].to(dev), mask_of=dev32(d["mask_of"], dev))
    return ikv.adjust_logits(d["logits"].to(dev), **{**args, **more})


@pytest.mark.parametrize("rows,vocab,history,biases,masks", [
    (1, 1, 1, 1, 1), (3, 31, 5, 2, 2), (2, 32, 100, 40, 1), (5, 33, 64, 1, 0), (7, 4096, 700, 33, 3),
    (4, 4097, 1, 1, 2), (3, 8191, 300, 100, 2), (2, 16384, 3000, 257, 5), (1, 151936, 900, 12, 1),
    (300, 500, 40, 3, 4)])
def test_against_64_bits(dev, rows, vocab, history, biases, masks):
    d = _inputs(dev, vocab + rows, rows, vocab, history, biases, masks)
    want, size = _want(**d)
    out = _call(dev, d)
    _near(out, want, size)
    assert torch.equal(_call(dev, d), out)


def test_in_place(dev):
    d = _inputs(dev, 3, 4, 5000, 200, 10, 2)
    want = _call(dev, d)
    x = d["logits"].to(dev)
    got = ikv.adjust_logits(x, out=x, history=d["history"].to(dev), n_history=dev32(d["n_history"], dev),
                            n_prompt=dev32(d["n_prompt"], dev), repetition=d["rep"].to(dev),
                            presence=d["pres"].to(dev), frequency=d["freq"].to(dev),
                            bias_tokens=d["bias_tokens"].to(dev), bias_values=d["bias_values"].to(dev),
                            n_bias=dev32(d["n_bias"], dev), masks=d["masks"].to(dev), mask_of=dev32(d["mask_of"], dev))
    assert got is x and torch.equal(x, want)


def test_parts_that_are_left_out(dev):
    x = torch.randn(3, 999, device=dev)
    x[0, 5] = math.nan
    x[1, 7] = -math.inf
    x[2, 9] = math.inf
    out = ikv.adjust_logits(x)
    assert torch.equal(out.view(torch.int32), x.view(torch.int32))
    tokens = dev32([[1, 2, 2], [3, 3, 3], [4, 5, 6]], dev)
    # only a presence: all tokens of the list, none from a prompt
    out = ikv.adjust_logits(x, history=tokens, presence=torch.tensor([1.0, 2.0, 0.5], device=dev))
    want = x.clone()
    for r, t, p in ((0, 1, 1.0), (0, 2, 1.0), (1, 3, 2.0), (2, 4, 0.5), (2, 5, 0.5), (2, 6, 0.5)):
        want[r, t] = x[r, t] - p
    assert torch.equal(out.view(torch.int32), want.view(torch.int32))
    # only a history: nothing changes
    assert torch.equal(ikv.adjust_logits(x, history=tokens).view(torch.int32), x.view(torch.int32))
    # one mask for all rows; what it hides may be anything
    words = torch.zeros(1, 32, dtype=torch.int32, device=dev)
    words[0, 0] = 1 << 4
    out = ikv.adjust_logits(x, masks=words)
    assert torch.equal(out[:, 4], x[:, 4])
    out[:, 4] = -math.inf
    assert (out == -math.inf).all()
    # an empty list of history and biases
    none = torch.empty(3, 0, dtype=torch.int32, device=dev)
    out = ikv.adjust_logits(x, history=none, bias_tokens=none, bias_values=none.float())
    assert torch.equal(out.view(torch.int32), x.view(torch.int32))


def test_infinities_and_the_largest_values(dev):
    """As the formula has it: -inf stays, a penalty may leave the range."""
    x = torch.tensor([[-math.inf, math.inf, 3e38, -3e38, 0.0, -0.0, 1.0, -1.0]], device=dev)
    every = dev32([list(range(8))], dev)
    out = ikv.adjust_logits(x, history=every, repetition=torch.tensor([2.0], device=dev)).cpu()[0]
    assert out[0] == -math.inf and out[1] == math.inf and out[2] == 1.5e38 and out[3] == -math.inf
    assert (out[4:6] == 0).all() and out[6] == 0.5 and out[7] == -2.0


def test_tokens_lengths_and_masks_out_of_range(dev):
    x = torch.randn(4, 100, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    one = torch.ones(4, device=dev)
    tokens = dev32([[5, 100, -1, 7]] * 4, dev)
    out = ikv.adjust_logits(x, history=tokens, presence=one, status=status)
    assert status.item() == 4
    want = x.clone()
    want[:, [5, 7]] -= 1.0
    assert torch.equal(out, want)
    status.zero_()
    out = ikv.adjust_logits(x, history=tokens[:, :1].contiguous(), n_history=dev32([2, -1, 1, 0], dev), presence=one,
                            status=status)
    assert status.item() == 1
    want = x.clone()
    want[2, 5] -= 1.0
    assert torch.equal(out, want)
    status.zero_()
    out = ikv.adjust_logits(x, bias_tokens=dev32([[1, 200]] * 4, dev), bias_values=torch.ones(4, 2, device=dev),
                            n_bias=dev32([2, 3, 1, -7], dev), status=status)
    assert status.item() == 1 | 4
    want = x.clone()
    want[[0, 2], 1] += 1.0
    assert torch.equal(out, want)
    status.zero_()
    masks = torch.full((2, 4), -1, dtype=torch.int32, device=dev)
    out = ikv.adjust_logits(x, masks=masks, mask_of=dev32([0, 2, -1, 1], dev), status=status)
    assert status.item() == 1
    assert (out[1] == -math.inf).all() and torch.equal(out[[0, 2, 3]], x[[0, 2, 3]])
    # a row that allows nothing is the sampler's -1
    token, _ = ikv.sample(out, torch.full((4,), 0.5, device=dev))
    assert token[1].item() == -1 and (token[[0, 2, 3]] >= 0).all()
    # n_prompt past the history: all of it is the prompt's
    out = ikv.adjust_logits(x, history=tokens[:, :1].contiguous(), n_prompt=dev32([9, 1, 0, -5], dev), presence=one)
    want = x.clone()
    want[2:, 5] -= 1.0
    assert torch.equal(out, want)


def test_of_biases_for_one_token_the_last_counts(dev):
    x = torch.zeros(1, 64, device=dev)
    n = 1000
    tokens = dev32([[7] * (n - 1) + [9]], dev)
    values = torch.arange(n, dtype=torch.float32, device=dev)[None]
    out = ikv.adjust_logits(x, bias_tokens=tokens, bias_values=values)
    assert out[0, 7] == n - 2 and out[0, 9] == n - 1 and out.sum() == 2 * n - 3


def test_captured_over_growing_histories(dev):
    rows, vocab = 5, 2000
    x = torch.randn(rows, vocab, device=dev)
    history = torch.randint(0, vocab, (rows, 50), device=dev, dtype=torch.int32)
    n = dev32([1] * rows, dev)
    pen = torch.full((rows,), 0.25, device=dev)
    out = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ikv.adjust_logits(x, history=history, n_history=n, frequency=pen, out=out)
    for step in range(5):
        n.copy_(dev32([(9 * step + r) % 51 for r in range(rows)], dev))
        history.add_(1).remainder_(vocab)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ikv.adjust_logits(x, history=history, n_history=n, frequency=pen)), step
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ikv.adjust_logits(x, history=history, n_history=n, frequency=pen, stream=side)
    side.synchronize()
    assert torch.equal(got, out)


def test_refusals(dev):
    x = torch.zeros(2, 40, device=dev)
    tokens = dev32([[1], [2]], dev)
    for bad, error in ((dict(history=tokens.long()), TypeError), (dict(history=tokens[:1]), ValueError),
                       (dict(history=tokens[0]), ValueError), (dict(history=tokens, n_history=dev32([1], dev)), ValueError),
                       (dict(bias_tokens=tokens), ValueError),
                       (dict(bias_tokens=tokens, bias_values=torch.zeros(2, 2, device=dev)), ValueError),
                       (dict(masks=torch.zeros(1, 1, dtype=torch.int32, device=dev)), ValueError),
                       (dict(out=torch.zeros(2, 41, device=dev)), ValueError),
                       (dict(presence=torch.zeros(2)), ValueError)):
        with pytest.raises(error):
            ikv.adjust_logits(x, **bad)
    with pytest.raises(ValueError):
        ikv.adjust_logits(x[0])
