"""Log probabilities of given tokens, entropies and likeliest tokens against 64-bit arithmetic on the CPU."""
import math

import pytest
import torch

import citlali_b200 as cb
from citlali_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def plain(x, tokens, top):
    x = x.double()
    x = torch.where(x.isfinite(), x, -math.inf)
    m = x.amax(-1, keepdim=True)
    some = m > -math.inf
    e = torch.exp(torch.where(some, x - m, -math.inf))
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    lp = torch.where(x > -math.inf, x - lse, -math.inf)
    p = torch.where(some, e / total, 0.0)
    entropy = -torch.where(p > 0, p * torch.where(p > 0, lp, 0.0), 0.0).sum(-1)
    value, index = torch.sort(x, dim=-1, descending=True, stable=True)
    value, index = value[:, :top], index[:, :top]
    ids = torch.where(value > -math.inf, index, -1)
    return lp, entropy, ids, torch.where(value > -math.inf, value - lse, -math.inf)


def check(x, tokens, top):
    rows, vocab = x.shape
    lp, entropy, ids, top_lp = plain(x, tokens, top)
    got = ops.token_logprobs(x.to(DEV), None if tokens is None else tokens.to(DEV), top)
    assert set(got) == {"entropy"} | ({"logprobs"} if tokens is not None else set()) | ({"top_ids", "top_logprobs"} if top else set())
    # a log probability is x - m - log S: one rounding of x - m and of the difference, S a sum of at most 16 + vocab / 256 / cluster terms
    # a thread (each off by 2^-21 through its exponent's rounding up to 24, less where the term is small) in a tree of 16 more levels
    spread = torch.where(x.double().isfinite(), x.double(), 0.0).abs().amax(-1)
    off = (vocab / 256 + 64) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * spread
    if tokens is not None:
        want = lp[torch.arange(rows), tokens.long()]
        have = got["logprobs"].cpu().double()
        assert torch.equal(have.isfinite(), want.isfinite())
        fine = want.isfinite()
        assert ((have - want).abs() <= off + 2.0 ** -22 * want.abs())[fine].all(), float((have - want)[fine].abs().max())
        assert (have[~fine] == want[~fine]).all()
    # the entropy is log S - T / S, T a sum of terms |u| e^u <= 1/e times S's
    have = got["entropy"].cpu().double()
    assert ((have - entropy).abs() <= 2 * off * (1 + entropy)).all(), float((have - entropy).abs().max())
    if top:
        assert torch.equal(got["top_ids"].cpu().long(), ids)
        have = got["top_logprobs"].cpu().double()
        assert torch.equal(have.isfinite(), top_lp.isfinite())
        fine = top_lp.isfinite()
        assert ((have - top_lp).abs() <= off[:, None] + 2.0 ** -22 * top_lp.abs())[fine].all()


@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 1, 0), (3, 5, 5), (2, 31, 31), (5, 33, 32), (1, 4096, 20), (7, 4097, 3), (2, 50257, 5),
                                            (9, 8191, 32), (3, 151936, 20), (700, 1001, 7), (1, 300001, 32), (4, 12289, 1),
                                            (3, 520, 32), (2, 700, 5), (3, 1500, 32), (4, 2047, 20), (2, 4100, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_against_64_bits(rows, vocab, top, dtype):
    g = torch.Generator().manual_seed(rows * 31 + vocab)
    x = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g).to(torch.int32)
    check(x, tokens, top)
    check(x, None, top)
    check(x, tokens, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_index(dtype):
    g = torch.Generator().manual_seed(2)
    x = torch.randint(-3, 4, (5, 20011), generator=g).to(dtype)
    check(x, torch.arange(5, dtype=torch.int32), 32)
    check(torch.full((2, 9000), 1.5).to(dtype), torch.tensor([0, 8999], dtype=torch.int32), 20)
    check(torch.arange(30000, dtype=torch.float32)[None].to(dtype), torch.tensor([29999], dtype=torch.int32), 32)      # rising all the way
    check(-torch.arange(30000, dtype=torch.float32)[None].to(dtype) / 100, torch.tensor([3], dtype=torch.int32), 32)


def test_masked_entries_and_numbers_that_are_none():
    g = torch.Generator().manual_seed(3)
    for vocab in (40, 151936):
        x = 4 * torch.randn(8, vocab, generator=g)
        x[0, ::2] = -math.inf                               # a grammar's mask
        x[1] = -math.inf
        x[1, 17] = -4.0                                     # one token left
        x[2] = -math.inf                                    # none left
        x[3, 5], x[3, 6], x[3, 7] = math.inf, math.nan, -math.nan
        x[4] = math.nan
        x[5, 3:] = torch.finfo(torch.float32).min           # masked by the type's lowest number
        x[6] = torch.finfo(torch.float32).min               # all of them: all alike
        x[7, 0] = torch.finfo(torch.float32).max
        check(x, torch.tensor([1, 17, 0, 6, 2, 2, 39, 0], dtype=torch.int32), 20)
        check(x, torch.tensor([2, 16, 5, 5, 2, 30, 0, 9], dtype=torch.int32), 32)


def test_rows_that_differ_by_a_constant_and_large_logits():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 5000, generator=g).round(decimals=2)
    check(x + torch.tensor([[0.0], [1e4], [-1e4]]), torch.tensor([1, 2, 3], dtype=torch.int32), 5)
    check(x * 1e5, torch.tensor([1, 2, 3], dtype=torch.int32), 5)


def test_tokens_outside_the_vocabulary_and_rows_left_alone():
    x = torch.randn(4, 100, generator=torch.Generator().manual_seed(5)).to(DEV)
    got = ops.token_logprobs(x, torch.tensor([-1, 100, 3, 1 << 30], dtype=torch.int32, device=DEV))["logprobs"].cpu()
    assert got[[0, 1, 3]].isnan().all() and got[2].isfinite()
    empty = ops.token_logprobs(x[:0], torch.zeros(0, dtype=torch.int32, device=DEV), 3)
    assert empty["logprobs"].shape == (0,) and empty["top_ids"].shape == (0, 3)


def test_captured_and_on_another_stream():
    g = torch.Generator().manual_seed(6)
    x = torch.randn(3, 40000, generator=g).to(DEV)
    t = torch.tensor([4, 5, 6], dtype=torch.int32, device=DEV)
    want = ops.token_logprobs(x, t, 4)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = ops.token_logprobs(x, t, 4)
    graph.replay()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = ops.token_logprobs(x, t, 4)
    torch.cuda.synchronize()
    for k in want:
        assert torch.equal(want[k], got[k]) and torch.equal(want[k], other[k])


def test_refusals():
    x = torch.zeros(2, 50, device=DEV)
    t = torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad, words in [(lambda: ops.token_logprobs(x, t, 33), "at most 32"), (lambda: ops.token_logprobs(x, t, -1), "at most 32"),
                       (lambda: ops.token_logprobs(x[:, :4].contiguous(), t, 5), "at most 32"),
                       (lambda: ops.token_logprobs(x, t.long()), "int32"), (lambda: ops.token_logprobs(x, t[:1]), "one a row"),
                       (lambda: ops.token_logprobs(x[0]), "rows"), (lambda: ops.token_logprobs(x[:, ::2]), "contiguous"),
                       (lambda: ops.token_logprobs(x.half(), t), "float32 or bfloat16"), (lambda: ops.token_logprobs(x.cpu()), "CUDA")]:
        with pytest.raises(cb.CitlaliError, match=words):
            bad()
    with pytest.raises(TypeError):
        ops.token_logprobs(x, t, 1.5)
