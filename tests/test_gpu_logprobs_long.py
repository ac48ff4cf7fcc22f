"""token_logprobs where a thread holds 64 logits: vocabularies past 262144, and prompts (many rows of middling
vocabularies), of one part and of several, in the three types.  Bounds and reference: see test_gpu_logprobs."""

import math

import pytest
import torch

from llm_accelerator_amd import _lib
from llm_accelerator_amd.logprobs import MAX_VOCAB, token_logprobs

TYPES = [torch.float32, torch.float16, torch.bfloat16]
LONG = [(262145, 32), (300007, 20), (MAX_VOCAB, 32)]
MANY = [(1400, 16390, 20), (2100, 4100, 32), (2060, 16384, 5), (1030, 20000, 1), (700, 33000, 32)]


def slots(rows, vocab):
    """Parts of all rows: without alternatives a part leaves 12 bytes and 4, each aligned to 256."""
    n = _lib.load().q4d_token_logprobs_workspace_bytes(rows, vocab, 0)
    return next(c for c in range(n // 16 + 1, 0, -1) if -(-(-(-12 * c // 256) * 256 + 4 * c) // 256) * 256 == n)


def test_sizes_take_parts_of_16384():
    """(So that the tests below are of the kernel that they stand for.)"""
    for rows, vocab in [(1, v) for v, _ in LONG] + [(r, v) for r, v, _ in MANY]:
        have, want = slots(rows, vocab), rows * -(-vocab // 16384)
        assert want <= have <= want + 63 and have < rows * -(-vocab // 4096), (rows, vocab)


def special(vocab, dtype, dev):
    """Rows that are hard for the choice of the best, and a random one."""
    g = torch.Generator(device=dev).manual_seed(vocab)
    at = torch.arange(vocab, device=dev)
    low, inf, nan = torch.finfo(dtype).min, math.inf, math.nan

    def rand():
        return (3 * torch.randn(vocab, generator=g, device=dev)).to(dtype).float()

    def left(n, side=False):
        r = rand()
        keep = at[:n] + vocab // 3 if side else torch.randperm(vocab, generator=g, device=dev)[:n]
        out = torch.full_like(r, -inf)
        out[keep] = r[keep]
        return out

    def where(cond, value, other=None):
        return torch.where(cond, value, rand() if other is None else other)
    rows = [
        torch.zeros(vocab, device=dev), (at % 2).float(), where(at % 2 == 0, -0.0, torch.zeros(vocab, device=dev)),
        (at / vocab).round(decimals=2), -(at / vocab).round(decimals=2), at * (50.0 / vocab), -at * (50.0 / vocab),  # equal, ordered
        torch.full((vocab,), -inf, device=dev), left(1), left(2), left(19), left(33), left(150), left(1000), left(1000, True),
        left(70, True), where(at < vocab // 2, -inf), where(at >= vocab // 2, low), torch.full((vocab,), low, device=dev),
        where(at >= 3, -inf), where(at < vocab - 4, -inf),                                                           # masked
        where(at % 256 == 17, 20.0 + at * (8.0 / vocab)), where(at % 2048 < 8, 21.0), where(at % 2048 < 8, 20.0 + (at % 64) / 8.0),
        where(at % 1024 < 4, 20.0 + (at % 61) / 8.0), where(at % 1024 // 8 == 3, 9.0), where(at // 512 % 4 == 1, 9.0 + (at % 7) / 4.0),
        where(at // 16384 == 1, 15.0 + (at % 97) / 16.0),                                                            # side by side
        where(at == vocab - 1, inf), where(at == 7, nan), where(at % 3 == 0, nan), torch.full((vocab,), nan, device=dev),
        where(at >= 9, -inf, where(at % 2 == 0, nan)), where(at < 80, nan, where(at >= vocab - 5, 1.0, torch.full((vocab,), -inf, device=dev))),
        where(at >= 100, nan, torch.full((vocab,), -inf, device=dev)), rand(), rand().round(),
    ]
    return torch.stack(rows).to(dtype)


def spread_targets(rows, vocab, dev):
    t = (torch.arange(rows, device=dev) * 7919 + 5) % vocab
    t[::5] = vocab - 1
    t[1::7] = 0
    t[3], t[4] = -1, vocab
    return t.int()


def within(got, x, t, top):
    """Results at hand against the reference, by the bounds of test_gpu_logprobs.check."""
    from test_gpu_logprobs import close, reference
    logprob, rank, entropy, top_logprobs, top_ids = got
    want = reference(x, t, top)
    h = torch.nan_to_num(want["entropy"])
    lse = (h + 434) * 2.0 ** -23
    logl = -torch.nan_to_num(torch.log_softmax(x.double().cpu(), -1).amax(-1))
    assert torch.equal(top_ids.cpu(), want["top_ids"]) and torch.equal(rank.cpu(), want["rank"])
    close(logprob, want["logprob"], lse)
    close(top_logprobs, want["top_logprobs"], lse[:, None])
    close(entropy, want["entropy"], lse + 2 * lse * (h + logl + 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,top", LONG)
def test_long_vocabularies(dev, vocab, top, dtype):
    from test_gpu_logprobs import check
    x = special(vocab, dtype, dev)
    check(x, spread_targets(len(x), vocab, dev), top)
    # the same rows, neither aligned nor an even number of elements apart
    wide = torch.full((len(x), vocab + 4), math.inf, device=dev, dtype=dtype)[:, : vocab + 3]
    wide[:, 1:vocab + 1] = x
    got = token_logprobs(wide[:, 1:vocab + 1], spread_targets(len(x), vocab, dev), top=top)
    want = token_logprobs(x, spread_targets(len(x), vocab, dev), top=top)
    for a, b in zip(got, want):
        assert torch.equal(torch.nan_to_num(a.float(), nan=7e30), torch.nan_to_num(b.float(), nan=7e30))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", MANY)
def test_prompts(dev, rows, vocab, top, dtype):
    """Hard rows among many, in rows padded to another length."""
    wide = torch.full((rows, vocab + 9), math.inf, device=dev, dtype=dtype)
    x = wide[:, 3:vocab + 3]
    g = torch.Generator(device=dev).manual_seed(rows)
    x.copy_(3 * torch.randn(rows, vocab, generator=g, device=dev))
    hard = special(vocab, dtype, dev)
    place = (torch.arange(len(hard), device=dev) * 17 + 5) % rows
    x[place] = hard
    x[rows - 1] = hard[14]
    t = spread_targets(rows, vocab, dev)
    got = token_logprobs(x, t, top=top)
    # (the reference sorts: the hard rows, their neighbours and some others)
    pick = torch.unique(torch.cat([place, (place + 1) % rows, torch.arange(0, rows, 97, device=dev), torch.tensor([rows - 1], device=dev)]))
    within([a[pick] for a in got], x[pick], t[pick], top)
