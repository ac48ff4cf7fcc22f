"""A token's log probability is one number: as a target, as an alternative of whatever place, in any lane that happens
to write it, and in a second call.  Rows of one part and of many."""

import math

import pytest
import torch

from llm_accelerator_amd.logprobs import token_logprobs

pytestmark = pytest.mark.gpu


def rows(n, vocab, dtype, dev):
    """Masked down to a few hundred tokens, here and there, and whole ones."""
    g = torch.Generator(device=dev).manual_seed(vocab)
    x = (3 * torch.randn(n, vocab, generator=g, device=dev)).to(dtype)
    for i in range(n // 2):
        keep = torch.randperm(vocab, generator=g, device=dev)[: 40 + 9 * i]
        masked = torch.full_like(x[i], -math.inf)
        masked[keep] = x[i, keep]
        x[i] = masked
    return x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [900, 4000, 9001, 40000, 151936, 300007])
def test_alternatives_have_the_targets_log_probability(dev, vocab, dtype):
    x = rows(40, vocab, dtype, dev)
    got = token_logprobs(x, top=32)
    for j in range(32):
        mine = token_logprobs(x, got.top_ids[:, j].contiguous())
        assert torch.equal(mine.logprob, got.top_logprobs[:, j]), j
        assert (mine.rank == j).all()


@pytest.mark.parametrize("vocab", [900, 9001, 151936])
def test_equal_logits_have_equal_log_probabilities(dev, vocab):
    """Runs of equal logits among others."""
    x = rows(24, vocab, torch.float32, dev)
    place = torch.rand(24, vocab, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).argsort(-1)[:, :20]
    x.scatter_(1, place, 15.0)
    got = token_logprobs(x, top=20)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :20]  # (a random logit may lie above the runs')
    assert torch.equal(got.top_ids, order.int())
    z = x.gather(1, order)
    alike = z[:, 1:] == z[:, :-1]
    assert alike.sum().item() > 24 * 15 and (got.top_logprobs[:, 1:] == got.top_logprobs[:, :-1])[alike].all()


@pytest.mark.parametrize("vocab", [9001, 151936, 300007])
def test_a_second_call_gives_the_same_bits(dev, vocab):
    x = rows(40, vocab, torch.float32, dev)
    t = torch.arange(40, device=dev, dtype=torch.int32) * 97
    first = token_logprobs(x, t, top=32)
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(token_logprobs(x, t, top=32), first))
