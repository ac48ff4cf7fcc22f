"""Microscaled tensors, products, scores and log probabilities as they are used together: the model's own head
quantised, its logits' log probabilities against the score without logits, alternatives of a prompt's tokens out
of the Q4 model's batched step; then captured into graphs, on other streams, by two callers at once."""

import numpy as np
import pytest
import torch

from llm_accelerator_amd.decode import BatchedDecoder
from llm_accelerator_amd.logprobs import token_logprobs
from llm_accelerator_amd.model import Qwen3Config, build_model, random_host_weights
from llm_accelerator_amd.mx import mx_linear, mx_quantize, mx_score

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def small(dev):
    cfg = Qwen3Config(num_hidden_layers=2, vocab_size=2048)
    host = random_host_weights(cfg, seed=3, num_layers=2)
    return cfg, build_model(cfg, host, max_ctx=32, device=dev)


def head_of(model):
    """The tied Q4 table's values, fp32."""
    q4 = model.lm_head.weight
    p = q4.packed
    lo, hi = (p & 15).to(torch.int8), (p >> 4).to(torch.int8)
    q = torch.stack((lo, hi), -1).flatten(1)
    q = torch.where(q >= 8, q - 16, q).float()
    return q * (q4.scale.float() / 16384).repeat_interleave(64, 1)


def test_alternatives_of_a_batched_step(dev, small):
    """Logits of BatchedDecoder.step: its own next token is the first alternative, rank 0."""
    cfg, model = small
    dec = BatchedDecoder(model, 5)
    tokens = torch.tensor([1, 7, 2047, 5, 900], dtype=torch.int32, device=dev)
    logits = torch.empty(5, cfg.vocab_size, device=dev)
    for pos in range(3):
        nxt, score = dec.step(tokens, torch.full((5,), pos, dtype=torch.int32, device=dev), logits)
        got = token_logprobs(logits, nxt, top=4)
        assert (got.rank == 0).all() and torch.equal(got.top_ids[:, 0], nxt)
        assert torch.equal(got.logprob, got.top_logprobs[:, 0])
        want = torch.log_softmax(logits.double(), -1)
        assert (got.logprob.double() - want.gather(1, nxt.long()[:, None])[:, 0]).abs().max().item() < 1e-4
        tokens = nxt.clone()


@pytest.mark.parametrize("m", [3, 30, 130])
def test_head_quantised_scored_and_ranked(dev, small, m):
    """A head in 4 bits: the score without logits is the logits' own, and the loss against the Q4 head is that of
    its values."""
    cfg, model = small
    table = head_of(model)
    head = mx_quantize(table, rule="ceil")
    rng = np.random.default_rng(m)
    hidden = torch.from_numpy(rng.standard_normal((m, cfg.hidden_size))).to(dev).to(torch.bfloat16)
    targets = torch.from_numpy(rng.integers(0, cfg.vocab_size, m)).to(dev).int()
    score = mx_score(hidden, head, targets)
    logits = mx_linear(hidden, head, out_dtype=torch.float32)
    lp = token_logprobs(logits, targets, top=8)
    exact = torch.log_softmax(hidden.double() @ head.dequantize().double().T, -1)
    size = (hidden.double().abs() @ head.dequantize().double().abs().T).amax()
    tol = (4 * cfg.hidden_size * 2.0 ** -23 * size + 2e-4).item()
    mine = exact.gather(1, targets.long()[:, None])[:, 0]
    assert (score.logprob - mine).abs().max().item() <= tol
    assert (lp.logprob - mine).abs().max().item() <= tol
    assert (score.best - lp.top_logprobs[:, 0]).abs().max().item() <= 2 * tol
    # the alternatives are the product's own order
    order = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :8].int()
    assert torch.equal(order, lp.top_ids)
    # blocks of 32 in 4 bits: e is the smallest with largest <= 6 2^e, so largest > 3 2^e; the widest step, from 4 to 6,
    # puts a value off by 2^e at most: a third of its block's largest
    err = (head.dequantize() - table).abs().view(-1, 32)
    assert (err <= table.abs().view(-1, 32).amax(-1, keepdim=True) / 3).all()


def all_calls(x, head, targets, logits):
    q = mx_quantize(x)
    y = mx_linear(q, head, out_dtype=torch.float32)
    z = mx_linear(x, head, out_dtype=torch.float32)
    s = mx_score(x, head, targets)
    t = token_logprobs(logits, targets, top=7)
    u = token_logprobs(z, targets, top=3)
    return [q.dequantize(), y, z, *s, *t, *u]


def inputs(rng, m, n, dev):
    x = torch.from_numpy(rng.standard_normal((m, 224))).to(dev).to(torch.float16)
    return x, torch.from_numpy(rng.integers(-2, n + 2, m)).to(dev).int(), torch.from_numpy(rng.standard_normal((m, 20001))).to(dev).float()


@pytest.mark.parametrize("m", [2, 90])
def test_captured_and_replayed(dev, m):
    """Every call in one graph, replayed over changing inputs with eager work of other sizes between the replays."""
    rng = np.random.default_rng(m)
    head = mx_quantize(torch.randn(1500, 224, device=dev))
    x, t, logits = inputs(rng, m, 1500, dev)
    all_calls(x, head, t, logits)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = all_calls(x, head, t, logits)
    for i in range(4):
        nx, nt, nl = inputs(rng, m, 1500, dev)
        if i == 2:
            nl[0] = float("-inf")
            nx[1, 3] = float("nan")
        x.copy_(nx)
        t.copy_(nt)
        logits.copy_(nl)
        g.replay()
        torch.cuda.synchronize()
        other = all_calls(*(lambda a, b, c: (a, head, b, c))(*inputs(rng, m + 3, 1500, dev)))  # eager work between
        want = all_calls(x, head, t, logits)
        for a, b in zip(out, want):
            assert torch.equal(a.nan_to_num(nan=7.0) if a.is_floating_point() else a, b.nan_to_num(nan=7.0) if b.is_floating_point() else b)
        del other


def test_two_graphs_side_by_side(dev):
    """Captured calls share no scratch: two graphs replayed on two streams at once."""
    rng = np.random.default_rng(1)
    head = mx_quantize(torch.randn(9000, 224, device=dev))
    made = []
    for m in (3, 70):
        x, t, logits = inputs(rng, m, 9000, dev)
        all_calls(x, head, t, logits)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = all_calls(x, head, t, logits)
        # (the graph reads x, t and logits where they are: they are kept)
        made.append((g, out, [v.clone() for v in all_calls(x, head, t, logits)], (x, t, logits)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(5):
        for s, (g, _, _, _) in zip(streams, made):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, out, want, _ in made:
        for a, b in zip(out, want):
            assert torch.equal(a.nan_to_num(nan=7.0) if a.is_floating_point() else a, b.nan_to_num(nan=7.0) if b.is_floating_point() else b)


def test_on_another_stream(dev):
    """Calls run on the current stream: after what it waits for, before what follows on it."""
    rng = np.random.default_rng(2)
    head = mx_quantize(torch.randn(3000, 224, device=dev))
    x, t, logits = inputs(rng, 40, 3000, dev)
    want = [v.clone() for v in all_calls(x, head, t, logits)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    late_x, late_l = torch.zeros_like(x), torch.zeros_like(logits)
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device=dev)
        for _ in range(20):
            big = big @ big * 1e-3  # keeps the stream busy
        late_x.copy_(x)
        late_l.copy_(logits)
        got = all_calls(late_x, head, t, late_l)
        kept = [v.clone() for v in got]
    s.synchronize()
    for a, b in zip(kept, want):
        assert torch.equal(a.nan_to_num(nan=7.0) if a.is_floating_point() else a, b.nan_to_num(nan=7.0) if b.is_floating_point() else b)


def test_two_streams_at_once(dev):
    rng = np.random.default_rng(4)
    head = mx_quantize(torch.randn(40000, 224, device=dev))
    jobs = []
    for m in (5, 33, 100):
        x, t, logits = inputs(rng, m, 40000, dev)
        jobs.append((x, t, logits, [v.clone() for v in all_calls(x, head, t, logits)], torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for x, t, logits, _, s in jobs:
            with torch.cuda.stream(s):
                outs.append(all_calls(x, head, t, logits))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        for a, b in zip(out, jobs[i % 3][3]):
            assert torch.equal(a.nan_to_num(nan=7.0) if a.is_floating_point() else a, b.nan_to_num(nan=7.0) if b.is_floating_point() else b)


def test_one_row_without_dims_and_targets_apart(dev):
    """hidden [cols] and logits [vocab] with a target of no dims; targets and logits that are slices; x of leading dims
    of which one is empty."""
    rng = np.random.default_rng(6)
    head = mx_quantize(torch.from_numpy(rng.standard_normal((900, 96))).to(dev).float())
    x = torch.from_numpy(rng.standard_normal((6, 96))).to(dev).to(torch.bfloat16)
    t = torch.from_numpy(rng.integers(0, 900, 12)).to(dev).int()
    whole = mx_score(x, head, t[::2])
    assert all(torch.equal(a, b) for a, b in zip(whole, mx_score(x, head, t[::2].contiguous())))
    one = mx_score(x[2], head, t[4])
    assert all(v.shape == () for v in one) and all(torch.equal(a, b[2]) for a, b in zip(one, mx_score(x[:3], head, t[:6:2])))
    logits = mx_linear(x, head, out_dtype=torch.float32)
    wide = torch.empty(6, 2000, device=dev)
    wide[:, 101:1001] = logits
    a, b = token_logprobs(wide[:, 101:1001], t[::2], top=3), token_logprobs(logits, t[::2].contiguous(), top=3)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    c = token_logprobs(wide[2, 101:1001], t[4], top=3)
    assert c.logprob.shape == c.rank.shape == c.entropy.shape == () and c.top_ids.shape == (3,)
    assert all(torch.equal(u, v[2]) for u, v in zip(c, b))
    assert mx_linear(x.view(2, 3, 96)[:, :0], head).shape == (2, 0, 900)
    assert mx_score(x.view(2, 3, 96)[:, :0], head, t.view(2, 6)[:, :0]).entropy.shape == (2, 0)
    empty = token_logprobs(logits.view(2, 3, 900)[:, :0], t.view(2, 6)[:, :0], top=2)
    assert empty.rank.shape == (2, 0) and empty.top_ids.shape == (2, 0, 2)


def test_a_tensor_times_itself(dev):
    rng = np.random.default_rng(7)
    a = mx_quantize(torch.from_numpy(rng.standard_normal((70, 160))).to(dev).float())
    v = a.dequantize().double()
    # 160 products, exact, and as many additions of half a step of sum |a a|; the output's rounding
    size = v.abs() @ v.abs().T
    assert ((mx_linear(a, a, out_dtype=torch.float32).double() - v @ v.T).abs() <= 161 * 2.0 ** -23 * size).all()
