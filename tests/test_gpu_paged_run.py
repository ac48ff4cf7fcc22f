"""The paged operators as a server uses them together: chunks of prompts beside decode steps, forks of a
common beginning, proposed tokens that are taken back, sequences that end, compaction, steps that
find no page, and a captured step replayed over all of it."""

import math
import random

import pytest
import torch

import paged_ref
from llm_accelerator_amd import _lib, common
from llm_accelerator_amd.model import KVCache, Qwen3Config
from llm_accelerator_amd.paged import PagedKVCache, RaggedBatch, RopeTable

pytestmark = pytest.mark.gpu
F, B = torch.float16, torch.bfloat16
LAYERS, D, EPS = 2, 64, 1e-6


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


class History:
    """What every sequence's positions were given, by position: projection rows and layer."""

    def __init__(self):
        self.rows = {}

    def fork(self, src, dst):
        self.rows[dst] = list(self.rows[src])


def step(cache, batch, x, qh, rope, gq, gk, ws=None):
    """A step of a model of LAYERS layers: x [layers, tokens, qh + 2 kvh, D]; outputs [layers, tokens, qh, D]."""
    kvh = cache.num_kv_heads
    cache.reserve(batch)
    out = []
    for layer in range(LAYERS):
        q = cache.append(layer, batch, x[layer, :, :qh], x[layer, :, qh:qh + kvh], x[layer, :, qh + kvh:], rope, gq, gk, EPS)
        out.append(cache.attention(layer, batch, q, ws=ws))
    return torch.stack(out)


def expect(rows, new, qh, kvh, rope, gq, gk, dtype):
    """64-bit outputs [layers, new, qh, D] of a sequence's last `new` positions, and their bound, from the
    projection rows alone.

    q and k are off by half a step of the cache's type (and 2^-18 of fp32 arithmetic) relative to the
    largest of a row at most, so a score by D^-1/2 times sum |q| |k| times twice that; a score off by d
    changes a probability by e^(2 d) at most."""
    x = torch.stack(rows, 1).double()                                   # [layers, T, heads, D]
    t = x.shape[1]
    cos, sin = rope.cos[:t], rope.sin[:t]
    half = torch.finfo(dtype).eps / 2
    outs, bounds = [], []
    for layer in range(LAYERS):
        q = paged_ref.turn(x[layer, -new:, :qh], gq, EPS, cos[-new:], sin[-new:], rope.interleaved)
        k = paged_ref.turn(x[layer, :, qh:qh + kvh], gk, EPS, cos, sin, rope.interleaved).repeat_interleave(qh // kvh, 1)
        v = x[layer, :, qh + kvh:].repeat_interleave(qh // kvh, 1)
        z = torch.stack([q[:, h] @ k[:, h].T for h in range(qh)]) * D ** -0.5             # [qh, new, T]
        hidden = torch.arange(t, device=x.device)[None] > torch.arange(t - new, t, device=x.device)[:, None]
        p = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
        out = torch.stack([p[h] @ v[:, h] for h in range(qh)], 1)
        size = torch.stack([p[h] @ v[:, h].abs() for h in range(qh)], 1)
        most = v.abs().amax(0)[None]
        norms = (q.norm(dim=-1).amax() * k.norm(dim=-1).amax()).item()
        # row maxima are at most norms, so an error relative to them is at most sqrt(D) times one relative
        # to the elements' own size: only the fp32 part is of that kind
        off = D ** -0.5 * norms * 2 * (half + 2.0 ** -18 * D ** 0.5)
        bound = paged_ref.attend_bound(out, size, most * p.amax(-1).T[..., None], dtype)
        outs.append(out)
        bounds.append(bound * (1 + 2 * off) + size * (2 * (math.exp(2 * off) - 1) + half))
    return torch.stack(outs), torch.stack(bounds)


def check(out, batch, seqs, counts, history, qh, kvh, rope, gq, gk, dtype):
    at = 0
    for s, c in zip(seqs, counts):
        if c:
            want, bound = expect(history.rows[s], c, qh, kvh, rope, gq, gk, dtype)
            err = (out[:, at:at + c].double() - want).abs()
            assert bool((err <= bound).all()), (s, c, float((err / bound).max()))
        at += c


@pytest.mark.parametrize("seed,dtype,qh,kvh,ps,inter", [(0, F, 4, 2, 16, False), (1, B, 6, 1, 32, False),
                                                       (2, F, 3, 3, 64, True), (3, B, 10, 2, 16, True),
                                                       (6, F, 8, 1, 16, False), (16, B, 4, 4, 32, True)])
def test_a_server(dev, seed, dtype, qh, kvh, ps, inter):
    """(Seeds 2, 6 and 16 come to steps that find no page.)"""
    rng = random.Random(seed)
    rows_of_table, pages = 10, 640 // ps
    cache = PagedKVCache(LAYERS, pages, ps, kvh, D, rows_of_table, 400, dtype, dev)
    rope = RopeTable.build(D, 400, 1e4, {"type": "yarn", "factor": 4, "original_max_ctx": 100} if inter else None, inter, dev)
    g = torch.Generator(device=dev).manual_seed(seed)
    gq, gk = (1 + 0.1 * torch.randn(D, generator=g, device=dev) for _ in range(2))
    history, model = History(), paged_ref.Pages(pages, ps, rows_of_table, cache.max_pages)
    live, refused = [], 0
    for turn in range(25):
        print(f"[server] seed={seed} turn={turn} live={live}", flush=True)
        idle = [s for s in range(rows_of_table) if s not in live]
        act = rng.choice(("new", "new", "fork", "end", "compact", "step", "step"))
        if act == "fork" and live and idle:
            src, dst = rng.choice(live), idle[0]
            cache.fork(i32([src], dev), i32([dst], dev))
            model.fork([src], [dst])
            history.fork(src, dst)
            live.append(dst)
        elif act == "end" and len(live) > 2:
            s = live.pop(rng.randrange(len(live)))
            cache.free(i32([s], dev))
            model.truncate([s])
        elif act == "compact":
            assert int(cache.compact().item()) == model.compact()
        counts = {s: rng.choice((1, 1, 1, 4, 0)) for s in live}
        if act == "new" and idle:
            live.append(idle[0])
            history.rows[idle[0]] = []
            counts[idle[0]] = rng.choice((1, 17, 60, 130))
        if not counts:
            continue
        seqs = list(counts)
        rng.shuffle(seqs)
        new = [counts[s] for s in seqs]
        pad = rng.choice((0, 3))
        batch = RaggedBatch.of(seqs, new, dev, tokens=max(1, sum(new) + pad))
        x = torch.randn(LAYERS, batch.tokens, qh + 2 * kvh, D, generator=g, device=dev)
        data = cache.data.clone()
        out = step(cache, batch, x, qh, rope, gq, gk)
        model.reserve(seqs, new)
        if model.status:
            # the step found no page: nothing has changed, and it can be had again when there are some
            assert model.status & _lib.STATUS_NOT_RESERVED
            assert torch.equal(cache.data, data) and cache.lengths.tolist() == model.lengths
            with pytest.raises(_lib.Q4DecError):
                cache.raise_for_status("step")
            model.status, refused = 0, refused + 1
            for s in [s for s in live if not history.rows[s]] + live[:2]:
                if s in live:
                    live.remove(s)
                    cache.free(i32([s], dev))
                    model.truncate([s])
            continue
        at = 0
        for s, c in zip(seqs, new):
            history.rows[s] += [x[:, at + i] for i in range(c)]
            at += c
        check(out, batch, seqs, new, history, qh, kvh, rope, gq, gk, dtype)
        assert cache.table.tolist() == model.table and cache.refs.tolist() == model.refs
        back = [s for s in seqs if counts[s] == 4]       # proposed tokens: some are taken back
        if back:
            keep = [len(history.rows[s]) - rng.randrange(4) for s in back]
            cache.truncate(i32(back, dev), i32(keep, dev))
            model.truncate(back, keep)
            for s, n in zip(back, keep):
                del history.rows[s][n:]
        assert cache.lengths.tolist() == model.lengths and cache.status() == model.status == 0
    assert refused or seed not in (2, 6, 16)


def test_a_captured_step(dev):
    """reserve, appends and attention of two layers as one graph, replayed on changing sequences and counts
    with eager work of another workspace between, against an eager cache; then replays that find no page."""
    qh, kvh, ps = 4, 2, 16
    caches = [PagedKVCache(LAYERS, 14, ps, kvh, D, 6, 160, F, dev) for _ in range(2)]
    rope = RopeTable.build(D, 160, 1e4, device=dev)
    batch = RaggedBatch.of([0, 1, 2], [40, 1, 7], dev, tokens=48)
    x = torch.zeros(LAYERS, 48, qh + 2 * kvh, D, device=dev)
    ws = caches[0].workspace(qh, batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        out = step(caches[0], batch, x, qh, rope, None, None, ws)
    torch.cuda.current_stream().wait_stream(side)
    for seqs, counts in (([0, 1, 2], [40, 1, 7]), ([5, 0, 3], [17, 1, 30]), ([2, 5, 0], [0, 0, 1]), ([4, 1, 3], [33, 15, 0]),
                         ([0, 1, 2], [1, 1, 1])):
        x.normal_()
        starts = [sum(counts[:i]) for i in range(4)]
        batch.seqs.copy_(i32(seqs, dev))
        batch.starts.copy_(i32(starts, dev))
        g.replay()
        want = step(caches[1], batch, x, qh, rope, None, None)
        assert torch.equal(out[:, :starts[3]], want[:, :starts[3]])
        assert torch.equal(caches[0].data, caches[1].data) and torch.equal(caches[0].table, caches[1].table)
        assert caches[0].status() == 0
    # three replays ahead of the host: the second finds no page (1 of 14 is free, it wants 3), the third
    # would fit but is held back
    good = caches[0].lengths.tolist()
    batch.seqs.copy_(i32([2, 1, 3], dev))
    states = []
    for counts in ([1, 1, 1], [40, 0, 0], [1, 0, 0]):
        batch.starts.copy_(i32([sum(counts[:i]) for i in range(4)], dev))
        g.replay()
        states.append((caches[0].data.clone(), caches[0].lengths.clone(), caches[0].table.clone(), caches[0].refs.clone()))
    for s, n in ((2, 1), (1, 1), (3, 1)):
        good[s] += n
    assert caches[0].lengths.tolist() == good
    assert all(torch.equal(a, b) for i in (1, 2) for a, b in zip(states[0], states[i]))
    # (the attention of the second finds fewer positions than new tokens)
    assert caches[0].status() == _lib.STATUS_NO_PAGES | _lib.STATUS_NOT_RESERVED | _lib.STATUS_BAD_SEQUENCE
    with pytest.raises(_lib.Q4DecError):
        caches[0].raise_for_status("replays")
    g.replay()
    good[2] += 1
    assert caches[0].lengths.tolist() == good and caches[0].status() == 0


def test_pages_give_what_one_tensor_gives(dev):
    """One sequence, token by token, through the contiguous cache's functions and through pages."""
    heads, kvh, d, t = 16, 8, 128, 70
    x = torch.randn(t, heads + 2 * kvh, d, device=dev)
    rope = RopeTable.build(d, 128, 1e6, device=dev)
    paged = PagedKVCache(1, 8, 16, kvh, d, 2, 128, F, dev)
    flat = KVCache(Qwen3Config(num_key_value_heads=kvh, head_dim=d), 1, 1, 128, dev)
    batch = RaggedBatch.of([1], [1], dev)
    kview, vview = common.layer_views(flat, 0)
    kview, vview = kview[0], vview[0]
    for i in range(t):
        paged.reserve(batch)
        row = x[i:i + 1]
        q = paged.append(0, batch, row[:, :heads], row[:, heads:heads + kvh], row[:, heads + kvh:], rope)
        got = paged.attention(0, batch, q)
        c, s = (torch.cat([a[i], a[i]]).view(1, 1, d) for a in (rope.cos, rope.sin))
        qr, kr = common.manual_apply_rope(row[:, :heads].transpose(0, 1)[None].contiguous(),
                                          row[:, heads:heads + kvh].transpose(0, 1)[None].contiguous(), c, s)
        kview = common.append_cache(kview, kr)
        vview = common.append_cache(vview, row[:, heads + kvh:].transpose(0, 1)[None].contiguous())
        want, _ = common.manual_cached_attention(qr, common.manual_repeat_kv(kview, heads // kvh),
                                                 common.manual_repeat_kv(vview, heads // kvh), d ** -0.5)
        # both keep k and v in fp16; the paged q, probabilities and output are fp16 too, the other's fp32:
        # half a step each, of q in a score of up to |q| |k| D^-1/2
        off = d ** -0.5 * float((qr.norm(dim=-1).amax() * kr.norm(dim=-1).amax()).item()) * 3 * 2.0 ** -11
        most = float(x[:i + 1, heads + kvh:].abs().max())
        err = (got.view(1, heads, 1, d).float() - want).abs().max().item()
        assert err <= most * (2 * (math.exp(2 * off) - 1) + 3 * 2.0 ** -11), i
