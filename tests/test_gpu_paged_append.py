"""Append into pages against 64 bits: types, layouts, head widths, parts of a head rotated, packed
inputs, padding, and what cannot be."""

import pytest
import torch

import paged_ref
from llm_accelerator_amd import _lib
from llm_accelerator_amd.paged import PagedKVCache, RaggedBatch, RopeTable

pytestmark = pytest.mark.gpu


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def setup(dev, lengths, counts, kvh, d, ps, dtype, rows=None):
    need = [-(-n // ps) for n in lengths]
    cache = PagedKVCache(2, sum(need) + 3, ps, kvh, d, rows or len(lengths), max(lengths) + ps, dtype, dev)
    cache.data.fill_(7.0)
    g = torch.Generator().manual_seed(sum(lengths) + ps)
    order = torch.randperm(sum(need) + 3, generator=g)
    at = 0
    for s, n in enumerate(need):
        cache.table[s, :n] = order[at:at + n].to(torch.int32)
        at += n
    cache.lengths[:len(lengths)] = i32(lengths, dev)
    return cache


CASES = [  # kv heads, q heads, dim, page, cache type, input type, rotated dims, interleaved, norm
    (8, 16, 128, 64, torch.float16, torch.float32, 128, False, True),
    (8, 16, 128, 16, torch.bfloat16, torch.bfloat16, 64, True, False),
    (2, 14, 64, 32, torch.float16, torch.float16, 64, False, False),
    (1, 3, 64, 128, torch.bfloat16, torch.float32, 16, False, True),
    (3, 3, 128, 256, torch.float16, torch.bfloat16, 96, False, True),
    (1, 1, 128, 16, torch.float16, torch.float32, 112, True, True),
    (2, 4, 64, 16, torch.bfloat16, torch.float16, 48, True, True),
    (4, 4, 128, 64, torch.float16, torch.float16, 0, False, True),
    (4, 32, 128, 64, torch.bfloat16, torch.bfloat16, 0, False, False),
]


@pytest.mark.parametrize("kvh,qh,d,ps,dtype,xt,rot,inter,norm", CASES)
def test_append_vs_fp64(dev, kvh, qh, d, ps, dtype, xt, rot, inter, norm):
    lengths, counts = [1, 70, 16, 300, 65, 129], [1, 5, 16, 1, 0, 129]
    seqs = [3, 0, 5, 1, 2, 4]
    print(f"[append] {kvh}/{qh} d={d} ps={ps} {dtype} {xt} rot={rot} inter={inter} norm={norm}", flush=True)
    cache = setup(dev, lengths, counts, kvh, d, ps, dtype)
    counts = [counts[s] for s in seqs]
    pad = 3
    t = sum(counts) + pad
    batch = RaggedBatch.of(seqs, counts, dev, tokens=t)
    g = torch.Generator(device=dev).manual_seed(kvh * qh + d)
    x = torch.randn(t, qh + 2 * kvh, d, generator=g, device=dev).to(xt)
    x[sum(counts):] = float("nan")                      # padding is not read
    q, k, v = x[:, :qh], x[:, qh:qh + kvh], x[:, qh + kvh:]
    gq, gk = ((1 + 0.1 * torch.randn(d, generator=g, device=dev) for _ in range(2)) if norm else (None, None))
    rope = RopeTable.build(rot, 301, 1e4, {"type": "yarn", "factor": 2, "original_max_ctx": 64}, inter, dev) if rot else None
    out = torch.full((t, qh, d), 5.0, dtype=dtype, device=dev)
    got = cache.append(1, batch, q, k, v, rope, gq, gk, 1e-6, out)
    assert got is out and cache.status() == 0
    assert bool((out[sum(counts):] == 5.0).all())
    want = torch.full_like(cache.data, 7.0).double()
    pos, row = [], []
    for s, c in zip(seqs, counts):
        pos += range(lengths[s] - c, lengths[s])
        row += [s] * c
    pos, row = torch.tensor(pos, device=dev), torch.tensor(row, device=dev)
    n = len(pos)
    cos, sin = (rope.cos[pos], rope.sin[pos]) if rot else (None, None)
    page, off = cache.table[row, pos // ps].long(), pos % ps
    want[1, 0, page, :, off] = paged_ref.turn(k[:n], gk, 1e-6, cos, sin, inter)
    want[1, 1, page, :, off] = v[:n].double()
    ref = paged_ref.turn(q[:n], gq, 1e-6, cos, sin, inter)
    half = torch.finfo(dtype).eps / 2
    # one rounding to the cache's type; fp32 norm (a sum of up to 128 squares, a square root, a division,
    # two products: under 2^-19) and two products of the rotation of values up to the row's largest
    for name, a, b in (("q", out[:n], ref), ("data", cache.data, want)):
        # subnormal results of fp16 are off by up to 2^-25
        bound = half * b.abs() + 2.0 ** -19 * b.abs().amax(-1, keepdim=True) + 2.0 ** -25
        assert bool(((a.double() - b).abs() <= bound).all()), (name, float((a.double() - b).abs().max()))
    assert torch.equal(cache.data[0], torch.full_like(cache.data[0], 7.0))
    assert torch.equal(cache.data[1][want[1] == 7.0], torch.full_like(cache.data[1], 7.0)[want[1] == 7.0])


def test_append_without_q_and_contiguous_copies(dev):
    """Rows that cannot be read in place (a transposed view, a row stride of 4 bytes more) are copied."""
    cache = setup(dev, [40, 9], [3, 2], 2, 64, 16, torch.float16)
    batch = RaggedBatch.of([0, 1], [3, 2], dev)
    k = torch.randn(5, 2, 64, device=dev)
    v = torch.randn(2, 5, 64, device=dev).transpose(0, 1)
    odd = torch.empty(5, 129, device=dev)[:, :128].view(5, 2, 64)
    odd.copy_(k)
    assert cache.append(0, batch, None, odd, v) is None
    first = cache.data.clone()
    cache.data.fill_(7.0)
    cache.append(0, batch, None, k, v.contiguous())
    assert torch.equal(cache.data, first)
    pages = cache.table[[0, 0, 0, 1, 1], [2, 2, 2, 0, 0]].long()
    assert torch.equal(cache.data[0, 1, pages, :, [5, 6, 7, 7, 8]], v.half())


def test_append_leaves_out_what_cannot_be(dev):
    def run(change, tokens=6, max_new=4, seqs=(0, 1, 2), starts=(0, 2, 5, 6)):
        cache = setup(dev, [20, 33, 7], [2, 3, 1], 2, 64, 16, torch.float16)
        change(cache)
        before = cache.data.clone()
        batch = RaggedBatch(i32(list(seqs), dev), i32(list(starts), dev), tokens, max_new)
        x = torch.ones(tokens, 2, 64, device=dev)
        out = cache.append(0, batch, x, x, x, RopeTable.build(64, 25, device=dev),
                           q_out=torch.full((tokens, 2, 64), 5.0, dtype=torch.float16, device=dev))
        left = [i for i in range(tokens) if bool((out[i] == 5.0).all())]
        changed = int((cache.data != before).any(-1).any(3).any(1).sum().item())   # (layer, page, row) with a new value
        return cache.status(), left, changed

    table = lambda c, s, k, p: c.table.__setitem__((s, k), p)  # noqa: E731
    B, P, S = _lib.STATUS_BAD_POSITION, _lib.STATUS_BAD_PAGE, _lib.STATUS_BAD_SEQUENCE
    nothing = lambda c: None  # noqa: E731
    # sequence 1 is past the rotation's 25 positions
    assert run(nothing) == (B, [2, 3, 4], 3)
    for page in (-1, 2 ** 31 - 1, -2 ** 31, 1000):
        assert run(lambda c: table(c, 0, 1, page)) == (B | P, [2, 3, 4], 1)   # q rows are written all the same
    assert run(nothing, seqs=(0, 1, 3)) == (B | S, [2, 3, 4, 5], 2)
    assert run(nothing, seqs=(-1, 1, 2)) == (B | S, [0, 1, 2, 3, 4], 1)
    assert run(nothing, max_new=1) == (S, [0, 1, 2, 3, 4], 1)
    assert run(lambda c: c.lengths.__setitem__(0, 1)) == (B | S, [0, 1, 2, 3, 4], 1)
    assert run(lambda c: c.lengths.__setitem__(2, 2 ** 30)) == (B | S, [2, 3, 4, 5], 2)
    assert run(nothing, starts=(0, 0, 0, 1)) == (0, [1, 2, 3, 4, 5], 1)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 200, 4096])
def test_many_sequences(dev, n):
    """The token's sequence is found among up to 4096, sequences without tokens among them."""
    counts = [(i * 7 + 1) % 3 for i in range(n)]
    cache = setup(dev, [3] * n, counts, 1, 64, 16, torch.float16)
    batch = RaggedBatch.of(list(range(n)), counts, dev)
    x = torch.arange(batch.tokens, device=dev, dtype=torch.float32).remainder(2048).view(-1, 1, 1).expand(-1, 1, 64).contiguous()
    cache.append(0, batch, None, x, x)
    assert cache.status() == 0
    tok = 0
    got = cache.data[0, 0, cache.table[:n, 0].long(), 0, :3, 0].cpu()
    for b, c in enumerate(counts):
        want = [7.0] * (3 - c) + [float((tok + i) % 2048) for i in range(c)]
        assert got[b].tolist() == want, b
        tok += c


def test_append_on_a_stream_and_in_a_graph(dev):
    cache = setup(dev, [28, 12], [2, 2], 2, 128, 32, torch.bfloat16)
    batch = RaggedBatch.of([1, 0], [2, 2], dev)
    x = torch.randn(4, 2, 128, device=dev)
    rope = RopeTable.build(128, 64, device=dev)
    want = cache.append(0, batch, x, x, -x, rope).clone()
    data = cache.data.clone()
    side = torch.cuda.Stream()
    cache.data.fill_(7.0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.append(0, batch, x, x, -x, rope)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(cache.data, data)
    out = torch.zeros_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        cache.append(0, batch, x, x, -x, rope, q_out=out)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(3):
        x.normal_()
        cache.lengths.add_(1)
        g.replay()
        replayed, data = out.clone(), cache.data.clone()
        out.zero_()
        cache.append(0, batch, x, x, -x, rope, q_out=out)
        assert torch.equal(out, replayed) and torch.equal(cache.data, data) and cache.status() == 0


@pytest.mark.parametrize("tokens,qh,kvh,d", [(2100, 14, 5, 64), (4500, 3, 2, 128), (11000, 14, 5, 64), (5000, 20, 3, 128)])
def test_many_tokens_as_few(dev, tokens, qh, kvh, d):
    """A wave takes one, two or four groups of head rows by how many there are: a token's values are those
    that it has in a small batch, bit for bit."""
    cache = setup(dev, [tokens], [tokens], kvh, d, 64, torch.float16)
    x = torch.randn(tokens, qh + 2 * kvh, d, device=dev)
    rope = RopeTable.build(d, tokens, device=dev)
    gamma = 1 + 0.1 * torch.randn(d, device=dev)
    split = lambda y: (y[:, :qh], y[:, qh:qh + kvh], y[:, qh + kvh:])  # noqa: E731
    got = cache.append(1, RaggedBatch.of([0], [tokens], dev), *split(x), rope, gamma, gamma)
    data = cache.data.clone()
    cache.data.fill_(7.0)
    out = torch.empty_like(got)
    for at in range(0, tokens, 100):
        n = min(100, tokens - at)
        cache.lengths[0] = at + n
        out[at:at + n] = cache.append(1, RaggedBatch.of([0], [n], dev), *split(x[at:at + n]), rope, gamma, gamma)
    assert torch.equal(out, got) and torch.equal(cache.data, data) and cache.status() == 0
