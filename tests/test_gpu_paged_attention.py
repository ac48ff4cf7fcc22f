"""Attention over pages against 64 bits: decode steps, chunks, whole prompts and mixtures; lengths
around the kernels' tiles, heads, types, page sizes; values that no token sees (Inf and NaN among
them), bad pages and batches, strides, streams and graphs."""

import pytest
import torch

import paged_ref
from llm_accelerator_amd import _lib
from llm_accelerator_amd.paged import PagedKVCache, PagedWorkspace, RaggedBatch

pytestmark = pytest.mark.gpu
F, B = torch.float16, torch.bfloat16


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def filled(dev, lengths, kvh, d, ps, dtype, seed=0, layers=1, garbage=True):
    """A cache whose sequences' positions are N(0, 1); everything else, the rows behind the last
    position among them, holds NaN and Inf."""
    need = [-(-n // ps) for n in lengths]
    pages = sum(need) + 2
    cache = PagedKVCache(layers, pages, ps, kvh, d, len(lengths), max(max(lengths), 1) + ps, dtype, dev)
    g = torch.Generator(device=dev).manual_seed(seed + sum(lengths))
    cache.data.normal_(generator=g)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    at = 0
    keep = torch.zeros(pages, ps, dtype=torch.bool)
    for s, n in enumerate(lengths):
        own = order[at:at + need[s]]
        cache.table[s, :need[s]] = own.to(torch.int32)
        keep[own] = (torch.arange(need[s] * ps) < n).view(need[s], ps)
        at += need[s]
    if garbage:
        bad = ~keep.to(dev)
        junk = torch.full_like(cache.data, float("nan"))
        junk[..., ::2] = float("inf")
        cache.data.copy_(torch.where(bad[None, None, :, None, :, None], junk, cache.data))
    cache.lengths.copy_(i32(lengths, dev))
    return cache


def compare(cache, batch, q, out, scaling, layer=0, keep=None):
    ref, size, tiny = paged_ref.attend(cache, layer, batch, q, scaling)
    seen = ~ref.isnan().all(-1).all(-1) if keep is None else keep
    err = (out.double() - ref)[seen].abs()
    bound = paged_ref.attend_bound(ref, size, tiny, q.dtype)[seen]
    print(f"[attend] worst {float((err / bound).max()) if err.numel() else 0:.3f} of the bound", flush=True)
    assert bool((err <= bound).all())
    return seen


DECODE = [  # lengths (one new token each), q heads, kv heads, dim, page, type
    ([1], 16, 8, 128, 64, F), ([2, 1, 15, 16, 17], 16, 8, 128, 16, F), ([31, 32, 33, 63, 64, 65], 2, 2, 128, 32, B),
    ([127, 128, 129, 1000], 16, 8, 128, 64, F), ([700], 16, 1, 128, 16, F), ([511, 512, 513], 8, 1, 64, 128, B),
    ([4097], 16, 8, 128, 64, F), ([9000, 40], 14, 2, 64, 16, F), ([300] * 40, 6, 2, 128, 64, B),
    ([1 + (53 * i) % 400 for i in range(130)], 4, 4, 64, 16, F), ([2500, 2000, 1, 64] + [100] * 30, 12, 4, 128, 256, F),
    ([5000 - 300 * i for i in range(8)], 3, 1, 128, 32, B), ([257], 5, 1, 64, 256, F),
]


@pytest.mark.parametrize("lengths,qh,kvh,d,ps,dtype", DECODE, ids=lambda v: f"{len(v)}x{max(v)}" if isinstance(v, list) else str(v))
def test_decode_vs_fp64(dev, lengths, qh, kvh, d, ps, dtype):
    cache = filled(dev, lengths, kvh, d, ps, dtype)
    n = len(lengths)
    batch = RaggedBatch.of(list(range(n))[::-1], [1] * n, dev)
    q = torch.randn(n, qh, d, device=dev, generator=torch.Generator(device=dev).manual_seed(n)).to(dtype)
    ws = cache.workspace(qh, batch)
    out = cache.attention(0, batch, q, 0.11, ws=ws)
    compare(cache, batch, q, out, 0.11)
    assert cache.status() == 0
    assert torch.equal(cache.attention(0, batch, q, 0.11, ws=ws), out)  # the workspace is as the first call found it


CHUNKS = [  # (length, new) of every sequence, q heads, kv heads, dim, page, type
    ([(2, 2)], 16, 8, 128, 64, F), ([(8, 8), (9, 3), (100, 7)], 16, 8, 128, 16, F), ([(17, 17)], 1, 1, 64, 16, B),
    ([(64, 64)], 2, 1, 128, 64, F), ([(65, 65), (63, 63), (1, 1)], 4, 2, 128, 32, F),
    ([(130, 129), (500, 33)], 16, 8, 128, 64, B), ([(257, 200)], 7, 1, 128, 128, F), ([(300, 1), (300, 150), (40, 0)], 8, 4, 64, 16, F),
    ([(3000, 5)], 16, 8, 128, 64, F), ([(2100, 16), (900, 8)], 16, 2, 128, 32, B), ([(1500, 300)], 16, 8, 128, 64, F),
    ([(129, 128), (4000, 64)], 16, 16, 64, 64, F), ([(i + 3, 1 + i % 3) for i in range(70)], 6, 3, 128, 16, F),
    ([(1025, 2)] * 3 + [(40, 40)], 32, 2, 128, 64, B), ([(700, 33)] * 5, 2, 2, 128, 64, F),
    ([(333, 333), (12, 12)], 16, 1, 128, 256, B), ([(4500, 18)], 8, 8, 128, 16, F),
    # at most 17 to 32 rows a kv head, sequences of one group of 16 among them
    ([(700, 4)], 64, 8, 128, 64, F), ([(5000, 4), (3, 3), (129, 2), (900, 0), (64, 1)], 16, 2, 128, 16, B),
    ([(300 + 31 * i, 1 + i % 8) for i in range(20)], 8, 2, 64, 32, F), ([(2, 2), (2000, 2)], 32, 2, 128, 256, F),
    ([(32, 32), (33, 17), (31, 31), (1000, 16)], 3, 3, 64, 16, B), ([(40 + i, 1 + i % 5) for i in range(90)], 12, 2, 128, 64, F),
]


@pytest.mark.parametrize("seqs,qh,kvh,d,ps,dtype", CHUNKS, ids=lambda v: f"{len(v)}x{max(v)}" if isinstance(v, list) else str(v))
def test_chunks_vs_fp64(dev, seqs, qh, kvh, d, ps, dtype):
    cache = filled(dev, [n for n, _ in seqs], kvh, d, ps, dtype, seed=3)
    batch = RaggedBatch.of(list(range(len(seqs))), [a for _, a in seqs], dev)
    g = torch.Generator(device=dev).manual_seed(len(seqs))
    q = (2 * torch.randn(batch.tokens, qh, d, device=dev, generator=g)).to(dtype)
    ws = cache.workspace(qh, batch)
    out = cache.attention(0, batch, q, ws=ws)
    compare(cache, batch, q, out, d ** -0.5)
    assert cache.status() == 0
    assert torch.equal(cache.attention(0, batch, q, ws=ws), out)


@pytest.mark.parametrize("dtype", [F, B], ids=["f16", "bf16"])
@pytest.mark.parametrize("new,length", [(5, 40), (12, 90), (16, 700), (40, 100), (150, 150)])
def test_what_a_token_does_not_see_does_not_reach_it(dev, new, length, dtype):
    """Inf and NaN in the keys and values of later tokens of the same chunk: earlier rows are as without
    them, later ones are not finite."""
    cache = filled(dev, [length], 2, 128, 16, dtype)
    batch = RaggedBatch.of([0], [new], dev)
    q = torch.randn(new, 4, 128, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(dtype)
    clean = cache.attention(0, batch, q)
    for first, value, plane in ((new - 1, float("nan"), 1), (new // 2, float("inf"), 1), (new // 2, float("nan"), 0),
                                (1, float("-inf"), 1), (new // 3 + 1, float("inf"), 0)):
        pos = length - new + first
        page, off = int(cache.table[0, pos // 16]), pos % 16
        saved = cache.data[0, plane, page, :, off].clone()
        cache.data[0, plane, page, :, off, 5:7] = value
        out = cache.attention(0, batch, q)
        assert bool(out[:first].isfinite().all()), (first, value, plane)
        err = (out[:first].double() - clean[:first].double()).abs()
        assert bool((err <= torch.finfo(dtype).eps * clean[:first].double().abs() + 2.0 ** -14).all())
        if plane == 1:
            assert not bool(out[first:, :, 5:7].isfinite().any())
            assert bool(out[first:, :, 8:].isfinite().all())
        elif value != value:
            assert not bool(out[first:].isfinite().any())
        cache.data[0, plane, page, :, off] = saved


def test_extreme_scores(dev):
    """Scores far apart, equal, and at the ends of fp16: no overflow on the way."""
    cache = filled(dev, [200, 200, 200], 1, 64, 16, F, garbage=False)
    for s, scale in ((0, 200.0), (1, 0.0), (2, 60000.0)):
        for i in range(13):
            cache.data[0, 0, int(cache.table[s, i])] = scale * torch.randn(1, 16, 64, device=dev).sign() if scale else 0
    for counts in ([1, 1, 1], [30, 30, 30]):
        batch = RaggedBatch.of([0, 1, 2], counts, dev)
        q = torch.randn(batch.tokens, 4, 64, device=dev, generator=torch.Generator(device=dev).manual_seed(4)).half()
        out = cache.attention(0, batch, q, 1.0)
        assert bool(out.isfinite().all())
        # scores up to 2^20 are rounded to 2^-4 in fp32 and so are the differences of exponents: only
        # the rows of one winner (60000) and of equal scores are pinned down
        ref, size, _ = paged_ref.attend(cache, 0, batch, q, 1.0)
        mid = slice(sum(counts[:1]), sum(counts[:2]))
        err = (out[mid].double() - ref[mid]).abs()
        assert bool((err <= 2.0 ** -11 * ref[mid].abs() + (2.0 ** -11 + 2.0 ** -14) * size[mid]).all())
    batch = RaggedBatch.of([0], [1], dev)
    q = torch.randn(1, 4, 64, device=dev).half()
    cache.data[0, 0].fill_(-60000.0)      # every score far below zero
    q.fill_(60000.0)
    out = cache.attention(0, batch, q, 1.0)
    v = torch.cat([cache.data[0, 1, int(p)][0] for p in cache.table[0, :13]])[:200].double()
    assert bool(((out[0].double() - v.mean(0)).abs() <= 2.0 ** -10 * v.abs().mean(0)).all())


@pytest.mark.parametrize("counts", [(1, 1, 1, 1), (3, 1, 2, 2), (12, 1, 16, 9), (40, 1, 17, 9)], ids=str)
def test_bad_pages_are_positions_that_are_not_there(dev, counts):
    lengths = [150, 90, 64, 47]
    cache = filled(dev, lengths, 2, 128, 16, F)
    cache.table[0, 1], cache.table[0, 9] = -1, 2 ** 31 - 1
    cache.table[2, :] = -2 ** 31                       # nothing of the sequence is there
    cache.table[3, 0] = cache.num_pages
    batch = RaggedBatch.of([0, 1, 2, 3], counts, dev)
    q = torch.randn(batch.tokens, 4, 128, device=dev).half()
    out = cache.attention(0, batch, q, out=torch.full_like(q, 3.0))
    compare(cache, batch, q, out, 128 ** -0.5)
    lo = sum(counts[:2])
    assert bool((out[lo:lo + counts[2]] == 0).all())
    assert cache.status() == _lib.STATUS_BAD_PAGE


@pytest.mark.parametrize("counts", [(1, 1, 1, 0), (2, 5, 3, 1), (20, 64, 30, 1)], ids=str)
def test_bad_sequences_and_padding_are_left_as_they_were(dev, counts):
    lengths = [150, 90, 64, 47]
    t = sum(counts) + 4
    for change in ("none", "row", "negative", "short", "long", "starts", "tokens", "new"):
        cache = filled(dev, lengths, 2, 128, 32, F)
        seqs, starts, tokens, most = [0, 1, 2, 3], [0], t, max(counts)
        for c in counts:
            starts.append(starts[-1] + c)
        bad = {1}
        if change == "row":
            seqs[1] = 4
        elif change == "negative":
            seqs[1] = -1
        elif change == "short":
            cache.lengths[1] = counts[1] - 1
        elif change == "long":
            cache.lengths[1] = 1 << 30
        elif change == "starts":     # entry 1 decreases, entry 0 is cut short
            starts[2] = starts[1] - 1
            bad = {1, 2}
        elif change == "tokens":
            starts[4] = t + 1
            bad = {3}
        elif change == "new" and max(counts) > min(c for c in counts if c):
            most = max(counts) - 1
            bad = {b for b, c in enumerate(counts) if c > most}
        else:
            bad = set()
        batch = RaggedBatch(i32(seqs, dev), i32(starts, dev), tokens, most)
        q = torch.randn(t, 4, 128, device=dev).half()
        q[sum(counts):] = float("nan")
        out = torch.full_like(q, 3.0)
        cache.attention(0, batch, q, out=out)
        good = torch.zeros(t, dtype=torch.bool, device=dev)
        for b, c in enumerate(counts):
            if b not in bad:
                good[starts[b]:starts[b + 1]] = True
        if change == "starts":
            continue_rows = range(starts[1], starts[1])   # what entry 2 covers overlaps: only bounds and status are pinned
            assert cache.status() == _lib.STATUS_BAD_SEQUENCE and not list(continue_rows)
            assert bool((out[sum(counts):] == 3.0).all())
            continue
        untouched = ~good
        assert bool((out[untouched] == 3.0).all()), change
        assert cache.status() == (_lib.STATUS_BAD_SEQUENCE if bad else 0), change
        for b in sorted(set(range(4)) - bad):
            one = RaggedBatch(i32([seqs[b]], dev), i32([0, counts[b]], dev), max(counts[b], 1), max(counts[b], 1))
            if counts[b]:
                lo = starts[b]
                compare(cache, one, q[lo:lo + counts[b]], out[lo:lo + counts[b]], 128 ** -0.5)


@pytest.mark.parametrize("counts", [[1, 1, 1], [4, 1, 2], [70, 3, 1]], ids=str)
def test_strides_in_place_layers_and_row_order(dev, counts):
    """q as a slice of a wider projection, out over q, another layer, a sequence twice."""
    cache = filled(dev, [200, 77, 140], 2, 128, 64, B, layers=3)
    batch = RaggedBatch.of([2, 0, 2], counts, dev)
    wide = torch.randn(batch.tokens, 11, 128, device=dev).to(B)
    q = wide[:, 3:9]
    want = cache.attention(2, batch, q.contiguous())
    compare(cache, batch, q.contiguous(), want, 128 ** -0.5, layer=2)
    rest = torch.cat((wide[:, :3], wide[:, 9:]), 1).clone()
    got = cache.attention(2, batch, q, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    assert torch.equal(torch.cat((wide[:, :3], wide[:, 9:]), 1), rest)


def test_python_refusals(dev):
    cache = filled(dev, [20, 30], 2, 64, 16, F)
    batch = RaggedBatch.of([0, 1], [1, 2], dev)
    q = torch.zeros(3, 4, 64, dtype=F, device=dev)
    bad = [dict(q=q.float()), dict(q=q[:2]), dict(q=q[:, :, :32]), dict(q=q[0]), dict(q=q.cpu()), dict(out=q.float()),
           dict(out=q[:2]), dict(out=torch.zeros(3, 4, 65, dtype=F, device=dev)[:, :, :64])]
    for kw in bad:
        with pytest.raises(ValueError):
            cache.attention(0, batch, **{"q": q, **kw})
    for kw, err in ((dict(layer=1), -2), (dict(q=q[:, :3].contiguous()), -11)):
        with pytest.raises(_lib.Q4DecError) as e:
            cache.attention(**{"layer": 0, "batch": batch, "q": q, **kw})
        assert e.value.code == err
    small = PagedWorkspace(cache, 4, 1, 1, 1)          # of decode steps: too small for a chunk
    chunk = RaggedBatch.of([0], [20], dev)
    with pytest.raises(_lib.Q4DecError) as e:
        cache.attention(0, chunk, torch.zeros(20, 4, 64, dtype=F, device=dev), ws=small)
    assert e.value.code == -9
    with pytest.raises(ValueError):
        cache.attention(0, RaggedBatch(None, i32([0, 1, 2, 3], dev), 3, 1), q)   # three sequences, two rows
    with pytest.raises(ValueError):
        cache.fork(i32([0], dev), i32([1, 1], dev))
    with pytest.raises(ValueError):
        cache.truncate(torch.zeros(1, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError):
        cache.append(0, batch, None, q[:, :2], q[:, :2].float())
    with pytest.raises(ValueError):
        cache.append(0, batch, None, q[:, :2], q[:, :2], q_out=q)
    with pytest.raises(ValueError):
        cache.append(0, batch, q, q[:, :2], q[:, :2], q_gamma=torch.ones(64, dtype=F, device=dev))
    with pytest.raises(ValueError):
        PagedKVCache.over(cache.data.float(), cache.table, cache.lengths, cache.refs)
    with pytest.raises(ValueError):
        PagedKVCache.over(cache.data, cache.table.long(), cache.lengths, cache.refs)
    with pytest.raises(_lib.Q4DecError):
        PagedKVCache(1, 4, 24, 2, 64, 2, 64, F, dev)


@pytest.mark.parametrize("counts", [[1] * 5, [3, 1, 2, 8, 5], [13, 1, 16, 2, 9], [90, 1, 33, 2, 1]], ids=str)
def test_streams_and_graphs_share_a_workspace_in_turn(dev, counts):
    """Two captured calls of one workspace, replayed in turn between eager ones, on lengths that change."""
    cache = filled(dev, [900, 600, 2000, 50, 130], 2, 128, 16, F)
    batches = [RaggedBatch.of([0, 1, 2, 3, 4], counts, dev), RaggedBatch.of([4, 2, 0], counts[:3], dev)]
    ws = cache.workspace(4, batches[0])
    qs = [torch.randn(b.tokens, 4, 128, device=dev).half() for b in batches]
    outs = [torch.zeros_like(q) for q in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for b, q, o in zip(batches, qs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
            cache.attention(0, b, q, out=o, ws=ws)
        graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    for lengths in ([900, 600, 2000, 50, 130], [130, 400, 1999, 16, 100], [899, 64, 200, 8, 128]):
        cache.lengths.copy_(i32(lengths, dev))
        ok = all(n >= c for n, c in zip(lengths, counts)) and lengths[4] >= counts[0] and lengths[0] >= counts[2]
        for g, b, q, o in zip(graphs, batches, qs, outs):
            q.normal_()
            o.fill_(3.0)
            g.replay()
            got = o.clone()
            assert torch.equal(cache.attention(0, b, q, out=torch.full_like(q, 3.0), ws=ws), got)
            if ok:
                compare(cache, b, q, got, 128 ** -0.5)
    side2 = torch.cuda.Stream()
    side2.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side2):
        got = cache.attention(0, batches[0], qs[0])
    torch.cuda.current_stream().wait_stream(side2)
    assert torch.equal(got, cache.attention(0, batches[0], qs[0], ws=ws)) or not ok


def test_two_calls_at_once_with_their_own_workspaces(dev):
    cache = filled(dev, [3000, 2000, 2500], 2, 128, 64, F)
    jobs = []
    for seqs, counts in (([0, 1, 2], [1, 1, 1]), ([2, 0], [5, 3]), ([1], [120])):
        b = RaggedBatch.of(seqs, counts, dev)
        q = torch.randn(b.tokens, 8, 128, device=dev).half()
        jobs.append((b, q, cache.workspace(8, b), torch.cuda.Stream()))
    want = [cache.attention(0, b, q) for b, q, _, _ in jobs]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        got.clear()
        for b, q, ws, st in jobs:
            with torch.cuda.stream(st):
                got.append(cache.attention(0, b, q, ws=ws))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("n", [20, 64, 130, 700])
def test_starts_that_go_back_and_forth_leave_the_workspace_as_it_was(dev, n):
    """More tiles than the token rows have: the bad batch is reported, the next call is as ever."""
    cache = filled(dev, [900] * n, 1, 128, 16, F)
    good = RaggedBatch.of(list(range(n))[:8], [60, 1, 30, 100, 1, 2, 5, 50], dev)
    q = torch.randn(good.tokens, 16, 128, device=dev).half()
    ws = max((cache.workspace(16, good), PagedWorkspace(cache, 16, n, 200, 200)), key=lambda w: w.nbytes)
    want = cache.attention(0, good, q, ws=ws)
    for low, high in ((0, 200), (150, 200), (3, 40)):
        starts = [(low, high)[b % 2] for b in range(n + 1)]
        bad = RaggedBatch(i32(list(range(n)), dev), i32(starts, dev), 200, 200)
        print(f"[bad] n={n} {low} {high}", flush=True)
        cache.attention(0, bad, torch.zeros(200, 16, 128, dtype=F, device=dev), ws=ws)
        assert cache.status() == _lib.STATUS_BAD_SEQUENCE
        cache._status.zero_()
        assert torch.equal(cache.attention(0, good, q, ws=ws), want)
    assert cache.status() == 0


def test_offsets_past_32_bits(dev):
    """A pool of more than 2^31 elements a plane, the sequence in its last pages."""
    kvh, d, ps = 8, 128, 64
    pages = (1 << 31) // (kvh * d * ps) + 9
    data = torch.empty(1, 2, pages, kvh, ps, d, dtype=F, device=dev)
    table = torch.full((2, 8), -1, dtype=torch.int32, device=dev)
    table[1] = torch.arange(pages - 8, pages, dtype=torch.int32, device=dev).flip(0)
    data[:, :, -8:].normal_()
    cache = PagedKVCache.over(data, table, i32([0, 500], dev), torch.zeros(pages, dtype=torch.int32, device=dev))
    for new in (1, 3, 60):
        batch = RaggedBatch.of([1], [new], dev)
        q = torch.randn(new, 16, d, device=dev).half()
        kv = torch.randn(new, kvh, d, device=dev).half()
        cache.append(0, batch, None, kv, -kv)
        at = torch.arange(500 - new, 500, device=dev)
        assert torch.equal(data[0, 1, table[1, at // ps].long(), :, at % ps], -kv)
        compare(cache, batch, q, cache.attention(0, batch, q), d ** -0.5)


@pytest.mark.parametrize("scaling", [0.0, -0.2, 3.0])
def test_any_finite_scaling(dev, scaling):
    cache = filled(dev, [90, 200], 2, 64, 16, F)
    for counts in ([1, 1], [40, 3]):
        batch = RaggedBatch.of([0, 1], counts, dev)
        q = torch.randn(batch.tokens, 6, 64, device=dev, generator=torch.Generator(device=dev).manual_seed(5)).half()
        compare(cache, batch, q, cache.attention(0, batch, q, scaling), scaling)


def test_one_workspace_for_calls_of_every_shape(dev):
    """The counters that a call finds are those the one before left, whatever its shape was."""
    caches = [filled(dev, [3000, 700, 90], 2, 128, 16, F), filled(dev, [2000, 50, 1200, 800], 5, 64, 32, F),
              filled(dev, [1500], 1, 128, 64, B)]
    ws = PagedWorkspace(caches[0], 32, 4, 400, 400)
    for cache in caches:
        big = PagedWorkspace(cache, 16 * cache.num_kv_heads, 4, 400, 400)
        ws = big if big.nbytes > ws.nbytes else ws
    jobs = []
    for i, (counts, qh) in enumerate([([1, 1, 1], 4), ([1] * 4, 15), ([1], 16), ([5, 60, 1], 8), ([100, 2, 1, 33], 5), ([300], 3),
                                      ([8, 8, 8], 4), ([3, 3, 3, 3], 80)]):
        cache = caches[2 if len(counts) == 1 else len(counts) - 3]
        batch = RaggedBatch.of(list(range(len(counts))), counts, dev)
        q = torch.randn(batch.tokens, qh, cache.head_dim, device=dev).to(cache.dtype)
        jobs.append((cache, batch, q, cache.attention(0, batch, q)))
    for order in (jobs, jobs[::-1], jobs[1:] + jobs[:1]):
        for cache, batch, q, want in order:
            assert torch.equal(cache.attention(0, batch, q, ws=ws), want)


@pytest.mark.parametrize("n", [64, 65, 300, 4096])
def test_many_sequences(dev, n):
    """As many sequences as lanes, one more, more than threads, and the most: decode steps, chunks and
    sequences without new tokens mixed."""
    lengths = [1 + (29 * i) % 90 for i in range(n)]
    counts = [min(lengths[i], (0, 1, 1, 3, 40)[(7 * i) % 5]) for i in range(n)]
    cache = filled(dev, lengths, 1, 64, 16, F)
    for most in (3, 40):
        few = [c if c <= most else 2 for c in counts]
        batch = RaggedBatch.of(list(range(n)), few, dev)
        q = torch.randn(batch.tokens, 3, 64, device=dev, generator=torch.Generator(device=dev).manual_seed(n)).half()
        out = cache.attention(0, batch, q)
        assert cache.status() == 0
        some = sorted({0, 1, n // 2, n - 2, n - 1} | set(range(0, n, max(1, n // 60))))
        at = batch.starts.tolist()
        rows = torch.cat([torch.arange(at[b], at[b + 1]) for b in some])
        one = RaggedBatch.of(some, [few[b] for b in some], dev)
        compare(cache, one, q[rows], out[rows], 64 ** -0.5)


def test_prompts_of_many_lengths_finish_in_any_order(dev):
    """Tiles of several sequences in the order of their steps: lengths on both sides of a tile and a step."""
    seqs = [(700, 700), (64, 64), (65, 65), (1300, 130), (127, 127), (128, 128), (129, 129), (900, 17), (33, 1), (2000, 511)]
    cache = filled(dev, [n for n, _ in seqs], 2, 128, 16, B)
    for qh in (2, 6, 14):
        batch = RaggedBatch.of(list(range(len(seqs))), [a for _, a in seqs], dev)
        q = torch.randn(batch.tokens, qh, 128, device=dev, generator=torch.Generator(device=dev).manual_seed(qh)).to(B)
        compare(cache, batch, q, cache.attention(0, batch, q), 128 ** -0.5)
