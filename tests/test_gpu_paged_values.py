"""Attention over pages where the values are hard: Inf and NaN that a token sees, by kind; scores that are
-Inf or of any scale; sums beyond the cache type's largest number; probabilities that must not be rounded
to 16 bits."""

import math

import pytest
import torch

import paged_ref
from llm_accelerator_amd import _lib
from llm_accelerator_amd.paged import PagedKVCache, RaggedBatch
from test_gpu_paged_attention import filled, i32

pytestmark = pytest.mark.gpu
F, B = torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


def queries(dev, batch, qh, d, dtype, seed=1):
    return torch.randn(batch.tokens, qh, d, device=dev, generator=torch.Generator(device=dev).manual_seed(seed)).to(dtype)


def at(cache, row, pos):
    return int(cache.table[row, pos // cache.page_size]), pos % cache.page_size


def check_kinds(cache, batch, q, out, scaling):
    """Every output is NaN, Inf or -Inf where the 64-bit one is, and within the bound elsewhere."""
    ref, size, tiny = paged_ref.attend(cache, 0, batch, q, scaling)
    assert torch.equal(out.isnan(), ref.isnan())
    assert torch.equal(out.isposinf(), ref.isposinf()) and torch.equal(out.isneginf(), ref.isneginf())
    ok = ref.isfinite()
    bound = paged_ref.attend_bound(ref, size, tiny, q.dtype)
    assert bool(((out.double() - ref).abs() <= bound)[ok].all())
    return ok


# (positions, new tokens) of every sequence, q heads, kv heads, dim, page, and places (sequence, position)
SEEN = [
    ([(1, 1)], 16, 8, 128, 64, [(0, 0)]),
    ([(700, 1)], 16, 8, 128, 64, [(0, 0), (0, 351), (0, 699)]),
    ([(300, 1), (37, 1), (2500, 1)], 4, 1, 64, 16, [(0, 5), (1, 36), (2, 1200)]),
    ([(9000, 1)], 8, 1, 128, 32, [(0, 40), (0, 8990)]),          # many parts
    ([(300, 5)], 16, 8, 128, 64, [(0, 100), (0, 296), (0, 299)]),
    ([(700, 4)], 16, 2, 64, 16, [(0, 100), (0, 698)]),           # two groups of rows
    ([(900, 60)], 4, 2, 128, 64, [(0, 40), (0, 838), (0, 870)]),  # a chunk: before its edge and in it
    ([(6000, 40)], 8, 1, 64, 16, [(0, 17), (0, 3001), (0, 5990)]),
    ([(300, 300)], 2, 2, 128, 128, [(0, 0), (0, 128), (0, 290)]),
    ([(500, 1), (400, 70), (90, 2)], 4, 2, 128, 16, [(0, 77), (1, 50), (1, 380), (2, 89)]),
]


@pytest.mark.parametrize("dtype", [F, B], ids=["f16", "bf16"])
@pytest.mark.parametrize("seqs,qh,kvh,d,ps,places", SEEN, ids=lambda v: "x".join(f"{a}:{b}" for a, b in v) if isinstance(v, list) else str(v))
def test_inf_and_nan_that_a_token_sees(dev, seqs, qh, kvh, d, ps, places, dtype):
    """Inf gives Inf, -Inf gives -Inf, NaN and both signs give NaN, in that dim alone."""
    cache = filled(dev, [n for n, _ in seqs], kvh, d, ps, dtype)
    batch = RaggedBatch.of(list(range(len(seqs))), [a for _, a in seqs], dev)
    q = queries(dev, batch, qh, d, dtype)
    ws = cache.workspace(qh, batch)
    for s, pos in places:
        page, off = at(cache, s, pos)
        saved = cache.data[0, 1, page, :, off].clone()
        for dim, value in ((3, INF), (d - 1, -INF), (17, NAN)):
            cache.data[0, 1, page, :, off, dim] = value
        other = max(0, pos - 1)                       # (the same position in the first case)
        page2, off2 = at(cache, s, other)
        saved2 = cache.data[0, 1, page2, :, off2, 40].clone()
        cache.data[0, 1, page2, :, off2, 40] = INF
        if other != pos:
            cache.data[0, 1, page, :, off, 40] = -INF
        print(f"[seen] {s} {pos}", flush=True)
        ok = check_kinds(cache, batch, q, cache.attention(0, batch, q, ws=ws), d ** -0.5)
        assert not bool(ok.all()) and cache.status() == 0
        cache.data[0, 1, page2, :, off2, 40] = saved2
        cache.data[0, 1, page, :, off] = saved
    assert bool(check_kinds(cache, batch, q, cache.attention(0, batch, q, ws=ws), d ** -0.5).all())


@pytest.mark.parametrize("dtype", [F, B], ids=["f16", "bf16"])
@pytest.mark.parametrize("length,new,qh,kvh", [(700, 1, 4, 2), (9000, 1, 8, 1), (300, 5, 4, 2), (900, 60, 4, 2), (6000, 40, 8, 1)])
def test_an_inf_of_the_smallest_weight_counts(dev, length, new, qh, kvh, dtype):
    """The first half's probabilities are e^-424 and less: nothing in 32 bits, and still Inf where V is Inf."""
    cache = filled(dev, [length], kvh, 128, 16, dtype)
    batch = RaggedBatch.of([0], [new], dev)
    q = queries(dev, batch, qh, 128, dtype)
    q[..., 0] = 8.0
    for pos in range(0, length // 2, 16):
        page, _ = at(cache, 0, pos)
        cache.data[0, 0, page, :, :min(16, length // 2 - pos), 0] = -600.0
    for pos in (5, length // 2 - 1):
        page, off = at(cache, 0, pos)
        cache.data[0, 1, page, :, off, 9] = INF
        cache.data[0, 1, page, :, off, 10] = -INF
        cache.data[0, 1, page, :, off, 11] = NAN
        out = cache.attention(0, batch, q)
        check_kinds(cache, batch, q, out, 128 ** -0.5)
        assert bool(out[..., 9].isposinf().all()) and bool(out[..., 10].isneginf().all())
        cache.data[0, 1, page, :, off, 9:12] = 0


def test_a_value_past_fp16_is_inf_from_the_append_on(dev):
    """v = 1e5 becomes Inf in an fp16 cache, and so do the outputs of the tokens that see it, however many they are."""
    cache = PagedKVCache(1, 40, 16, 2, 64, 2, 512, F, dev)
    for counts in ([1, 90], [1, 1], [5, 2], [20, 1]):
        batch = RaggedBatch.of([0, 1], counts, dev)
        cache.reserve(batch)
        x = torch.randn(batch.tokens, 8, 64, device=dev)
        x[:, 6:, 7] = 1e5
        x[:, 6:, 8] = -1e5
        out = cache.attention(0, batch, cache.append(0, batch, x[:, :4], x[:, 4:6], x[:, 6:]))
        assert bool(out[..., 7].isposinf().all()) and bool(out[..., 8].isneginf().all())
        out[..., 7:9] = 0
        assert bool(out.isfinite().all()) and cache.status() == 0


def two_groups(dev, length, new, kvh, d, ps, dtype):
    """A cache and a query of exact scores: the even positions' are 0, the odd ones' -scaling.  With a scaling
    of -log(1 / 2 + eps / 4) an odd position's weight is half-way between two numbers of the cache's type,
    and V, 1 and -(2 - eps), cancels: 16-bit weights move the output by a third of eps, which nothing hides."""
    cache = filled(dev, [length], kvh, d, ps, dtype, garbage=False)
    pos = torch.arange(length, device=dev)
    page, off = cache.table[0, pos // ps].long(), pos % ps
    odd = (pos % 2 == 1).to(dtype)
    k = torch.zeros(length, kvh, d, device=dev, dtype=dtype)
    k[:, :, 0] = odd[:, None]
    v = torch.where(pos % 2 == 1, torch.finfo(dtype).eps - 2.0, 1.0).to(dtype).view(-1, 1, 1).expand(length, kvh, d)
    cache.data[0, 0, page, :, off] = k
    cache.data[0, 1, page, :, off] = v
    q = torch.zeros(new, 4 * kvh, d, device=dev, dtype=dtype)
    q[..., 0] = -1.0
    return cache, q


@pytest.mark.parametrize("dtype", [F, B], ids=["f16", "bf16"])
@pytest.mark.parametrize("length,new,d", [(64, 1, 64), (600, 1, 128), (3000, 4, 64), (600, 3, 128), (600, 8, 64), (640, 120, 128),
                                          (4000, 30, 64), (256, 256, 128)])
def test_probabilities_keep_more_than_16_bits(dev, length, new, d, dtype):
    """Scores are exact (a product of two numbers, scaled in fp32), so a weight is off by 2^-20 (exponent of up to
    2 in base 2, its factors and the exponential: 2^-23 each, and the maximum's), the weights' remainders by 2^-22
    (fp16) or 2^-16 (bf16), or 2^-25 of the largest, which may be taken 2^8 low only where scores differ by more;
    sums of up to `length` fp32 terms of one size by 2^-24 of length / 4 (a wave's or half wave's share, joined in
    few more steps), and the output by its own half step."""
    step = torch.finfo(dtype).eps
    scaling = -math.log(0.5 + 0.25 * step)
    cache, q = two_groups(dev, length, new, 1, d, 16, dtype)
    batch = RaggedBatch.of([0], [new], dev)
    out = cache.attention(0, batch, q, scaling)
    ref, size, _ = paged_ref.attend(cache, 0, batch, q, scaling)
    rest = 2.0 ** -22 if dtype == F else 2.0 ** -16
    bound = step / 2 * ref.abs() + (2.0 ** -20 + rest + 2.0 ** -24 * (length / 4 + 64)) * size
    worst = float(((out.double() - ref).abs() / bound).max())
    print(f"[precision] {worst:.3f} of the bound", flush=True)
    assert worst <= 1


@pytest.mark.parametrize("length,new,qh,kvh", [(2, 1, 2, 1), (700, 1, 4, 2), (9000, 1, 8, 1), (700, 4, 8, 1), (300, 60, 4, 2),
                                              (6000, 40, 8, 1), (256, 256, 2, 2)])
def test_means_of_the_largest_bf16_values_are_finite(dev, length, new, qh, kvh):
    """A weighted mean of values up to 3.2e38 is no larger than they are, though their sum passes fp32: equal
    scores, scores that rise by 6 (in base 2) from one 64 positions to the next, and random ones."""
    cache = filled(dev, [length], kvh, 128, 16, B, garbage=False)
    batch = RaggedBatch.of([0], [new], dev)
    pos = torch.arange(length, device=dev)
    page, off = cache.table[0, pos // 16].long(), pos % 16
    v = torch.linspace(2.0e38, 3.2e38, 128, device=dev).to(B)
    cache.data[0, 1, page, :, off] = v.expand(length, kvh, 128).contiguous()
    q = torch.zeros(new, qh, 128, dtype=B, device=dev)
    q[..., 0] = 1.0
    for kind in ("equal", "rising", "random"):
        k = torch.zeros(length, kvh, 128, device=dev)
        if kind == "rising":
            k[..., 0] = ((pos // 64) * 4.0).clamp(max=200)[:, None]
        elif kind == "random":
            k[..., 0] = 3 * torch.randn(length, kvh, device=dev, generator=torch.Generator(device=dev).manual_seed(2))
        cache.data[0, 0, page, :, off] = k.to(B)
        out = cache.attention(0, batch, q, 1.0)
        assert bool(out.isfinite().all()), kind
        # the mean of one value is that value; weights and sums as in test_probabilities_keep_more_than_16_bits
        bound = (2.0 ** -8 + 2.0 ** -16 + 2.0 ** -14) * v.double()
        assert bool(((out.double() - v.double()).abs() <= bound).all()), kind


def test_large_and_small_dims_side_by_side(dev):
    """Dims of 3e38 beside dims of 1e-25: the large ones' sums are taken with room above, the small ones keep theirs."""
    for new, length in ((1, 500), (50, 500)):
        cache = filled(dev, [length], 1, 64, 16, B, garbage=False)
        batch = RaggedBatch.of([0], [new], dev)
        cache.data[0, 1, :, :, :, :32] *= 1e38
        cache.data[0, 1, :, :, :, :32] = cache.data[0, 1, :, :, :, :32].clamp(-3.3e38, 3.3e38)
        cache.data[0, 1, :, :, :, 32:] *= 1e-25
        cache.data[0, 1, :, :, :, 0] = 3.2e38
        q = queries(dev, batch, 2, 64, B)
        out = cache.attention(0, batch, q, 0.02)
        assert bool(check_kinds(cache, batch, q, out, 0.02).all())


@pytest.mark.parametrize("dtype", [F, B], ids=["f16", "bf16"])
@pytest.mark.parametrize("length,new,qh,kvh", [(1, 1, 2, 1), (700, 1, 4, 2), (9000, 1, 8, 1), (300, 5, 4, 2), (900, 60, 4, 2),
                                              (6000, 40, 8, 1), (200, 200, 2, 2)])
def test_scores_that_are_all_minus_inf(dev, length, new, qh, kvh, dtype):
    """exp(-Inf - -Inf) is NaN, as in the definition; zeros are for tokens that see no position.  One finite
    score is enough for finite outputs."""
    cache = filled(dev, [length, length], kvh, 64, 16, dtype, garbage=False)
    batch = RaggedBatch.of([0, 1], [new, new], dev)
    q = queries(dev, batch, qh, 64, dtype)
    q[..., 0] = 1.0
    cache.data[0, 0, :, :, :, 0] = -INF
    out = cache.attention(0, batch, q)
    assert bool(out.isnan().all()) and cache.status() == 0
    page, off = at(cache, 1, length - new)
    cache.data[0, 0, page, :, off, 0] = 0.5
    ok = check_kinds(cache, batch, q, cache.attention(0, batch, q), 64 ** -0.5)
    assert bool(ok[new:].all()) and not bool(ok[:new].any())
    # no page of the first sequence is there: zeros, and the second is as before
    cache.table[0] = -1
    out = cache.attention(0, batch, q)
    assert bool((out[:new] == 0).all()) and bool(out[new:].isfinite().all())


@pytest.mark.parametrize("counts", [[1, 1], [40, 3]], ids=str)
def test_scalings_near_zero(dev, counts):
    """Scores are scaled by the value that is given, however small; by 0 they are all equal, but Inf x 0 is NaN."""
    cache = filled(dev, [90, 200], 2, 64, 16, B)
    batch = RaggedBatch.of([0, 1], counts, dev)
    q = queries(dev, batch, 6, 64, B, 5)
    for scaling, size in ((1e-33, 1e16), (-1e-33, 1e16), (3e-36, 1e18), (0.0, 1.0), (-0.0, 1e18)):
        rows = torch.arange(90, device=dev)
        page, off = cache.table[0, rows // 16].long(), rows % 16
        saved = cache.data[0, 0, page, :, off].clone()
        cache.data[0, 0, page, :, off] = saved * size
        big = (q.float() * size).to(B)
        check_kinds(cache, batch, big, cache.attention(0, batch, big, scaling), scaling)
        cache.data[0, 0, page[7], :, off[7], 3] = INF
        out = cache.attention(0, batch, q, 0.0)
        assert bool(out[:counts[0]].isnan().all()) and bool(out[counts[0]:].isfinite().all())
        cache.data[0, 0, page, :, off] = saved


def wider(cache, max_pages):
    """The same cache with room for more pages a row."""
    table = torch.full((cache.num_seqs, max_pages), -1, dtype=torch.int32, device=cache.device)
    table[:, :cache.max_pages] = cache.table
    return PagedKVCache.over(cache.data, table, cache.lengths, cache.refs)


MANY = [  # the chunks (positions, new tokens) among decode steps, sequences in all, q heads, kv heads, dim, page, type
    ([(6000, 20)], 65, 16, 1, 64, 16, F),                        # some 20 parts: joined in two levels
    ([(600, 600)], 66, 16, 1, 128, 32, B),                       # first tiles of fewer steps than the last's parts
    ([(4000, 300), (2000, 20), (2500, 77)], 70, 4, 2, 128, 64, F),
    ([(3000, 600), (5000, 50), (129, 128)], 130, 6, 3, 64, 16, B),
    ([(2000, 120), (1000, 1000)], 300, 2, 2, 128, 16, F),
    ([(2600, 33)] * 5, 69, 8, 1, 64, 64, F),
]


@pytest.mark.parametrize("chunks,n,qh,kvh,d,ps,dtype", MANY, ids=lambda v: f"{len(v)}x{max(v)}" if isinstance(v, list) else str(v))
def test_more_sequences_than_lanes_with_chunks_in_parts(dev, chunks, n, qh, kvh, d, ps, dtype):
    """Against 64 bits, repeated on one workspace, and bit for bit the same whatever the table has room for."""
    seqs = [(1 + (29 * i) % 90, i % 4 != 0) for i in range(n - len(chunks))]
    for i, c in enumerate(chunks):
        seqs.insert((37 * i + 11) % n, c)
    cache = filled(dev, [t for t, _ in seqs], kvh, d, ps, dtype, seed=n)
    batch = RaggedBatch.of(list(range(n)), [int(a) for _, a in seqs], dev)
    q = queries(dev, batch, qh, d, dtype, n)
    ws = cache.workspace(qh, batch)
    out = cache.attention(0, batch, q, ws=ws)
    check_kinds(cache, batch, q, out, d ** -0.5)
    assert cache.status() == 0
    assert torch.equal(cache.attention(0, batch, q, ws=ws), out)
    for room in (2 * cache.max_pages, (1 << 20) // ps):
        assert torch.equal(wider(cache, room).attention(0, batch, q, ws=ws), out), room
    assert torch.equal(cache.attention(0, batch, q, ws=ws), out)


@pytest.mark.parametrize("dtype", [F, B], ids=["f16", "bf16"])
@pytest.mark.parametrize("length,new", [(1, 1), (300, 1), (5000, 1), (90, 12), (700, 40), (4000, 25), (150, 150)])
def test_inf_and_nan_in_keys(dev, length, new, dtype):
    """A score of Inf or NaN makes the tokens that see it NaN, one of -Inf is a weight of 0, for each head by the
    signs of its query; tokens that do not see it are as without it."""
    cache = filled(dev, [length], 2, 128, 16, dtype)
    batch = RaggedBatch.of([0], [new], dev)
    q = queries(dev, batch, 8, 128, dtype)
    clean = cache.attention(0, batch, q)
    kinds = set()
    for pos in sorted({0, length // 2, max(0, length - new + new // 2), length - 1}):
        page, off = at(cache, 0, pos)
        saved = cache.data[0, 0, page, :, off].clone()
        for value, dims in ((INF, slice(5, 6)), (-INF, slice(5, 6)), (INF, slice(5, 7)), (NAN, slice(9, 10))):
            cache.data[0, 0, page, :, off, dims] = value
            out = cache.attention(0, batch, q)
            ok = check_kinds(cache, batch, q, out, 128 ** -0.5)
            kinds |= {bool(x) for x in ok.flatten().unique()}
            before = max(0, pos - (length - new))           # the tokens that do not see it
            err = (out[:before].double() - clean[:before].double()).abs()
            assert bool((err <= torch.finfo(dtype).eps * clean[:before].double().abs() + 2.0 ** -14).all())
            cache.data[0, 0, page, :, off] = saved
    assert kinds == {False, True} or length == 1
    assert torch.equal(cache.attention(0, batch, q), clean)


@pytest.mark.parametrize("counts", [(2, 1, 3, 1), (5, 4, 6, 2), (30, 64, 20, 9), (3, 40, 50, 1)], ids=str)
def test_entries_beside_a_bad_one(dev, counts):
    """starts go back by one: the entry that decreases is left out, and so is nothing else.  All rows but the
    one that two entries claim are compared."""
    cache = filled(dev, [150, 90, 64, 47], 2, 128, 32, F)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    starts[2] = starts[1] - 1                      # entry 1 is bad, entry 2 begins on entry 0's last row
    counts = [b - a for a, b in zip(starts, starts[1:])]
    lengths = [150, 90, max(64, counts[2]), 47]
    if counts[2] > 64:
        cache = filled(dev, lengths, 2, 128, 32, F)
    batch = RaggedBatch(i32([0, 1, 2, 3], dev), i32(starts, dev), starts[4], max(counts))
    q = queries(dev, batch, 4, 128, F)
    out = torch.full_like(q, 3.0)
    cache.attention(0, batch, q, out=out)
    for b, contested in ((0, counts[0] - 1), (2, 0), (3, None)):
        rows = q[starts[b]:starts[b + 1]]
        one = RaggedBatch.of([b], [counts[b]], dev)
        ref, size, tiny = paged_ref.attend(cache, 0, one, rows, 128 ** -0.5)
        bad = (out[starts[b]:starts[b + 1]].double() - ref).abs() > paged_ref.attend_bound(ref, size, tiny, F)
        bad = bad.flatten(1).any(1)
        if contested is not None:
            bad[contested] = False
        assert not bool(bad.any()), b
    assert cache.status() == _lib.STATUS_BAD_SEQUENCE


@pytest.mark.parametrize("counts", [[1, 1, 1], [5, 1, 3], [70, 1, 20]], ids=str)
def test_values_that_come_and_go_between_replays(dev, counts):
    """A captured call: Inf, NaN and the largest bf16 values appear in V and are
    gone again, and every replay is as the eager call and as 64 bits."""
    cache = filled(dev, [3000, 500, 900], 2, 128, 16, B)
    batch = RaggedBatch.of([0, 1, 2], counts, dev)
    q = queries(dev, batch, 4, 128, B)
    ws, out = cache.workspace(4, batch), torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        cache.attention(0, batch, q, out=out, ws=ws)
    torch.cuda.current_stream().wait_stream(side)
    clean = cache.data.clone()
    want = cache.attention(0, batch, q)
    for value in (INF, None, NAN, 3.3e38, None, -INF):
        cache.data.copy_(clean)
        if value is not None:
            for s, pos in ((0, 1500), (1, 3), (2, 899)):
                page, off = at(cache, s, pos)
                cache.data[0, 1, page, :, off, 20:24] = value
        g.replay()
        check_kinds(cache, batch, q, out, 128 ** -0.5)
        got = out.clone()
        again = cache.attention(0, batch, q, ws=ws)
        assert torch.equal(got.isnan(), again.isnan()) and torch.equal(got.nan_to_num(1.0), again.nan_to_num(1.0))
        if value is None:
            assert torch.equal(got, want)
    assert cache.status() == 0


@pytest.mark.parametrize("length,new", [(9000, 1), (2000, 300)])
def test_every_value_nan_or_inf(dev, length, new):
    cache = filled(dev, [length], 1, 64, 64, F)
    batch = RaggedBatch.of([0], [new], dev)
    q = queries(dev, batch, 4, 64, F)
    cache.data[0, 1, ..., :32] = NAN
    cache.data[0, 1, ..., 32:] = -INF
    out = cache.attention(0, batch, q)
    assert bool(out[..., :32].isnan().all()) and bool(out[..., 32:].isneginf().all())


@pytest.mark.parametrize("dtype", [F, B], ids=["f16", "bf16"])
@pytest.mark.parametrize("length,new,qh,kvh", [(1, 1, 2, 1), (700, 1, 4, 2), (9000, 1, 8, 1), (700, 4, 8, 1), (900, 60, 4, 2),
                                              (6000, 40, 8, 1)])
def test_an_inf_of_weight_zero_is_nan(dev, length, new, qh, kvh, dtype):
    """The score -Inf has the weight 0, and 0 x Inf is NaN; the other dims are as without the position."""
    cache = filled(dev, [length], kvh, 128, 16, dtype)
    batch = RaggedBatch.of([0], [new], dev)
    q = queries(dev, batch, qh, 128, dtype)
    q[..., 0] = 1.0
    for pos in {0, length // 3, length - 1}:
        page, off = at(cache, 0, pos)
        saved = cache.data[0, :, page, :, off].clone()
        cache.data[0, 0, page, :, off, 0] = -INF
        cache.data[0, 1, page, :, off, 30] = INF
        out = cache.attention(0, batch, q)
        check_kinds(cache, batch, q, out, 128 ** -0.5)
        assert bool(out[-1, :, 30].isnan().all()) and (length == 1 or bool(out[:, :, 31].isfinite().all()))
        cache.data[0, :, page, :, off] = saved
