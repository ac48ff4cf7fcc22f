"""Pages of the paged cache against a host model of the rules: reserving, forking, truncating and
compacting in random order, all-or-nothing failures, entries that cannot be, and the copied rows."""

import random

import pytest
import torch

import paged_ref
from llm_accelerator_amd import _lib
from llm_accelerator_amd.paged import PagedKVCache, RaggedBatch

pytestmark = pytest.mark.gpu

HELD = _lib.STATUS_NOT_RESERVED


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def pair(dev, num_pages, ps, num_seqs, max_pages, layers=2, kvh=2, d=64, dtype=torch.float16):
    """A cache and its host model; every row of every page holds a value of its own."""
    cache = PagedKVCache(layers, num_pages, ps, kvh, d, num_seqs, max_pages * ps, dtype, dev)
    marks = torch.arange(num_pages * ps, device=dev).view(num_pages, 1, ps, 1) % 1024
    cache.data.copy_((marks + torch.arange(layers * 2, device=dev).view(layers, 2, 1, 1, 1, 1) / 4
                      + torch.arange(kvh, device=dev).view(kvh, 1, 1) / 16).expand(cache.data.shape))
    model = paged_ref.Pages(num_pages, ps, num_seqs, max_pages)
    for p in range(num_pages):
        model.rows[p] = [(p * ps + r) % 1024 for r in range(ps)]
    return cache, model


def same(cache, model, rows=True):
    assert cache.lengths.tolist() == model.lengths
    assert cache.refs.tolist() == model.refs
    assert cache.table.tolist() == model.table
    assert cache.status() == model.status
    if rows:
        layers, _, pages, kvh, ps, d = cache.data.shape
        want = torch.tensor(model.rows, device=cache.device, dtype=torch.float64).view(1, 1, pages, 1, ps, 1)
        want = (want + torch.arange(layers * 2, device=cache.device).view(layers, 2, 1, 1, 1, 1) / 4
                + torch.arange(kvh, device=cache.device).view(kvh, 1, 1) / 16)
        assert torch.equal(cache.data, want.expand(cache.data.shape).to(cache.dtype))


def reserve(cache, model, seqs, counts):
    cache.reserve(RaggedBatch.of(seqs, counts, cache.device))
    model.reserve(seqs, counts)


@pytest.mark.parametrize("ps,dtype,d", [(16, torch.float16, 64), (64, torch.bfloat16, 128), (256, torch.float16, 128)])
def test_fork_then_write_copies_the_shared_rows(dev, ps, dtype, d):
    """Three forks of a partly filled page: two copies where all holders write, three where one does not."""
    for writers in ([1, 2, 3, 0], [3, 0, 2], [0], [2, 1]):
        print(f"[fork] ps={ps} writers={writers}", flush=True)
        cache, model = pair(dev, 23, ps, 6, 5, d=d, dtype=dtype)
        reserve(cache, model, [5, 0], [ps, 2 * ps + ps // 2 + 1])
        cache.fork(i32([0, 0, 0], dev), i32([2, 1, 3], dev))
        model.fork([0, 0, 0], [2, 1, 3])
        same(cache, model)
        reserve(cache, model, writers, [1 + 7 * i for i in range(len(writers))])
        same(cache, model)
        assert model.status == 0


@pytest.mark.parametrize("seed", range(6))
def test_random_walk(dev, seed):
    rng = random.Random(seed)
    ps, seqs, max_pages = rng.choice((16, 32)), 12, 6
    cache, model = pair(dev, 37, ps, seqs, max_pages)
    for step in range(40):
        op = rng.choice(("reserve", "reserve", "reserve", "fork", "truncate", "free", "compact"))
        print(f"[walk] seed={seed} step={step} {op}", flush=True)
        some = rng.sample(range(seqs), rng.randrange(1, 6))
        if op == "reserve":
            reserve(cache, model, some, [rng.choice((0, 1, 1, ps, rng.randrange(3 * ps))) for _ in some])
        elif op == "fork":
            src = [rng.randrange(seqs) for _ in some]
            cache.fork(i32(src, dev), i32(some, dev))
            model.fork(src, some)
        elif op == "truncate":
            keep = [rng.randrange(model.lengths[s] + 1) for s in some]
            cache.truncate(i32(some, dev), i32(keep, dev))
            model.truncate(some, keep)
        elif op == "free":
            cache.free(i32(some[:2], dev))
            model.truncate(some[:2])
        else:
            assert int(cache.compact().item()) == model.compact()
        same(cache, model)
        cache._status.zero_()
        model.status = 0


def test_reserve_is_all_or_nothing(dev):
    cache, model = pair(dev, 9, 16, 4, 8)
    reserve(cache, model, [0, 1], [40, 20])
    for seqs, counts, bit in (([2, 3], [48, 17], _lib.STATUS_NO_PAGES), ([0, 0], [1, 1], _lib.STATUS_BAD_SEQUENCE),
                              ([2, 4], [1, 1], _lib.STATUS_BAD_SEQUENCE), ([-1, 2], [1, 1], _lib.STATUS_BAD_SEQUENCE),
                              ([2, 0], [1, 100], _lib.STATUS_BAD_POSITION)):
        reserve(cache, model, seqs, counts)
        same(cache, model)
        assert model.status == bit | HELD
        with pytest.raises(_lib.Q4DecError):
            cache.raise_for_status("reserve")
        model.status = 0
    reserve(cache, model, [7, 2, -3], [0, 64, 0])  # no new tokens: passed over whatever the row is
    same(cache, model)
    # counts that cannot be: decreasing starts, past the token rows, past max_new
    for starts, tokens, most in (([0, 5, 3], 8, 8), ([0, 4, 9], 8, 8), ([0, 6, 7], 8, 5), ([-2, 1, 2], 8, 8)):
        cache.reserve(RaggedBatch(i32([2, 3], dev), i32(starts, dev), tokens, most))
        model.status = _lib.STATUS_BAD_SEQUENCE | HELD
        same(cache, model)
        cache._status.zero_()
    # a partly filled last page whose entry is outside the pool
    for bad in (-1, 9, 2 ** 31 - 1):
        cache.table[0, 2] = bad
        model.table[0][2] = bad
        model.status = 0
        cache._status.zero_()
        reserve(cache, model, [3, 0], [1, 1])
        same(cache, model)
        assert model.status == _lib.STATUS_BAD_PAGE | HELD


def test_fork_and_truncate_leave_out_what_cannot_be(dev):
    cache, model = pair(dev, 20, 16, 8, 4)
    reserve(cache, model, [0, 1, 2], [20, 33, 5])
    src, dst = [0, 0, 1, 9, 0, 3, 1, -1], [3, 3, 2, 4, -1, 5, 0, 6]   # 3 twice, 2 and 0 not empty, 3 -> 5: 3 is a target
    cache.fork(i32(src, dev), i32(dst, dev))
    model.fork(src, dst)
    same(cache, model)
    assert model.status == _lib.STATUS_BAD_SEQUENCE
    model.status = 0
    cache._status.zero_()
    seqs, keep = [1, 1, 0, 8, 2, -1, 7], [20, 3, 21, 0, -1, 0, 0]
    cache.truncate(i32(seqs, dev), i32(keep, dev))
    model.truncate(seqs, keep)
    same(cache, model)
    cache.table[0, 1] = model.table[0][1] = 20
    cache.fork(i32([0], dev), i32([6], dev))
    model.fork([0], [6])
    same(cache, model)
    cache.free(i32([0], dev))
    model.truncate([0])
    same(cache, model)
    assert model.status & _lib.STATUS_BAD_PAGE


def test_large_pool_and_many_sequences(dev):
    """More pages than one round of the block's scan, more sequences than threads, and 2^16 rows."""
    cache, model = pair(dev, 5000, 16, 65536, 40, layers=1, kvh=1)
    seqs = [(7919 * i) % 65536 for i in range(1500)]
    counts = [1 + (37 * i) % 50 for i in range(1500)]
    reserve(cache, model, seqs, counts)
    same(cache, model, rows=False)
    cache.free(i32(seqs[::3], dev))
    model.truncate(seqs[::3])
    reserve(cache, model, [65535, 0], [500, 640])
    same(cache, model, rows=False)
    assert int(cache.compact().item()) == model.compact()
    same(cache, model)


def test_empty_lists_and_full_rows(dev):
    cache, model = pair(dev, 4, 16, 2, 4)
    cache.fork(i32([], dev), i32([], dev))
    cache.free(i32([], dev))
    assert int(cache.compact().item()) == 0
    reserve(cache, model, [1], [64])      # the last page, the last position
    same(cache, model)
    reserve(cache, model, [1], [1])
    same(cache, model)
    assert model.status == _lib.STATUS_BAD_POSITION | HELD
    assert int(cache.compact().item()) == 4


def test_pages_in_a_captured_graph(dev):
    """fork, reserve and truncate of one captured step, replayed on other sequences."""
    cache, model = pair(dev, 64, 16, 10, 6)
    reserve(cache, model, [0, 1], [21, 30])
    src, dst, keep = i32([0, 1], dev), i32([2, 3], dev), i32([2, 3], dev)
    batch = RaggedBatch.of([2, 0, 3, 1], [1, 1, 1, 1], dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        cache.fork(src, dst)
        cache.reserve(batch)
        cache.free(keep)
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c, d in ((0, 1, 2, 3), (1, 0, 5, 4), (0, 1, 9, 8), (1, 0, 2, 3)):
        src.copy_(i32([a, b], dev))
        dst.copy_(i32([c, d], dev))
        keep.copy_(i32([d, c], dev))
        batch.seqs.copy_(i32([c, a, d, b], dev))
        g.replay()
        model.fork([a, b], [c, d])
        model.reserve([c, a, d, b], [1, 1, 1, 1])
        model.truncate([d, c])
        same(cache, model)
    assert model.status == 0


def test_more_pages_at_once_than_are_listed_at_a_time(dev):
    """One call takes 20,000 pages of 45,000, between pages that are held: several lists of 16,384."""
    cache, model = pair(dev, 45000, 16, 64, 600, layers=1, kvh=1)
    reserve(cache, model, list(range(20)), [16 * 300 + i for i in range(20)])
    cache.free(i32(list(range(0, 20, 3)), dev))
    model.truncate(list(range(0, 20, 3)))
    cache.fork(i32([1, 2], dev), i32([60, 61], dev))
    model.fork([1, 2], [60, 61])
    reserve(cache, model, [60] + list(range(20, 56)) + [61], [16 * 40] + [16 * 560 - i for i in range(36)] + [5])
    same(cache, model, rows=False)
    assert model.status == 0 and sum(r != 0 for r in model.refs) > 20000 + 3600
    reserve(cache, model, [0, 56], [9000, 9600])
    same(cache, model)


@pytest.mark.parametrize("rows", [300, 1365, 2048])
def test_many_shared_last_pages(dev, rows):
    """Every sequence of the batch shares its last page: with one that writes too, with one that does not, or
    with both."""
    cache, model = pair(dev, 4 * rows, 16, 3 * rows, 3, layers=1, kvh=1)
    first = list(range(rows))
    reserve(cache, model, first, [1 + i % 15 for i in first])
    second = [rows + i for i in first]
    cache.fork(i32(first, dev), i32(second, dev))
    model.fork(first, second)
    third = first[::3]
    cache.fork(i32(third, dev), i32([2 * rows + i for i in third], dev))
    model.fork(third, [2 * rows + i for i in third])
    both = [s for i in first for s in ((i, rows + i) if i % 2 else (rows + i, i))]
    reserve(cache, model, both, [1] * len(both))
    same(cache, model)
    assert model.status == 0
