"""Steps of a paged cache at their borders: rows of a length that is no multiple of the page, and steps that are
refused while others are on their way."""

import pytest
import torch

from llm_accelerator_amd import _lib
from llm_accelerator_amd.paged import PagedKVCache, RaggedBatch, RopeTable

pytestmark = pytest.mark.gpu
F = torch.float16


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def state(cache):
    return [x.clone() for x in (cache.data, cache.table, cache.lengths, cache.refs)]


def unchanged(cache, before):
    return all(torch.equal(a, b) for a, b in zip(state(cache), before))


@pytest.mark.parametrize("max_ctx,ps", [(100, 64), (1, 16), (129, 128), (128, 64)])
def test_rows_end_at_max_ctx(dev, max_ctx, ps):
    """Not at the end of the last page: the step that would pass it is refused as a whole, before a rotation that
    covers max_ctx runs out and leaves positions unwritten."""
    made = PagedKVCache(1, 9, ps, 2, 64, 3, max_ctx, F, dev)
    assert made.max_ctx == max_ctx and made.max_pages == -(-max_ctx // ps)
    over = PagedKVCache.over(made.data.clone(), made.table.clone(), made.lengths.clone(), made.refs.clone(), max_ctx)
    rope = RopeTable.build(64, max_ctx, device=dev)
    for cache in (made, over):
        def step(seqs, counts):
            batch = RaggedBatch.of(seqs, counts, dev)
            x = torch.randn(batch.tokens, 4, 64, device=dev)
            cache.reserve(batch)
            cache.append(0, batch, None, x[:, :2], x[:, 2:], rope)
        step([1, 0], [max_ctx, 1])
        assert cache.status() == 0 and cache.lengths.tolist() == [1, max_ctx, 0]
        before = state(cache)
        for seqs, counts in (([1], [1]), ([2, 1], [1, 1]), ([2], [max_ctx + 1])):
            step(seqs, counts)
            assert cache.status() == _lib.STATUS_BAD_POSITION | _lib.STATUS_NOT_RESERVED and unchanged(cache, before)
            cache._status.zero_()
        step([2], [max_ctx])
        assert cache.status() == 0 and cache.lengths.tolist() == [1, max_ctx, max_ctx]
    room = PagedKVCache.over(made.data, made.table, made.lengths, made.refs)
    assert room.max_ctx == made.max_pages * ps
    for bad in (0, -1, room.max_ctx + 1):
        with pytest.raises(ValueError):
            PagedKVCache.over(made.data, made.table, made.lengths, made.refs, bad)


def test_page_calls_run_on_after_a_refused_reserve(dev):
    """A captured step of fork, reserve, append and free, launched ahead: after the refusal nothing is written
    into a page and no length grows, but forks and frees are carried out, since freeing is what makes room."""
    cache = PagedKVCache(1, 5, 16, 2, 64, 6, 64, F, dev)
    first = RaggedBatch.of([0, 1], [17, 20], dev)          # two pages each, one is free
    cache.reserve(first)
    src, dst, gone = i32([0], dev), i32([2], dev), i32([5], dev)
    batch = RaggedBatch.of([2], [1], dev)
    x = torch.randn(1, 4, 64, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        cache.fork(src, dst)
        cache.reserve(batch)
        cache.append(0, batch, None, x[:, :2], x[:, 2:])
        cache.free(gone)
    torch.cuda.current_stream().wait_stream(side)
    g.replay()                                             # takes the last page for the fork's own copy
    assert cache.status() == 0 and cache.lengths.tolist() == [17, 20, 18, 0, 0, 0]
    data = cache.data.clone()
    for s, d, r in ((1, 3, 5), (2, 4, 1)):                 # no page for the fork of 1; then all is held back
        src.copy_(i32([s], dev))
        dst.copy_(i32([d], dev))
        gone.copy_(i32([r], dev))
        batch.seqs.copy_(i32([d], dev))
        g.replay()
    assert cache.status() == _lib.STATUS_NO_PAGES | _lib.STATUS_NOT_RESERVED
    assert torch.equal(cache.data, data)
    assert cache.lengths.tolist() == [17, 0, 18, 20, 18, 0]   # 3 and 4 are forks that have not grown, 1 is gone
    assert cache.refs.sum().item() == 2 + 2 + 2 + 2
    with pytest.raises(_lib.Q4DecError):
        cache.raise_for_status("step")
    cache.free(i32([0, 2], dev))
    batch.seqs.copy_(i32([3], dev))
    cache.reserve(batch)
    assert cache.status() == 0 and cache.lengths.tolist() == [0, 0, 0, 21, 18, 0]
