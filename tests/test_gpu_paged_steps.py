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
