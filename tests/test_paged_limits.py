"""What the paged cache's entry points refuse about sizes, without a device."""

import ctypes

import pytest

from llm_accelerator_amd import _lib
from llm_accelerator_amd.paged import RaggedBatch
from test_paged_host import SHAPE, calls, pages, ragged


@pytest.mark.parametrize("max_ctx", [-1, 16 * 64 + 1, 2 ** 31 - 1])
def test_a_max_ctx_past_the_table_is_refused(max_ctx):
    lib, p = _lib.load(), pages(max_ctx=max_ctx)
    for name, call in calls(lib, p, ragged()).items():
        assert call() == SHAPE, name
    assert lib.q4d_pages_workspace_bytes(ctypes.byref(p)) == 0


@pytest.mark.parametrize("max_ctx", [0, 1, 1000, 16 * 64])
def test_a_max_ctx_within_the_table_is_taken(max_ctx):
    assert _lib.load().q4d_pages_workspace_bytes(ctypes.byref(pages(max_ctx=max_ctx))) > 0


def test_a_batch_has_rows_for_its_tokens():
    for counts, tokens in (([3, 4], 6), ([1], 0), ([0, 9], -1)):
        with pytest.raises(ValueError):
            RaggedBatch.of(list(range(len(counts))), counts, tokens=tokens)
