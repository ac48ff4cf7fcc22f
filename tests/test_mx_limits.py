"""How many rows mx_score takes: 2^23, and no more tiles of 64 rows x 256 tokens than a launch has (2^23), which a
workspace is asked for in vain as well: it is refused before anything of that size is allocated."""

import ctypes

import pytest
import torch

from llm_accelerator_amd import _lib
from llm_accelerator_amd._lib import Q4dMX

FAKE = 0x7F0000000000  # aligned, never dereferenced: validation fails before launch
F16, SHAPE = 0, -11
# (tokens, columns, most rows): 2^23 rows, 2^23 tiles, and 32768 tiles of 256 tokens (256 of 64 rows)
LIMITS = [(48, 64, 1 << 23), (16384, 32, 1 << 23), (16385, 32, (1 << 23) // 65 * 64), (151936, 1024, 903808), (32768 * 256, 128, 16384)]


@pytest.mark.parametrize("vocab,cols,most", LIMITS)
def test_the_workspace_is_refused_with_the_score(vocab, cols, most):
    lib = _lib.load()
    size = lib.q4d_mx_score_workspace_bytes
    assert size(vocab, cols, most) > 0
    w = ctypes.byref(Q4dMX(FAKE, FAKE, vocab, cols))
    for m in (most + 1, 2 * most, 2 ** 31 - 1):
        assert size(vocab, cols, m) == 0
        assert lib.q4d_mx_score(w, FAKE, F16, cols, m, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 60, None) == SHAPE


@pytest.mark.gpu
def test_refused_before_its_memory_is_asked_for(dev):
    from llm_accelerator_amd.mx import MXTensor, mx_score
    head = MXTensor(torch.zeros(151936, 16, dtype=torch.uint8, device=dev), torch.full((151936, 1), 127, dtype=torch.uint8, device=dev))
    x = torch.zeros(903809, 32, device=dev, dtype=torch.float16)
    t = torch.zeros(903809, device=dev, dtype=torch.int32)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="rows"):
        mx_score(x, head, t)
    assert torch.cuda.max_memory_allocated() - before < 1 << 26  # the workspace would be 8.6 GB


@pytest.mark.gpu
def test_the_most_rows_of_a_head(dev):
    """903808 rows of 151936 tokens, 2^23 tiles but for 140.  Every product of a row is 0 but that of one token, a power
    of two times the row's only value: what the score is follows from 151936 alone.  The products are exact, so the
    bound is the softmax's: log sum e^z is off by (H + 402) 2^-23 (an exponential by (|d| + 2) 2^-23 of itself, a
    term passes at most 400 additions and rescalings), the mean t / l of |z - max| <= H - best by twice that of
    H - best + 1; 2^-22 of 1 + the result for the subtractions and the result's own rounding."""
    import math

    from llm_accelerator_amd.mx import MXTensor, mx_score
    vocab, rows = 151936, 903808
    packed = torch.zeros(vocab, 16, dtype=torch.uint8, device=dev)
    packed[150001, 0] = 4  # 2 in column 0
    head = MXTensor(packed, torch.full((vocab, 1), 127, dtype=torch.uint8, device=dev))
    x = torch.zeros(rows, 32, device=dev, dtype=torch.float16)
    value = torch.arange(rows, device=dev) % 4
    x[:, 0] = value.half()  # z: 0, 2, 4, 6
    t = torch.where(torch.arange(rows, device=dev) % 3 == 0, 150001, 7).int()
    got = mx_score(x, head, t)
    for v in range(4):
        lse = math.log(vocab - 1 + math.exp(2 * v))
        best, h = 2 * v - lse, lse - math.exp(2 * v - lse) * 2 * v
        off, step = (h + 402) * 2.0 ** -23, 2.0 ** -22
        mine = value == v
        assert (got.entropy[mine].double() - h).abs().max().item() <= off + 2 * off * (h - best + 1) + step * (h + 1)
        assert (got.best[mine].double() - best).abs().max().item() <= off + step * (1 - best)
        want = torch.where(t[mine] == 7, -lse, best).double()
        assert (got.logprob[mine].double() - want).abs().max().item() <= off + step * (1 + lse)
