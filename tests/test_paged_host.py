"""The paged cache without a device: what the entry points refuse before any launch, the checks of
batches and pages that the kernels share with the host, and the rotation tables."""

import ctypes
import math
import subprocess
import tempfile
from functools import lru_cache
from pathlib import Path

import pytest
import torch

from llm_accelerator_amd import _lib, paged
from llm_accelerator_amd._lib import Q4dPages, Q4dRagged, Q4dRope

ROOT = Path(__file__).resolve().parents[1]
ROCM = Path("/opt/rocm")
FAKE = 0x7F0000000000  # aligned, never dereferenced: validation fails before launch
NULL, ADDR, CAPACITY, LAYER, SHAPE, DTYPE = -7, -4, -9, -2, -11, -13


def pages(**kw):
    d = dict(data=FAKE, dtype=0, num_layers=2, num_pages=40, num_kv_heads=8, page_size=64, head_dim=128, table=FAKE,
             lengths=FAKE, refs=FAKE, num_seqs=4, max_pages=16, status=FAKE)
    return Q4dPages(**{**d, **kw})


def ragged(**kw):
    return Q4dRagged(**{**dict(seqs=FAKE, starts=FAKE, n=4, tokens=10, max_new=10), **kw})


BAD_PAGES = [(dict(data=None), NULL), (dict(table=None), NULL), (dict(lengths=None), NULL), (dict(refs=None), NULL),
             (dict(status=None), NULL), (dict(dtype=1), DTYPE), (dict(dtype=9), DTYPE), (dict(page_size=8), SHAPE),
             (dict(page_size=48), SHAPE), (dict(page_size=512), SHAPE), (dict(head_dim=96), SHAPE),
             (dict(num_layers=0), SHAPE), (dict(num_pages=0), SHAPE), (dict(num_pages=(1 << 22) + 1), SHAPE),
             (dict(num_kv_heads=257), SHAPE), (dict(num_seqs=65537), SHAPE), (dict(max_pages=0), SHAPE),
             (dict(max_pages=(1 << 18) + 1), SHAPE), (dict(data=FAKE + 8), ADDR), (dict(table=FAKE + 2), ADDR)]
BAD_BATCH = [(dict(starts=None), NULL), (dict(n=0), SHAPE), (dict(n=4097), SHAPE), (dict(tokens=0), SHAPE),
             (dict(tokens=(1 << 24) + 1), SHAPE), (dict(max_new=0), SHAPE), (dict(starts=FAKE + 2), ADDR),
             (dict(seqs=FAKE + 1), ADDR)]


def calls(lib, p, r):
    """Every entry point on these descriptors, with the other arguments in order."""
    big = 1 << 40
    p, r = ctypes.byref(p), ctypes.byref(r)
    return {
        "reserve": lambda: lib.q4d_pages_reserve(p, r, FAKE, big, None),
        "append": lambda: lib.q4d_paged_append(p, 0, r, FAKE, 2048, 16, FAKE, 1024, FAKE, 1024, 0, None, None, 1e-6,
                                               None, FAKE, None),
        "attention": lambda: lib.q4d_paged_attention(p, 0, r, FAKE, 2048, 16, 0.1, FAKE, 2048, FAKE, big, None),
        "fork": lambda: lib.q4d_pages_fork(p, FAKE, FAKE, 1, None),
        "truncate": lambda: lib.q4d_pages_truncate(p, FAKE, None, 1, None),
        "compact": lambda: lib.q4d_pages_compact(p, None, FAKE, big, None),
    }


@pytest.mark.parametrize("change,code", BAD_PAGES, ids=lambda v: str(v))
def test_bad_cache_descriptors_are_refused(change, code):
    lib = _lib.load()
    p = pages(**change)
    for name, call in calls(lib, p, ragged()).items():
        assert call() == code, name
    assert lib.q4d_pages_workspace_bytes(ctypes.byref(p)) == 0
    assert lib.q4d_paged_attention_workspace_bytes(ctypes.byref(p), 16, 4, 10, 10) == 0


@pytest.mark.parametrize("change,code", BAD_BATCH, ids=lambda v: str(v))
def test_bad_batches_are_refused(change, code):
    made = calls(_lib.load(), pages(), ragged(**change))
    for name in ("reserve", "append", "attention"):
        assert made[name]() == code, name


@pytest.mark.parametrize("arg,value,code", [
    (1, -1, LAYER), (1, 2, LAYER), (3, None, NULL), (15, None, NULL), (6, None, NULL), (8, None, NULL), (10, 7, DTYPE),
    (5, 0, SHAPE), (5, 4097, SHAPE), (4, 2047, SHAPE), (7, 1000, SHAPE), (9, 1 << 33, SHAPE), (4, 2050, ADDR),
    (7, 1025, ADDR), (3, FAKE + 4, ADDR), (6, FAKE + 8, ADDR), (8, FAKE + 2, ADDR), (11, FAKE + 4, ADDR),
    (15, FAKE + 8, ADDR)])
def test_append_refuses(arg, value, code):
    args = [ctypes.byref(pages()), 0, ctypes.byref(ragged()), FAKE, 2048, 16, FAKE, 1024, FAKE, 1024, 0, None, None,
            1e-6, None, FAKE, None]
    args[arg] = value
    assert _lib.load().q4d_paged_append(*args) == code


def test_append_without_q_takes_no_heads():
    args = [ctypes.byref(pages()), 0, ctypes.byref(ragged()), None, 0, 16, FAKE, 1024, FAKE, 1024, 0, None, None, 1e-6,
            None, None, None]
    assert _lib.load().q4d_paged_append(*args) == SHAPE


@pytest.mark.parametrize("change,code", [
    (dict(cos=None), NULL), (dict(sin=None), NULL), (dict(max_ctx=0), SHAPE), (dict(rotary_dim=24), SHAPE),
    (dict(rotary_dim=0), SHAPE), (dict(rotary_dim=144), SHAPE), (dict(interleaved=2), SHAPE), (dict(cos=FAKE + 4), ADDR)])
def test_append_refuses_rotations(change, code):
    rope = Q4dRope(**{**dict(cos=FAKE, sin=FAKE, max_ctx=64, rotary_dim=128, interleaved=0), **change})
    assert _lib.load().q4d_paged_append(ctypes.byref(pages()), 0, ctypes.byref(ragged()), FAKE, 2048, 16, FAKE, 1024,
                                        FAKE, 1024, 0, None, None, 1e-6, ctypes.byref(rope), FAKE, None) == code


@pytest.mark.parametrize("arg,value,code", [
    (1, 2, LAYER), (1, -1, LAYER), (3, None, NULL), (7, None, NULL), (9, None, NULL), (5, 12, SHAPE), (5, 0, SHAPE),
    (5, 136, SHAPE), (4, 2040, SHAPE), (8, 2040, SHAPE), (8, 1 << 33, SHAPE), (4, 2052, ADDR), (8, 2049, ADDR),
    (3, FAKE + 8, ADDR), (7, FAKE + 2, ADDR), (9, FAKE + 128, ADDR), (10, 16, CAPACITY), (6, float("nan"), SHAPE),
    (6, float("inf"), SHAPE)])
def test_attention_refuses(arg, value, code):
    args = [ctypes.byref(pages()), 0, ctypes.byref(ragged()), FAKE, 2048, 16, 0.1, FAKE, 2048, FAKE, 1 << 40, None]
    args[arg] = value
    assert _lib.load().q4d_paged_attention(*args) == code


def test_more_blocks_than_a_launch_has_are_refused():
    lib = _lib.load()
    p = pages(num_kv_heads=256, head_dim=64)
    r = ragged(tokens=1 << 24, max_new=1 << 24)
    p, r, big, wide = ctypes.byref(p), ctypes.byref(r), 1 << 40, 4096 * 64
    assert lib.q4d_paged_attention(p, 0, r, FAKE, wide, 4096, 0.1, FAKE, wide, FAKE, big, None) == SHAPE
    assert lib.q4d_paged_append(p, 0, r, FAKE, wide, 4096, FAKE, wide, FAKE, wide, 0, None, None, 1e-6, None, FAKE,
                                None) == SHAPE


def test_page_calls_refuse():
    lib, p, r = _lib.load(), ctypes.byref(pages()), ctypes.byref(ragged())
    need = lib.q4d_pages_workspace_bytes(p)
    assert need >= 4 * 3 * (40 + 4096)
    assert lib.q4d_pages_reserve(p, r, None, need, None) == NULL
    assert lib.q4d_pages_reserve(p, r, FAKE + 4, need, None) == ADDR
    assert lib.q4d_pages_reserve(p, r, FAKE, need - 1, None) == CAPACITY
    assert lib.q4d_pages_compact(p, None, FAKE, need - 1, None) == CAPACITY
    assert lib.q4d_pages_compact(p, FAKE + 2, FAKE, need, None) == ADDR
    assert lib.q4d_pages_fork(p, None, FAKE, 1, None) == NULL
    assert lib.q4d_pages_fork(p, FAKE, FAKE, 0, None) == SHAPE
    assert lib.q4d_pages_fork(p, FAKE, FAKE, 65537, None) == SHAPE
    assert lib.q4d_pages_fork(p, FAKE + 2, FAKE, 1, None) == ADDR
    assert lib.q4d_pages_truncate(p, None, FAKE, 1, None) == NULL
    assert lib.q4d_pages_truncate(p, FAKE, FAKE + 1, 1, None) == ADDR
    assert lib.q4d_pages_truncate(p, FAKE, None, -1, None) == SHAPE
    assert lib.q4d_paged_attention_workspace_init(None, 256, None) == NULL
    assert lib.q4d_paged_attention_workspace_init(FAKE + 16, 256, None) == ADDR
    for bad in ((15, 4, 10, 10), (136, 4, 10, 10), (16, 0, 10, 10), (16, 4097, 10, 10), (16, 4, 0, 1), (16, 4, 10, 0)):
        assert lib.q4d_paged_attention_workspace_bytes(p, *bad) == 0, bad


# ---------------------------------------------------------------- device-side checks, on the host
SHIM = r"""
#include "q4d_paged.h"
using namespace q4d;
extern "C" {
int shim_seq_count(int s0, int s1, int tokens, int max_new) { return seq_count(s0, s1, tokens, max_new); }
// out: row, first, count, len
void shim_seq_span(int32_t* lengths, int num_seqs, int max_pages, int shift, const int32_t* seqs, const int32_t* starts,
                   int n, int tokens, int max_new, int b, int* out) {
  PagedView p = {};
  p.lengths = lengths; p.num_seqs = num_seqs; p.max_pages = max_pages; p.page_shift = shift;
  const SeqSpan s = seq_span(p, RaggedView{seqs, starts, n, tokens, max_new}, b);
  out[0] = s.row; out[1] = s.first; out[2] = s.count; out[3] = s.len;
}
int shim_in_range(int i, int n) { return in_range(i, n); }
size_t shim_page_elem(int num_pages, int kvh, int d, int shift, int page, int j) {
  PagedView p = {};
  p.num_pages = num_pages; p.kvh = kvh; p.d = d; p.page_shift = shift;
  return page < 0 ? plane_elems(p) : page_elem(p, page, j);
}
}
"""


@lru_cache(maxsize=None)
def shim():
    with tempfile.TemporaryDirectory() as d:
        src, so = Path(d) / "shim.cpp", Path(d) / "shim.so"
        src.write_text(SHIM)
        subprocess.run([str(ROCM / "llvm/bin/clang++"), "-shared", "-fPIC", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__",
                        f"-I{ROOT / 'llm_accelerator_amd' / 'csrc'}", f"-I{ROCM / 'include'}", str(src), "-o", str(so)],
                       check=True)
        lib = ctypes.CDLL(str(so))
    lib.shim_page_elem.restype = ctypes.c_size_t
    return lib


def span(lengths, seqs, starts, b, tokens=100, max_new=100, max_pages=10, shift=4):
    out = (ctypes.c_int * 4)()
    arr = lambda v: None if v is None else (ctypes.c_int32 * len(v))(*v)  # noqa: E731
    shim().shim_seq_span(arr(lengths), len(lengths), max_pages, shift, arr(seqs), arr(starts), len(starts) - 1, tokens,
                         max_new, b, out)
    return list(out)


def test_counts_that_cannot_be():
    f = shim().shim_seq_count
    assert f(0, 5, 5, 5) == 5 and f(3, 3, 5, 5) == 0 and f(5, 5, 5, 1) == 0
    for bad in ((-1, 3, 5, 5), (4, 3, 5, 5), (0, 6, 5, 9), (0, 5, 5, 4), (-2 ** 31, 2 ** 31 - 1, 5, 5),
                (2 ** 31 - 1, -2 ** 31, 5, 5), (6, 6, 5, 5)):
        assert f(*bad) == -1, bad


def test_spans_of_a_batch():
    assert span([7, 30], [1, 0], [0, 4, 9], 0) == [1, 0, 4, 30]
    assert span([7, 30], None, [0, 4, 9], 1) == [1, 4, 5, 30]
    assert span([7, 30], [-5, 0], [3, 3, 9], 0)[2] == 0          # no new tokens: whatever the row is
    for bad in (span([7, 30], [2, 0], [0, 4, 9], 0), span([7, 30], [-1, 0], [0, 4, 9], 0),  # a row that is none
                span([7, 30], [0, 1], [0, 8, 9], 0),              # fewer positions than new tokens
                span([161, 30], [0, 1], [0, 8, 9], 0),            # more positions than the table holds
                span([-1, 30], [0, 1], [0, 8, 9], 0), span([7, 30], [1, 0], [4, 2, 9], 0),
                span([7, 30], [1, 0], [0, 4, 9], 0, tokens=3), span([7, 30], [1, 0], [0, 4, 9], 0, max_new=3)):
        assert bad[2] < 0


def test_page_ranges_and_offsets_past_32_bits():
    assert [shim().shim_in_range(i, 4) for i in (-1, 0, 3, 4, -2 ** 31, 2 ** 31 - 1)] == [0, 1, 1, 0, 0, 0]
    big = 1 << 22
    assert shim().shim_page_elem(big, 8, 128, 8, -1, 0) == big * 8 * 128 * 256
    assert shim().shim_page_elem(big, 8, 128, 8, big - 1, 7) == ((big - 1) * 8 + 7) * 256 * 128


# ---------------------------------------------------------------- rotation tables
def test_rope_angles_are_exact_at_far_positions():
    cos, sin = paged.rope_angles(128, 32768, 1e6)
    for pos, i in ((0, 0), (1, 0), (32767, 0), (32767, 1), (30011, 17), (32767, 63)):
        angle = pos * 1e6 ** (-2 * i / 128)
        # the 64-bit angle is off by its own rounding (2^-53 of 32767), the fp32 result by half a step
        assert abs(cos[pos, i].item() - math.cos(angle)) <= 2 ** -25 + 2e-11
        assert abs(sin[pos, i].item() - math.sin(angle)) <= 2 ** -25 + 2e-11


def angles(**kw):
    inv, factor = paged._inv_freq(64, 1e4, kw or None)
    return inv, factor


def test_rope_scaling_rules():
    plain, one = angles()
    assert one == 1.0
    linear, f = angles(type="linear", factor=4)
    assert f == 1.0 and torch.allclose(linear, plain / 4, rtol=1e-15)
    ntk, f = angles(type="ntk", factor=4)
    assert f == 1.0 and ntk[0] == 1.0 and abs(ntk[-1] / plain[-1] - 0.25) < 1e-14
    yarn, f = angles(type="yarn", factor=4, original_max_ctx=2048)
    assert abs(f - (0.1 * math.log(4) + 1)) < 1e-15
    ratio = yarn / plain
    turns = 2048 * plain / (2 * math.pi)
    assert bool((ratio[turns > 40] == 1).all()) and bool(((ratio[turns < 0.8] - 0.25).abs() < 1e-14).all())
    assert bool((ratio[1:] <= ratio[:-1] + 1e-15).all())
    for kind in ("linear", "ntk", "yarn"):
        same, f = angles(type=kind, factor=1, original_max_ctx=2048)
        assert f == 1.0 and torch.allclose(same, plain, rtol=1e-14)


def test_python_arguments_are_checked():
    for bad in (dict(rotary_dim=20, max_ctx=8, theta=1e4), dict(rotary_dim=16, max_ctx=0, theta=1e4),
                dict(rotary_dim=16, max_ctx=8, theta=1.0)):
        with pytest.raises(ValueError):
            paged.rope_angles(**bad)
    with pytest.raises(ValueError):
        paged.rope_angles(16, 8, 1e4, {"type": "other", "factor": 2})
    with pytest.raises(ValueError):
        paged.rope_angles(16, 8, 1e4, {"type": "linear", "factor": 0.5})
    with pytest.raises(ValueError):
        paged.RaggedBatch(None, torch.zeros(3, dtype=torch.int32), 4, 1)
    with pytest.raises(ValueError):
        paged.RaggedBatch.of([0, 1], [1])
    with pytest.raises(ValueError):
        paged.RaggedBatch.of([0, 1], [1, -1])
    with pytest.raises(ValueError):
        paged.RopeTable(torch.zeros(4, 8), torch.zeros(4, 8))
    with pytest.raises(ValueError):
        paged.PagedKVCache(1, 4, 16, 2, 64, 2, 64, device="cpu")


def test_status_names():
    assert _lib.status_names(16 | 32 | 64 | 128) == ["NO_PAGES", "BAD_SEQUENCE", "BAD_PAGE", "NOT_RESERVED"]
    assert _lib.status_names(256) == ["UNKNOWN"]


def test_calls_run_on_the_cache_s_device(monkeypatch):
    """On another current device: the cache's is made current for the call, with its own stream, and the
    caller's again afterwards, whether the call succeeds, fails or raises."""
    cache = paged.PagedKVCache.__new__(paged.PagedKVCache)
    cache._index = 3
    now, log = [0], []
    monkeypatch.setattr(paged, "_device", lambda: now[0])
    monkeypatch.setattr(paged, "_stream", lambda i: 100 + i)
    monkeypatch.setattr(torch.cuda, "set_device", lambda i: now.__setitem__(0, i))

    class Lib:
        def q4d_some_call(self, *args):
            log.append((now[0], args))
            if args[0] == "raise":
                raise TypeError
            return args[0]
    cache._lib = Lib()
    for here in (0, 3):
        now[0] = here
        cache._call("q4d_some_call", 0, "x")
        assert log[-1] == (3, (0, "x", 103)) and now[0] == here
        with pytest.raises(_lib.Q4DecError):
            cache._call("q4d_some_call", SHAPE)
        assert now[0] == here
        with pytest.raises(TypeError):
            cache._call("q4d_some_call", "raise")
        assert now[0] == here
