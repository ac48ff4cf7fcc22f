"""Paged KV cache: many sequences in pages of one pool, and ragged batches over them.

No counterpart in the reference, whose cache is one tensor per sequence
(``Qwen3-0.6B-Base/python_each_module/common.py:186-189``); the operators stand beside
``append_cache`` and ``manual_cached_attention`` of :mod:`.common`:

* :class:`PagedKVCache` -- the pool, table, lengths and page counts on the device, with
  :meth:`~PagedKVCache.reserve`, :meth:`~PagedKVCache.fork`, :meth:`~PagedKVCache.truncate` /
  :meth:`~PagedKVCache.free` and :meth:`~PagedKVCache.compact` for the pages, and per layer
  :meth:`~PagedKVCache.append` and :meth:`~PagedKVCache.attention`;
* :class:`RaggedBatch` -- the sequences of a call and their new tokens: chunks of prompts and
  single decode tokens side by side;
* :class:`RopeTable` -- rotation angles: halves or neighbouring pairs, all or part of a head,
  scaled for long contexts.

Every call is launched on torch's current stream of the cache's device, allocates nothing that
outlives it, does not synchronise, and can be captured into a graph.  Arguments that the host can
see are checked (``ValueError`` / :class:`~llm_accelerator_amd._lib.Q4DecError`); what only the
device knows is checked there, left out where it cannot be, and reported by
:meth:`~PagedKVCache.status` (``Q4D_STATUS_*`` bits).
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import Q4D_BF16, Q4D_F16, Q4D_F32, Q4dPages, Q4dRagged, Q4dRope, check

# The device and stream queries of torch.cuda.current_device / current_stream without the objects
# around them: 0.2 us a call instead of 1.6, where a whole call is 6 to 9.
_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream

_DTYPES = {torch.float16: Q4D_F16, torch.bfloat16: Q4D_BF16, torch.float32: Q4D_F32}


def _ints(t: torch.Tensor, name: str, device, n: int | None = None) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise ValueError(f"{name} must be a contiguous int32 tensor{'' if n is None else f' of {n} elements'} on {device}")
    return t


class RaggedBatch:
    """New tokens of several sequences: sequence ``b`` is table row ``seqs[b]`` (``None``: row b), its
    new tokens, its last positions, are rows ``starts[b]`` .. ``starts[b + 1] - 1`` of the token
    tensors.  ``seqs`` [n] and ``starts`` [n + 1] are device int32 and may change between calls (a
    captured step is replayed on other sequences); ``tokens`` is the number of token rows and
    ``max_new`` a bound on a sequence's new tokens (1: a decode step)."""

    def __init__(self, seqs: torch.Tensor | None, starts: torch.Tensor, tokens: int, max_new: int):
        if not starts.is_cuda:
            raise ValueError("starts must be a GPU tensor (libq4dec has no CPU path)")
        n = starts.numel() - 1
        self.starts = _ints(starts, "starts", starts.device)
        self.seqs = None if seqs is None else _ints(seqs, "seqs", starts.device, n)
        if not 1 <= n <= 4096 or not 1 <= int(tokens) <= 1 << 24 or int(max_new) < 1:
            raise ValueError("a batch has 1 .. 4096 sequences, 1 .. 2^24 token rows and max_new >= 1")
        self.n, self.tokens, self.max_new = n, int(tokens), int(max_new)
        self._index = starts.get_device()
        self._desc = Q4dRagged(None if seqs is None else seqs.data_ptr(), starts.data_ptr(), n, self.tokens,
                               min(self.max_new, self.tokens))
        self._ref = ctypes.byref(self._desc)

    @classmethod
    def of(cls, seqs, counts, device="cuda", tokens: int | None = None) -> "RaggedBatch":
        """From host lists: table rows and the new tokens of each; ``tokens`` rows may hold padding."""
        if len(seqs) != len(counts) or not counts or min(counts) < 0:
            raise ValueError("one count of new tokens, zero or more, per sequence")
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + int(c))
        if tokens is not None and tokens < starts[-1]:
            raise ValueError(f"{tokens} token rows for {starts[-1]} new tokens")
        both = torch.tensor([int(s) for s in seqs] + starts, dtype=torch.int32).to(device)
        return cls(both[:len(seqs)], both[len(seqs):], max(1, starts[-1]) if tokens is None else tokens,
                   max(1, max(counts)))


def _inv_freq(rotary_dim: int, theta: float, scaling: dict | None) -> tuple[torch.Tensor, float]:
    """(frequencies in 64 bits, factor of cos and sin)."""
    r = rotary_dim
    freq = torch.arange(0, r, 2, dtype=torch.float64) / r
    inv = theta ** -freq
    if scaling is None:
        return inv, 1.0
    kind, factor = scaling["type"], float(scaling["factor"])
    if factor < 1:
        raise ValueError("scaling factor must be at least 1")
    if kind == "linear":     # positions / factor
        return inv / factor, 1.0
    if kind == "ntk":        # a larger base: the lowest frequency is divided by factor, the highest kept
        return (theta * factor ** (r / (r - 2))) ** -freq if r > 2 else inv / factor, 1.0
    if kind == "yarn":       # by wavelength: long ones divided by factor, short ones kept, a ramp between
        old = float(scaling["original_max_ctx"])
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))

        def dim_of(turns):   # the pair that turns `turns` times over the old context
            return r * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(dim_of(fast)), 0), min(math.ceil(dim_of(slow)), r - 1)
        ramp = ((torch.arange(r // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return inv * (1 - ramp) + inv / factor * ramp, float(scaling.get("attention_factor", 0.1 * math.log(factor) + 1.0))
    raise ValueError(f"unknown rotary scaling {kind!r}: linear, ntk or yarn")


class RopeTable:
    """cos and sin of position x frequency, fp32 [max_ctx, rotary_dim / 2]; dims past ``rotary_dim``
    stay as they are.  Pairs are (i, i + rotary_dim / 2) (``manual_rotate_half``, common.py:148-152)
    or, ``interleaved``, (2 i, 2 i + 1)."""

    def __init__(self, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool = False):
        if (cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32
                or not cos.is_contiguous() or not sin.is_contiguous() or cos.device != sin.device or not cos.is_cuda):
            raise ValueError("cos and sin must be contiguous fp32 GPU tensors [max_ctx, rotary_dim / 2]")
        self.cos, self.sin, self.interleaved = cos, sin, bool(interleaved)
        self.max_ctx, self.rotary_dim, self._index = cos.shape[0], 2 * cos.shape[1], cos.get_device()
        self._desc = Q4dRope(cos.data_ptr(), sin.data_ptr(), self.max_ctx, self.rotary_dim, int(self.interleaved))
        self._ref = ctypes.byref(self._desc)

    @classmethod
    def build(cls, rotary_dim: int, max_ctx: int, theta: float = 1_000_000.0, scaling: dict | None = None,
              interleaved: bool = False, device="cuda") -> "RopeTable":
        """Angles made in 64 bits (far positions lose nothing) and rounded once.  ``scaling``: ``None``,
        ``{"type": "linear" | "ntk", "factor": f}`` or ``{"type": "yarn", "factor": f,
        "original_max_ctx": n}`` (optional ``beta_fast`` 32, ``beta_slow`` 1, ``attention_factor``)."""
        cos, sin = rope_angles(rotary_dim, max_ctx, theta, scaling)
        return cls(cos.to(device), sin.to(device), interleaved)


def rope_angles(rotary_dim: int, max_ctx: int, theta: float, scaling: dict | None = None):
    """(cos, sin) on the host, fp32 [max_ctx, rotary_dim / 2]."""
    if rotary_dim <= 0 or rotary_dim % 16 or max_ctx <= 0 or theta <= 1:
        raise ValueError("rotary_dim must be a multiple of 16, max_ctx positive, theta above 1")
    inv, factor = _inv_freq(rotary_dim, float(theta), scaling)
    angle = torch.arange(max_ctx, dtype=torch.float64)[:, None] * inv
    return (angle.cos() * factor).float().contiguous(), (angle.sin() * factor).float().contiguous()


class PagedWorkspace:
    """Scratch of :meth:`PagedKVCache.attention`.  Calls that may overlap (two streams, two captured
    graphs replayed side by side) need one each."""

    def __init__(self, cache: "PagedKVCache", q_heads: int, n: int, tokens: int, max_new: int):
        self.nbytes = int(_lib.load().q4d_paged_attention_workspace_bytes(cache._ref, q_heads, n, tokens,
                                                                          min(max_new, tokens)))
        if self.nbytes == 0:
            raise _lib.Q4DecError(-11, "q4d_paged_attention_workspace_bytes")
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=cache.device)
        self.ptr, self._index = self.buf.data_ptr(), cache._index
        cache._call("q4d_paged_attention_workspace_init", self.ptr, self.nbytes)


class PagedKVCache:
    """Pool [layers][K, V][pages][kv heads][page size][head dim] (fp16 or bf16), ``table`` [rows, max
    pages], ``lengths`` [rows] and ``refs`` [pages] (int32, on the device).  A sequence grows to
    ``max_ctx`` positions at most (a table of angles should have as many).  Calls that change a cache
    must not overlap each other or calls that read it."""

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 num_seqs: int, max_ctx: int, dtype=torch.float16, device="cuda"):
        kw = dict(dtype=torch.int32, device=device)
        self._setup(torch.zeros((num_layers, 2, num_pages, num_kv_heads, page_size, head_dim), dtype=dtype, device=device),
                    torch.full((num_seqs, -(-max_ctx // page_size)), -1, **kw), torch.zeros(num_seqs, **kw),
                    torch.zeros(num_pages, **kw), max_ctx)

    @classmethod
    def over(cls, data: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
             max_ctx: int | None = None) -> "PagedKVCache":
        """A cache over tensors that the caller holds (``max_ctx`` ``None``: what a table row has room for)."""
        cache = cls.__new__(cls)
        cache._setup(data, table, lengths, refs, max_ctx)
        return cache

    def _setup(self, data, table, lengths, refs, max_ctx) -> None:
        if data.dim() != 6 or data.shape[1] != 2 or not data.is_contiguous() or table.dim() != 2:
            raise ValueError("data must be contiguous [layers, 2, pages, kv heads, page size, head dim], table [rows, max pages]")
        if not data.is_cuda:
            raise ValueError("data must be a GPU tensor (libq4dec has no CPU path)")
        if data.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("the cache is fp16 or bf16")
        self.device, self.dtype = data.device, data.dtype
        self.data, self.table = data, _ints(table, "table", data.device)
        self.num_layers, _, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = data.shape
        self.num_seqs, self.max_pages = table.shape
        room = self.max_pages * self.page_size
        self.max_ctx = room if max_ctx is None else int(max_ctx)
        if not 1 <= self.max_ctx <= room:
            raise ValueError(f"max_ctx must be 1 .. {room}, what a table row has room for")
        self.lengths = _ints(lengths, "lengths", data.device, self.num_seqs)
        self.refs = _ints(refs, "refs", data.device, self.num_pages)
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._desc = Q4dPages(data.data_ptr(), _DTYPES[data.dtype], self.num_layers, self.num_pages, self.num_kv_heads,
                              self.page_size, self.head_dim, table.data_ptr(), lengths.data_ptr(), refs.data_ptr(),
                              self.num_seqs, self.max_pages, self._status.data_ptr(), self.max_ctx)
        self._ref = ctypes.byref(self._desc)
        self._lib = _lib.load()
        self._ws_bytes = int(self._lib.q4d_pages_workspace_bytes(self._ref))
        if self._ws_bytes == 0:
            raise _lib.Q4DecError(-11, "q4d_pages_workspace_bytes")
        self._ws = torch.empty(self._ws_bytes, dtype=torch.uint8, device=self.device)
        self._wsp = self._ws.data_ptr()
        self._index = data.get_device()

    def _call(self, name: str, *args) -> None:
        """The entry point on the cache's device and its current stream."""
        call = getattr(self._lib, name)
        here = _device()
        if here == self._index:
            rc = call(*args, _stream(here))
        else:
            torch.cuda.set_device(self._index)
            try:
                rc = call(*args, _stream(self._index))
            finally:
                torch.cuda.set_device(here)
        if rc:
            check(rc, name)

    def _check_batch(self, batch: RaggedBatch) -> None:
        if batch._index != self._index:
            raise ValueError(f"the batch is on {batch.starts.device}, the cache on {self.device}")
        if batch.seqs is None and batch.n > self.num_seqs:
            raise ValueError(f"a batch of {batch.n} sequences without seqs, the cache has {self.num_seqs} rows")

    # -- pages -------------------------------------------------------------------------
    def reserve(self, batch: RaggedBatch) -> None:
        """Every sequence grows by its new tokens: lengths, pages, and a copy of a partly filled last
        page that others hold too.  All or nothing; a refused one also holds back later calls and
        :meth:`append` until :meth:`raise_for_status` clears the word; the other page calls are carried
        out all the same (q4d_pages_reserve)."""
        self._check_batch(batch)
        self._call("q4d_pages_reserve", self._ref, batch._ref, self._wsp, self._ws_bytes)

    def fork(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Row ``dst[i]``, which is empty, becomes a copy of row ``src[i]`` that shares its pages."""
        n = _ints(src, "src", self.device).numel()
        _ints(dst, "dst", self.device, n)
        if n:
            self._call("q4d_pages_fork", self._ref, src.data_ptr(), dst.data_ptr(), n)

    def truncate(self, seqs: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        """Row ``seqs[i]`` keeps its first ``lengths[i]`` positions (``None``: none)."""
        n = _ints(seqs, "seqs", self.device).numel()
        if lengths is not None:
            _ints(lengths, "lengths", self.device, n)
        if n:
            self._call("q4d_pages_truncate", self._ref, seqs.data_ptr(), None if lengths is None else lengths.data_ptr(), n)

    def free(self, seqs: torch.Tensor) -> None:
        """Rows ``seqs`` let go of all their pages."""
        self.truncate(seqs)

    def compact(self) -> torch.Tensor:
        """Held pages move to the lowest numbers; returns how many there are (device int32 [1])."""
        used = torch.empty(1, dtype=torch.int32, device=self.device)
        self._call("q4d_pages_compact", self._ref, used.data_ptr(), self._wsp, self._ws_bytes)
        return used

    # -- a layer -----------------------------------------------------------------------
    def _token_rows(self, x: torch.Tensor, name: str, tokens: int, heads: int | None = None):
        """(x, address, elements from row to row, heads) of x [tokens, heads, head_dim], heads side by
        side; copied only if its rows cannot be read in place."""
        shape = x.shape
        if len(shape) != 3 or shape[0] != tokens or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise ValueError(f"{name} must be [{tokens}, {'heads' if heads is None else heads}, {self.head_dim}], got {tuple(shape)}")
        if x.get_device() != self._index:
            raise ValueError(f"{name} is on {x.device}, the cache on {self.device}")
        ptr, width = x.data_ptr(), shape[1] * shape[2]
        if x.is_contiguous():
            if ptr % 16 == 0:
                return x, ptr, width, shape[1]
            x = x.clone()
        else:
            step, head, one = x.stride()
            if (one == 1 and (head == shape[2] or shape[1] == 1) and step >= width and step * x.element_size() % 16 == 0
                    and ptr % 16 == 0):
                return x, ptr, step, shape[1]
            x = x.contiguous()
        return x, x.data_ptr(), width, shape[1]

    def append(self, layer: int, batch: RaggedBatch, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
               rope: RopeTable | None = None, q_gamma: torch.Tensor | None = None, k_gamma: torch.Tensor | None = None,
               eps: float = 1e-6, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """k and v [tokens, kv_heads, head_dim] of the batch's tokens into their sequences' pages, with
        the head norm (fp32 gammas, optional) and rotation (optional) of q and k; returns the ready q
        rows [tokens, q_heads, head_dim] in the cache's type (``None`` without q).  The inputs may be
        slices of one projection.  Rows in no sequence are left as they were (they hold anything in a
        ``q_out`` of the call's own)."""
        self._check_batch(batch)
        tokens, kind = batch.tokens, k.dtype
        if kind not in _DTYPES or v.dtype != kind or (q is not None and q.dtype != kind):
            raise ValueError("q, k and v must be of one type: fp32, fp16 or bf16")
        k, kp, ks, _ = self._token_rows(k, "k", tokens, self.num_kv_heads)
        v, vp, vs, _ = self._token_rows(v, "v", tokens, self.num_kv_heads)
        qp, qs, qh, op = None, 0, 0, None
        if q is not None:
            q, qp, qs, qh = self._token_rows(q, "q", tokens)
            if q_out is None:
                q_out = torch.empty((tokens, qh, self.head_dim), dtype=self.dtype, device=self.device)
            elif (q_out.shape != q.shape or q_out.dtype != self.dtype or not q_out.is_contiguous()
                  or q_out.get_device() != self._index):
                raise ValueError(f"q_out must be contiguous {self.dtype} {tuple(q.shape)} on {self.device}")
            op = q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        for g, name in ((q_gamma, "q_gamma"), (k_gamma, "k_gamma")):
            if g is not None and (g.dtype != torch.float32 or g.numel() != self.head_dim or not g.is_contiguous()
                                  or g.get_device() != self._index):
                raise ValueError(f"{name} must be contiguous fp32 [{self.head_dim}] on {self.device}")
        if rope is not None and (rope._index != self._index or rope.rotary_dim > self.head_dim):
            raise ValueError(f"the rotation must be on {self.device} and at most {self.head_dim} dims wide")
        self._call("q4d_paged_append", self._ref, layer, batch._ref, qp, qs, qh, kp, ks, vp, vs, _DTYPES[kind],
                   None if q_gamma is None else q_gamma.data_ptr(), None if k_gamma is None else k_gamma.data_ptr(), eps,
                   None if rope is None else rope._ref, op)
        return q_out

    def workspace(self, q_heads: int, batch: RaggedBatch) -> PagedWorkspace:
        """Scratch for :meth:`attention` on this batch and smaller ones."""
        return PagedWorkspace(self, q_heads, batch.n, batch.tokens, batch.max_new)

    def attention(self, layer: int, batch: RaggedBatch, q: torch.Tensor, scaling: float | None = None,
                  out: torch.Tensor | None = None, ws: PagedWorkspace | None = None) -> torch.Tensor:
        """softmax(q k^T scaling) v of the batch's tokens over their sequences' cached positions up to
        their own; q and the result [tokens, q_heads, head_dim] in the cache's type (``scaling``
        ``None``: head_dim ** -0.5).  ``ws``: scratch kept by the caller (:meth:`workspace`); without
        one the call makes its own.  ``out`` may be ``q`` itself.  Rows in no sequence are left as they
        were (zeros in an ``out`` of the call's own)."""
        self._check_batch(batch)
        if q.dtype != self.dtype:
            raise ValueError(f"q must be {self.dtype}, as the cache")
        q, qp, qs, qh = self._token_rows(q, "q", batch.tokens)
        if out is None:
            out = torch.zeros((batch.tokens, qh, self.head_dim), dtype=self.dtype, device=self.device)
        given, op, os, _ = self._token_rows(out, "out", batch.tokens, qh)
        if given is not out or out.dtype != self.dtype:
            raise ValueError(f"out must be {self.dtype} {tuple(q.shape)} on {self.device}, heads side by side, rows 16-byte aligned")
        if ws is None:
            ws = self.workspace(qh, batch)
        elif ws._index != self._index:
            raise ValueError(f"the workspace is on {ws.buf.device}, the cache on {self.device}")
        self._call("q4d_paged_attention", self._ref, layer, batch._ref, qp, qs, qh,
                   self.head_dim ** -0.5 if scaling is None else scaling, op, os, ws.ptr, ws.nbytes)
        return out

    # -- state -------------------------------------------------------------------------
    def status(self) -> int:
        """The device status word (Q4D_STATUS_* bits; synchronises)."""
        return int(self._status.item())

    def raise_for_status(self, what: str) -> None:
        """Raise Q4DecError(Q4D_ERR_STATUS) if a call left something out; the word is cleared."""
        st = self.status()
        if st:
            self._status.zero_()
            _lib.check_status(st, what)


__all__ = ["PagedKVCache", "PagedWorkspace", "RaggedBatch", "RopeTable", "rope_angles"]
