"""Microscaled 4-bit floats: the 4-bit format that the MI355X's matrix units read as it is.

No counterpart in the reference, whose 4-bit weights are integers with a scale per 64 columns
(``Source/Q4_FORMAT.md:75-140``, :class:`~llm_accelerator_amd.model.Q4Tensor`); the operators stand
beside ``quantize_weight_q4``, ``manual_linear_from_weight`` and the LM head's argmax:

* :func:`mx_quantize` -- a matrix as an :class:`MXTensor` (blocks of 32 codes and a power of two);
  :meth:`MXTensor.dequantize` -- the values back;
* :func:`mx_linear` -- ``x @ W.T`` with such weights, x in 16 bits or an :class:`MXTensor` itself;
* :func:`mx_score` -- how likely given tokens are under an output head of such weights, without the
  logits in memory.

Every call is launched on torch's current stream of its tensors' device, does not synchronise, keeps
nothing between calls and can be captured into a graph.  Arguments are checked (``ValueError`` /
:class:`~llm_accelerator_amd._lib.Q4DecError`).
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import numpy as np
import torch

from . import _lib
from ._lib import Q4D_BF16, Q4D_F16, Q4D_F32, Q4dMX
from .model import call_on

BLOCK = 32
_DTYPES = {torch.float16: Q4D_F16, torch.bfloat16: Q4D_BF16, torch.float32: Q4D_F32}
_RULES = {"floor": 0, "ceil": 1}


TILE_ROWS, TILE_COLS = 32, 128  # of the order in memory (q4d_mx_t)
_MOST = 0x7FFFFF00              # rows or columns, counted in 32 bits behind the C interface


def _order(rows_bytes: torch.Tensor, width: int) -> torch.Tensor:
    """[rows, blocks * width] bytes as [row tiles, column tiles, 32 rows, 4 blocks, width], zeros past both ends."""
    rows, n = rows_bytes.shape[0], rows_bytes.shape[1] // width
    rt, kt = -(-rows // TILE_ROWS), -(-n // 4)
    full = rows_bytes.new_zeros((rt * TILE_ROWS, kt * 4, width))
    full[:rows, :n] = rows_bytes.view(rows, n, width)
    return full.view(rt, TILE_ROWS, kt, 4, width).transpose(1, 2)


class MXTensor:
    """A matrix of microscaled 4-bit floats, from rows of codes ``packed`` uint8 [rows, cols/2] (the even
    column in the low nibble) and ``scale`` uint8 [rows, cols/32] (2^(scale - 127); 255: NaN).

    It keeps a copy of its own in the order that the kernels read (:attr:`codes` and :attr:`scales`, tiles
    of 32 rows and 128 columns); :attr:`packed` and :attr:`scale` are the rows again, made at each access."""

    def __init__(self, packed: torch.Tensor, scale: torch.Tensor):
        if packed.dtype != torch.uint8 or scale.dtype != torch.uint8:
            raise TypeError("MXTensor needs uint8 packed codes and uint8 scales")
        if packed.dim() != 2 or packed.shape[0] == 0 or packed.shape[1] == 0 or packed.shape[1] % (BLOCK // 2):
            raise ValueError(f"packed must be [rows, cols/2] with cols a multiple of {BLOCK}, got {tuple(packed.shape)}")
        rows, cols = packed.shape[0], 2 * packed.shape[1]
        if scale.shape != (rows, cols // BLOCK):
            raise ValueError(f"scale shape {tuple(scale.shape)} does not match packed {tuple(packed.shape)}")
        if packed.device != scale.device:
            raise ValueError(f"packed is on {packed.device}, scale on {scale.device}")
        packed, scale = packed.contiguous(), scale.contiguous()
        if not packed.is_cuda:
            codes, scales = _order(packed, 16).transpose(2, 3).reshape(-1), _order(scale, 1).reshape(-1)
            self._setup(torch.cat((codes, scales)), rows, cols)
            return
        if packed.data_ptr() % 4:
            packed = packed.clone()
        self._new(packed, rows, cols)
        call_on(self._index, "q4d_mx_pack", packed.data_ptr(), scale.data_ptr(), self._ref)

    def _setup(self, memory: torch.Tensor, rows: int, cols: int) -> "MXTensor":
        """Over ``memory``: the codes' bytes, then the scales'."""
        at = memory.data_ptr()
        self._memory, self.shape = memory, (rows, cols)
        self._desc = Q4dMX(at, at + memory.numel() // 17 * 16, rows, cols)  # 2048 and 128 bytes a tile
        self._ref = ctypes.byref(self._desc)
        self._index = memory.get_device()
        return self

    def _new(self, like: torch.Tensor, rows: int, cols: int) -> "MXTensor":
        """Memory for rows x cols on the device of ``like``."""
        if rows > _MOST or cols > _MOST:
            raise ValueError(f"an MXTensor has at most {_MOST} rows and columns, got {rows} x {cols}")
        return self._setup(like.new_empty(-(-rows // TILE_ROWS) * -(-cols // TILE_COLS) * 2176, dtype=torch.uint8), rows, cols)

    # (copies and pickles: the descriptor holds addresses, and is made anew over the memory that came)
    def __getstate__(self) -> tuple:
        return self._memory, self.shape

    def __setstate__(self, state: tuple) -> None:
        memory, shape = state
        self._setup(memory, *shape)

    @property
    def codes(self) -> torch.Tensor:
        return self._memory[:self._memory.numel() // 17 * 16]

    @property
    def scales(self) -> torch.Tensor:
        return self._memory[self._memory.numel() // 17 * 16:]

    def _rows(self) -> tuple[torch.Tensor, torch.Tensor]:
        rows, cols = self.shape
        if self._index >= 0:
            packed = self._memory.new_empty((rows, cols // 2))
            scale = self._memory.new_empty((rows, cols // BLOCK))
            call_on(self._index, "q4d_mx_unpack", self._ref, packed.data_ptr(), scale.data_ptr())
            return packed, scale
        rt, kt = -(-rows // TILE_ROWS), -(-cols // TILE_COLS)
        packed = self.codes.view(rt, kt, 4, TILE_ROWS, 16).permute(0, 3, 1, 2, 4).reshape(rt * TILE_ROWS, -1)
        scale = self.scales.view(rt, kt, TILE_ROWS, 4).permute(0, 2, 1, 3).reshape(rt * TILE_ROWS, -1)
        return packed[:rows, :cols // 2].contiguous(), scale[:rows, :cols // BLOCK].contiguous()

    @property
    def packed(self) -> torch.Tensor:
        return self._rows()[0]

    @property
    def scale(self) -> torch.Tensor:
        return self._rows()[1]

    @property
    def device(self) -> torch.device:
        return self._memory.device

    @property
    def nbytes(self) -> int:
        return self._memory.numel()

    def to(self, device) -> "MXTensor":
        return MXTensor.__new__(MXTensor)._setup(self._memory.to(device), *self.shape)

    def numpy(self) -> tuple[np.ndarray, np.ndarray]:
        packed, scale = self._rows()
        return packed.cpu().numpy(), scale.cpu().numpy()

    @classmethod
    def from_numpy(cls, packed: np.ndarray, scale: np.ndarray, device="cpu") -> "MXTensor":
        return cls(torch.from_numpy(np.ascontiguousarray(packed, dtype=np.uint8)).to(device),
                   torch.from_numpy(np.ascontiguousarray(scale, dtype=np.uint8)).to(device))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values [rows, cols]: exact in fp32 and bf16 (Inf past their largest number), rounded once
        in fp16."""
        if dtype not in _DTYPES:
            raise ValueError(f"dtype must be fp32, fp16 or bf16, got {dtype}")
        _on_gpu(self)
        y = self._memory.new_empty(self.shape, dtype=dtype)
        call_on(self._index, "q4d_mx_dequantize", self._ref, y.data_ptr(), _DTYPES[dtype])
        return y


def _on_gpu(t) -> None:
    if t._index < 0:
        raise ValueError("the MXTensor must be on a GPU (libq4dec has no CPU path)")


def _rows(x: torch.Tensor, name: str, cols: int | None = None):
    """(x, its rows, elements from row to row) of x [..., cols], copied only if its rows cannot be read in place."""
    shape = x.shape
    if len(shape) == 2 and x.is_cuda and shape[1] == (cols or shape[1]) and x.data_ptr() % 16 == 0 and x.is_contiguous():
        return x, shape[0], shape[1]  # (cols are multiples of 32, so the rows are aligned as the first is)
    if not x.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (libq4dec has no CPU path)")
    if x.dim() == 0 or (cols is not None and x.shape[-1] != cols):
        raise ValueError(f"{name} must be [..., {'cols' if cols is None else cols}], got {tuple(x.shape)}")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    step = x.stride(0) if x.shape[0] > 1 else x.shape[1]
    if (x.data_ptr() % 16 or (x.shape[1] > 1 and x.stride(1) != 1) or step < x.shape[1] or step >= 1 << 24
            or step * x.element_size() % 16):
        x = x.clone(memory_format=torch.contiguous_format)
        step = x.shape[1]
    return x, x.shape[0], step


def mx_quantize(x: torch.Tensor, rule: str = "floor") -> MXTensor:
    """x [rows, cols] (or [..., cols], whose leading dims become rows; fp32, fp16 or bf16) as an
    :class:`MXTensor`.  A block's power of two is 2^e, e = floor(log2(largest magnitude)) - 2
    (``"floor"``, the format's own rule: magnitudes past 6 x 2^e become that) or the smallest e with which
    none passes 6 x 2^e (``"ceil"``); values go to the nearest code, ties to the even one.  A block with
    Inf or NaN is NaN."""
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be fp32, fp16 or bf16, got {x.dtype}")
    if rule not in _RULES:
        raise ValueError(f"unknown rule {rule!r}: floor or ceil")
    if x.dim() and (x.shape[-1] == 0 or x.shape[-1] % BLOCK):
        raise ValueError(f"the last dim must be a multiple of {BLOCK}, got {x.shape[-1]}")
    x, rows, step = _rows(x, "x")
    if rows == 0:
        raise ValueError("expected at least one row")
    cols = x.shape[1]
    got = MXTensor.__new__(MXTensor)._new(x, rows, cols)
    call_on(got._index, "q4d_mx_quantize", x.data_ptr(), _DTYPES[x.dtype], step, _RULES[rule], got._ref)
    return got


def mx_linear(x: torch.Tensor | MXTensor, weight: MXTensor, out_dtype: torch.dtype | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T``: x [..., cols] in fp16 or bf16, where the weights enter as numbers of that type
    (``weight.dequantize(x.dtype)``: exact in bf16; in fp16 blocks whose scale lies outside 2^-23 .. 2^13 are
    rounded or Inf, and numbers below 2^-14 are added with the precision of 2^-14), or an :class:`MXTensor`
    [rows, cols], where both enter as they are.  fp32 sums, rounded once to ``out_dtype`` (fp32, fp16 or bf16; ``None``: x's type, bf16 for an
    MXTensor).  ``out``: a contiguous result of the caller's, apart from x."""
    if not isinstance(weight, MXTensor):
        raise TypeError("weight must be an MXTensor")
    _on_gpu(weight)
    n, cols = weight.shape
    codes = isinstance(x, MXTensor)
    if codes:
        _on_gpu(x)
        if x.shape[1] != cols:
            raise ValueError(f"x has {x.shape[1]} columns, the weights {cols}")
        index, lead, kind, m = x._index, x.shape[:1], torch.bfloat16, x.shape[0]
    else:
        kind = x.dtype
        if kind is not torch.bfloat16 and kind is not torch.float16:
            raise ValueError(f"x must be fp16, bf16 or an MXTensor, got {kind}")
        lead = x.shape[:-1]
        x, m, step = _rows(x, "x", cols)
        index = x.get_device()
    if index != weight._index:
        raise ValueError(f"x is on {x.device}, the weights on {weight.device}")
    if out is None:
        y_kind = kind if out_dtype is None else out_dtype
        if y_kind not in _DTYPES:
            raise ValueError(f"out_dtype must be fp32, fp16 or bf16, got {y_kind}")
        out = weight._memory.new_empty((*lead, n), dtype=y_kind)
    else:
        y_kind = out.dtype
        if (y_kind not in _DTYPES or out_dtype not in (None, y_kind) or out.shape != (*lead, n) or not out.is_contiguous()
                or out.get_device() != index or out.data_ptr() % 16):
            raise ValueError(f"out must be contiguous {(*lead, n)} in fp32, fp16 or bf16 (out_dtype) on {weight.device}, 16-byte aligned")
    if m == 0:
        return out
    if m > _MOST:
        raise ValueError(f"x has at most {_MOST} rows, got {m}")
    if codes:
        call_on(index, "q4d_mx_matmul", weight._ref, x._ref, out.data_ptr(), _DTYPES[y_kind])
    else:
        call_on(index, "q4d_mx_linear", weight._ref, x.data_ptr(), _DTYPES[kind], step, m, out.data_ptr(), _DTYPES[y_kind])
    return out


class MXScores(NamedTuple):
    logprob: torch.Tensor   # of the given tokens
    entropy: torch.Tensor   # of the distributions
    best: torch.Tensor      # the largest log probability


def mx_score(hidden: torch.Tensor, weight: MXTensor, targets: torch.Tensor) -> MXScores:
    """How likely ``targets`` [...] (int32) are under the output head ``weight`` [vocab, cols] at the rows
    ``hidden`` [..., cols] (fp16 or bf16, with weights of that type): the log softmax of ``mx_linear(hidden, weight)`` in fp32 at the
    targets, its entropy and its maximum, fp32 [...] each, without the products in memory.  Up to 2^23 rows, and
    ceil(rows / 64) x ceil(vocab / 256) up to 2^23 (903808 rows of 151936 tokens).
    A target outside the vocabulary (a padded row's) gives NaN, and so does a row whose products hold NaN, +Inf or
    nothing but -Inf."""
    if not isinstance(weight, MXTensor):
        raise TypeError("weight must be an MXTensor")
    _on_gpu(weight)
    if hidden.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"hidden must be fp16 or bf16, got {hidden.dtype}")
    lead = hidden.shape[:-1]
    x, m, step = _rows(hidden, "hidden", weight.shape[1])
    index = x.get_device()
    if index != weight._index:
        raise ValueError(f"hidden is on {x.device}, the weights on {weight.device}")
    if targets.dtype != torch.int32 or targets.shape != lead or targets.get_device() != index:
        raise ValueError(f"targets must be int32 {tuple(lead)} on {x.device}")
    targets = targets.contiguous()
    if m > 1 << 23:
        raise ValueError(f"up to 2^23 rows, got {m}")
    nbytes = _lib.load().q4d_mx_score_workspace_bytes(*weight.shape, m) if m else 0
    if m and not nbytes:
        raise ValueError(f"ceil(rows / 64) x ceil(vocab / 256) up to 2^23, got {m} rows of {weight.shape[0]}")
    got = x.new_empty((3, *lead), dtype=torch.float32)
    if m:
        ws = x.new_empty(nbytes, dtype=torch.uint8)
        base, row = got.data_ptr(), 4 * m
        call_on(index, "q4d_mx_score", weight._ref, x.data_ptr(), _DTYPES[x.dtype], step, m, targets.data_ptr(), base,
                base + row, base + 2 * row, ws.data_ptr(), nbytes)
    return MXScores(*got.unbind(0))


__all__ = ["MXTensor", "MXScores", "mx_quantize", "mx_linear", "mx_score"]
