"""Microscaled floats and log probabilities without a device: the reference the GPU tests use, and what
the C entry points and the Python side refuse before a launch."""

import ctypes

import numpy as np
import pytest
import torch

import mx_ref
from llm_accelerator_amd import _lib
from llm_accelerator_amd._lib import Q4dMX
from llm_accelerator_amd.logprobs import token_logprobs
from llm_accelerator_amd.mx import MXTensor, mx_linear, mx_quantize, mx_score

FAKE = 0x7F0000000000  # aligned, never dereferenced: validation fails before launch
F16, F32, BF16 = 0, 1, 2
NULL, ADDR, SHAPE, DTYPE, CAPACITY = -7, -4, -11, -13, -9


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def mx(rows=48, cols=64, w=FAKE, s=FAKE):
    return ctypes.byref(Q4dMX(w, s, rows, cols))


def test_reference_rounds_ties_to_even_codes():
    x = np.zeros((1, 32))
    x[0, :15] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 5.01, 0.2499, -0.25, -5, 7.9, -7.0, 4.99]
    packed, scale = mx_ref.quantize(x)
    assert scale[0, 0] == 127  # floor(log2(7.9)) - 2 = 0
    got = mx_ref.values(packed, scale)[0]
    assert got[:15].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 6, 0, 0, -4, 6, -6, 4]
    assert (got[15:] == 0).all()


@pytest.mark.parametrize("most,floor,ceil", [(6.0, 0, 0), (6.0001, 0, 1), (4.0, 0, 0), (3.999, -1, 0), (3.0, -1, -1), (7.99, 0, 1),
                                             (8.0, 1, 1), (2.0 ** -126, -127, -127), (2.0 ** -149, -127, -127), (0.0, -127, -127),
                                             (3.4e38, 125, 126)])
def test_reference_exponents(most, floor, ceil):
    assert mx_ref.exponent(most, "floor") == floor
    assert mx_ref.exponent(most, "ceil") == ceil


def test_reference_round_trip_of_every_code():
    packed = np.arange(256, dtype=np.uint8).reshape(16, 16)
    scale = np.full((16, 1), 130, dtype=np.uint8)
    v = mx_ref.values(packed, scale)
    assert v[0, 0] == 0 and v[0, 2] == 4.0 and v[0, 3] == 0 and v[15, 31] == -48.0
    back, s = mx_ref.quantize(v, "ceil")
    assert (mx_ref.values(back, s) == v).all()


def test_sizes(lib):
    assert lib.q4d_mx_code_bytes(1, 32) == lib.q4d_mx_code_bytes(32, 128) == 2048 and lib.q4d_mx_scale_bytes(1, 32) == 128
    assert lib.q4d_mx_code_bytes(33, 160) == 4 * 2048 and lib.q4d_mx_scale_bytes(33, 160) == 4 * 128
    assert lib.q4d_mx_code_bytes(151936, 1024) == 151936 * 512
    assert lib.q4d_mx_code_bytes(2 ** 31 - 1, 128) == lib.q4d_mx_code_bytes(32, 2 ** 31 - 32) == 0
    assert lib.q4d_mx_code_bytes(2 ** 27, 4096) == 2 ** 38 and lib.q4d_mx_code_bytes(2 ** 27, 4128) == 0


def test_quantize_refusals(lib):
    def call(x=FAKE, dt=BF16, ld=64, rows=48, cols=64, rule=0, p=FAKE, s=FAKE):
        return lib.q4d_mx_quantize(x, dt, ld, rule, mx(rows, cols, p, s), None)
    assert call(x=None) == call(p=None) == call(s=None) == lib.q4d_mx_quantize(FAKE, BF16, 64, 0, None, None) == NULL
    assert call(dt=3) == DTYPE
    assert call(rows=0) == call(cols=48, ld=48) == call(cols=0) == call(ld=32) == call(rule=2) == call(rule=-1) == SHAPE
    assert call(rows=2 ** 31 - 1, cols=1024, ld=1024) == SHAPE  # more tiles than 32 bits count
    assert call(x=FAKE + 8) == call(p=FAKE + 8) == call(ld=68) == call(dt=F32, ld=66) == ADDR


def test_pack_refusals(lib):
    for call in (lambda p, s, t: lib.q4d_mx_pack(p, s, t, None), lambda p, s, t: lib.q4d_mx_unpack(t, p, s, None)):
        assert call(None, FAKE, mx()) == call(FAKE, None, mx()) == call(FAKE, FAKE, None) == call(FAKE, FAKE, mx(w=None)) == NULL
        assert call(FAKE, FAKE, mx(cols=33)) == SHAPE
        assert call(FAKE + 2, FAKE, mx()) == call(FAKE, FAKE, mx(w=FAKE + 8)) == call(FAKE, FAKE, mx(s=FAKE + 2)) == ADDR


def test_dequantize_refusals(lib):
    assert lib.q4d_mx_dequantize(None, FAKE, F32, None) == NULL
    assert lib.q4d_mx_dequantize(mx(w=None), FAKE, F32, None) == lib.q4d_mx_dequantize(mx(s=None), FAKE, F32, None) == NULL
    assert lib.q4d_mx_dequantize(mx(), None, F32, None) == NULL
    assert lib.q4d_mx_dequantize(mx(cols=40), FAKE, F32, None) == lib.q4d_mx_dequantize(mx(rows=0), FAKE, F32, None) == SHAPE
    assert lib.q4d_mx_dequantize(mx(), FAKE, 5, None) == DTYPE
    assert lib.q4d_mx_dequantize(mx(w=FAKE + 4), FAKE, F32, None) == lib.q4d_mx_dequantize(mx(), FAKE + 4, F32, None) == ADDR


def test_linear_refusals(lib):
    def call(w=mx(), x=FAKE, dt=F16, stride=64, m=3, y=FAKE, ydt=F32):
        return lib.q4d_mx_linear(w, x, dt, stride, m, y, ydt, None)
    assert call(w=None) == call(x=None) == call(y=None) == NULL
    assert call(dt=F32) == call(ydt=9) == DTYPE
    assert call(m=0) == call(m=-1) == call(stride=32) == call(w=mx(cols=33)) == SHAPE
    assert call(x=FAKE + 2) == call(stride=68) == call(y=FAKE + 2) == ADDR


def test_matmul_refusals(lib):
    assert lib.q4d_mx_matmul(mx(), None, FAKE, F32, None) == lib.q4d_mx_matmul(None, mx(), FAKE, F32, None) == NULL
    assert lib.q4d_mx_matmul(mx(), mx(cols=96), FAKE, F32, None) == SHAPE
    assert lib.q4d_mx_matmul(mx(), mx(), FAKE, 4, None) == DTYPE


def test_score_refusals(lib):
    need = lib.q4d_mx_score_workspace_bytes(48, 64, 3)
    assert need > 0 and lib.q4d_mx_score_workspace_bytes(0, 64, 3) == lib.q4d_mx_score_workspace_bytes(48, 64, 0) == 0
    assert lib.q4d_mx_score_workspace_bytes(48, 40, 3) == 0

    def call(w=mx(), x=FAKE, dt=F16, stride=64, m=3, targets=FAKE, out=FAKE, ws=FAKE, nbytes=need):
        return lib.q4d_mx_score(w, x, dt, stride, m, targets, out, out, out, ws, nbytes, None)
    assert call(w=None) == call(x=None) == call(targets=None) == call(out=None) == call(ws=None) == NULL
    assert call(dt=F32) == DTYPE
    assert call(m=0) == call(stride=8) == SHAPE
    assert call(ws=FAKE + 16) == call(targets=FAKE + 2) == ADDR
    assert call(nbytes=need - 1) == CAPACITY


def test_logprobs_refusals(lib):
    need = lib.q4d_token_logprobs_workspace_bytes(3, 100, 5)
    assert need > 0
    for rows, vocab, top in ((0, 100, 5), (3, 0, 0), (3, 100, 33), (3, 4, 5), (3, 100, -1), (3, (1 << 20) + 1, 5)):
        assert lib.q4d_token_logprobs_workspace_bytes(rows, vocab, top) == 0
        assert lib.q4d_token_logprobs(FAKE, F32, 1 << 21, rows, vocab, FAKE, top, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, None) == SHAPE

    def call(x=FAKE, dt=F32, stride=100, targets=FAKE, lp=FAKE, rank=FAKE, ent=FAKE, tl=FAKE, ti=FAKE, ws=FAKE, nbytes=need):
        return lib.q4d_token_logprobs(x, dt, stride, 3, 100, targets, 5, lp, rank, ent, tl, ti, ws, nbytes, None)
    assert call(x=None) == call(lp=None) == call(rank=None) == call(ent=None) == call(tl=None) == call(ti=None) == call(ws=None) == NULL
    assert call(dt=7) == DTYPE
    assert call(stride=99) == SHAPE
    assert call(x=FAKE + 2) == call(ws=FAKE + 8) == call(targets=FAKE + 1) == ADDR
    assert call(nbytes=need - 1) == CAPACITY


def test_python_refuses_host_tensors_and_shapes():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="GPU"):
        mx_quantize(x)
    with pytest.raises(ValueError, match="multiple of 32"):
        mx_quantize(torch.zeros(4, 48))
    with pytest.raises(ValueError, match="rule"):
        mx_quantize(x, rule="up")
    with pytest.raises(ValueError, match="fp32"):
        mx_quantize(x.double())
    with pytest.raises(ValueError, match="GPU"):
        token_logprobs(x)
    with pytest.raises(TypeError):
        MXTensor(torch.zeros(4, 16), torch.zeros(4, 1, dtype=torch.uint8))
    with pytest.raises(ValueError, match="match"):
        MXTensor(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8))
    with pytest.raises(ValueError, match="multiple"):
        MXTensor(torch.zeros(4, 8, dtype=torch.uint8), torch.zeros(4, 0, dtype=torch.uint8))
    w = MXTensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8))
    assert w.shape == (4, 64) and w.nbytes == 2048 + 128  # one tile
    for call in (lambda: w.dequantize(), lambda: mx_linear(x.half(), w), lambda: mx_score(x.half(), w, torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        mx_linear(x.half(), x)


@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 96), (32, 128), (33, 160), (70, 288)])
def test_order_in_memory_and_back(rows, cols):
    rng = np.random.default_rng(0)
    p, s = mx_ref.random_mx(rng, rows, cols)
    t = MXTensor.from_numpy(p, s)
    p2, s2 = t.numpy()
    assert (p == p2).all() and (s == s2).all()
    codes, scales, kt = t.codes.numpy(), t.scales.numpy(), -(-cols // 128)
    for row, block in ((0, 0), (rows - 1, cols // 32 - 1), (rows // 2, cols // 64)):
        tile = row // 32 * kt + block // 4
        at = tile * 2048 + block % 4 * 512 + row % 32 * 16
        assert (codes[at:at + 16] == p[row, 16 * block:16 * block + 16]).all()
        assert scales[tile * 128 + row % 32 * 4 + block % 4] == s[row, block]
    for row in range(rows):  # columns past the last are zeros
        for block in range(cols // 32, 4 * kt):
            tile = row // 32 * kt + block // 4
            at = tile * 2048 + block % 4 * 512 + row % 32 * 16
            assert not codes[at:at + 16].any() and scales[tile * 128 + row % 32 * 4 + block % 4] == 0


def test_sizes_past_the_counts(lib):
    def linear(stride, m, w=mx()):
        return lib.q4d_mx_linear(w, FAKE, F16, stride, m, FAKE, F32, None)
    assert linear(1 << 24, 2) == linear(1 << 40, 2 ** 31 - 1) == SHAPE
    assert linear(64, 2 ** 31 - 1, mx(rows=2 ** 27, cols=64)) == SHAPE  # more tiles than a launch has
    assert lib.q4d_mx_score_workspace_bytes(48, 64, 1 << 23) > 0 == lib.q4d_mx_score_workspace_bytes(48, 64, (1 << 23) + 1)
    assert lib.q4d_mx_score(mx(), FAKE, F16, 64, (1 << 23) + 1, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 60, None) == SHAPE
    assert lib.q4d_mx_matmul(mx(rows=2 ** 31 - 256, cols=32), mx(rows=9, cols=32), FAKE, F32, None) == SHAPE
    assert lib.q4d_token_logprobs_workspace_bytes(1 << 23, 16384, 0) > 0 == lib.q4d_token_logprobs_workspace_bytes(1 << 23, 16385, 0)
    for rows, cols in ((1, 1 << 32), ((1 << 32) + 1, 32)):
        with pytest.raises(ValueError, match="at most"):
            MXTensor.__new__(MXTensor)._new(torch.zeros(1), rows, cols)


def test_calls_run_on_the_tensors_device(monkeypatch):
    """On another current device: the tensors' is made current for the call, with its own stream, and the caller's
    again afterwards, whether the call succeeds, fails or raises."""
    from llm_accelerator_amd import model
    now, log = [0], []

    class Lib:
        def q4d_some_call(self, *args):
            log.append((now[0], args))
            if args[0] == "raise":
                raise TypeError
            return args[0]
    monkeypatch.setattr(model, "_device", lambda: now[0])
    monkeypatch.setattr(model, "_stream", lambda i: 100 + i)
    monkeypatch.setattr(torch.cuda, "set_device", lambda i: now.__setitem__(0, i))
    monkeypatch.setattr(_lib, "load", Lib)
    for here in (0, 3):
        now[0] = here
        model.call_on(3, "q4d_some_call", 0, "x")
        assert log[-1] == (3, (0, "x", 103)) and now[0] == here
        with pytest.raises(_lib.Q4DecError):
            model.call_on(3, "q4d_some_call", SHAPE)
        assert now[0] == here
        with pytest.raises(TypeError):
            model.call_on(3, "q4d_some_call", "raise")
        assert now[0] == here
