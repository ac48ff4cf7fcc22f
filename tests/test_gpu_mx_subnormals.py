"""Products of subnormal weights, activations and results.

Bounds as in test_gpu_mx_linear, with steps of 2^-149 where fp32 results are subnormal.  In fp16 the matrix units add a
product of a subnormal number (or zero) as if that number were as large as the least normal one, 2^-14: a step of an
addition is then 2^-23 of sum max(|x|, 2^-14) max(|w|, 2^-14)."""

import numpy as np
import pytest
import torch

import mx_ref
from llm_accelerator_amd.mx import MXTensor, mx_linear

pytestmark = pytest.mark.gpu
SIZES = [(3, 64, 32), (3, 64, 96), (5, 4096, 1024), (64, 8192, 160), (300, 4105, 96), (1001, 6147, 224), (20, 49200, 96)]


def weights(rng, n, k, scale, dev):
    p, _ = mx_ref.random_mx(rng, n, k)
    s = np.full((n, k // 32), scale, dtype=np.uint8)
    return MXTensor.from_numpy(p, s, device=dev), torch.from_numpy(mx_ref.values(p, s)).to(dev)


def check(y, xv, wv, least=0.0):
    k = xv.shape[1]
    size = xv.abs().clamp(min=least) @ wv.abs().clamp(min=least).T
    err = (y.double() - xv @ wv.T).abs()
    bound = k * 2.0 ** -23 * size + (k + 1) * 2.0 ** -149
    assert (err <= bound).all(), f"{(err / bound).max().item():.3g} of the bound"


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("scale,x2", [(0, 100), (1, 100), (2, 60), (0, 0), (27, -32), (127, -130), (200, -131)])
def test_bf16(dev, m, n, k, scale, x2):
    rng = np.random.default_rng(scale)
    w, wv = weights(rng, n, k, scale, dev)
    x = (torch.from_numpy(rng.standard_normal((m, k))) * 2.0 ** x2).to(torch.bfloat16).to(dev)
    check(mx_linear(x, w, out_dtype=torch.float32), x.double(), wv)


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("scale,x2", [(100, 0), (103, 0), (104, 3), (108, -8), (115, 0), (127, -18), (127, -22), (120, -10), (104, -16)])
def test_fp16(dev, m, n, k, scale, x2):
    """Weights and activations from 2^-24 on; the weights are the fp16 numbers that dequantize gives."""
    rng = np.random.default_rng(scale)
    w, _ = weights(rng, n, k, scale, dev)
    x = (torch.from_numpy(rng.standard_normal((m, k))) * 2.0 ** x2).half().to(dev)
    check(mx_linear(x, w, out_dtype=torch.float32), x.double(), w.dequantize(torch.float16).double(), 2.0 ** -14)


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("ws,xs", [(0, 250), (0, 127), (0, 110), (60, 60), (63, 63), (10, 100), (250, 120), (1, 0)])
def test_codes(dev, m, n, k, ws, xs):
    rng = np.random.default_rng(ws)
    w, wv = weights(rng, n, k, ws, dev)
    x, xv = weights(rng, m, k, xs, dev)
    check(mx_linear(x, w, out_dtype=torch.float32), xv, wv)
