"""mx_score against the log softmax of the products in 64 bits.

Tolerance.  The logits z are off by dz <= K 2^-23 sum |x w| (see test_gpu_mx_linear).  Log probabilities
move by 2 max dz at most; the entropy, whose derivative by z_i is p_i |log p_i + H|, by 2 H max dz.  The
sums of the softmax: an exponential is off by (|d| + 2) 2^-23 of itself, weighted by its share that is
(H + 2) 2^-23 of the sum; a term passes at most 400 additions and rescalings of 2^-23 each (32 in a lane,
the lanes, waves and parts of a row).  So log sum e^z is off by (H + 402) 2^-23, and t / l, a mean of
|z - max| <= H + log l, by twice that of H + log l + 1.
"""

import numpy as np
import pytest
import torch

import mx_ref
from llm_accelerator_amd.logprobs import token_logprobs
from llm_accelerator_amd.mx import MXTensor, mx_linear, mx_score

pytestmark = pytest.mark.gpu


def head(rng, n, k, dev, lo=121, hi=125):
    p, s = mx_ref.random_mx(rng, n, k, lo, hi)
    return MXTensor.from_numpy(p, s, device=dev), torch.from_numpy(mx_ref.values(p, s)).to(dev)


def check(got, x, w, targets):
    z = x.double() @ w.T
    dz = (x.shape[1] * 2.0 ** -23 * (x.double().abs() @ w.abs().T)).amax(-1)
    lp = torch.log_softmax(z, -1)
    h = -(lp.exp() * lp).sum(-1)
    best = lp.amax(-1)
    lse = (h + 402) * 2.0 ** -23
    for name, a, b, tol in (("logprob", got.logprob, lp.gather(1, targets.long()[:, None])[:, 0], 2 * dz + lse),
                            ("best", got.best, best, 2 * dz + lse),
                            ("entropy", got.entropy, h, 2 * h * dz + lse + 2 * lse * (h - best + 1))):
        # the result's own rounding and those of the subtractions
        tol = tol + 2.0 ** -22 * (b.abs() + 1)
        err = (a.double() - b).abs()
        assert (err <= tol).all(), f"{name}: {(err / tol).max().item():.2f} of the bound"


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 5000, 1024), (2, 2, 64), (7, 257, 96), (16, 4096, 1024), (17, 300, 160), (21, 20000, 1024),
                                   (33, 16, 288), (48, 3001, 512), (64, 1000, 2048), (65, 255, 64), (128, 256, 1024), (131, 9001, 224),
                                   (300, 2000, 1056), (5, 33000, 1024), (32, 40001, 96), (33, 32768, 1024), (64, 33333, 992), (2, 32800, 4096),
                                   (20, 32801, 4096), (64, 32799, 2048)])
def test_shapes(dev, m, n, k, kind):
    rng = np.random.default_rng(m + 3 * n + 5 * k)
    w, wv = head(rng, n, k, dev)
    x = torch.from_numpy(rng.standard_normal((m, k)) / np.sqrt(k) * 8).to(dev).to(kind)
    targets = torch.from_numpy(rng.integers(0, n, m)).to(dev).int()
    targets[0], targets[-1] = 0, n - 1
    got = mx_score(x, w, targets)
    assert all(v.shape == (m,) and v.dtype == torch.float32 for v in got)
    check(got, x, wv, targets)


def test_one_token_certain(dev):
    """One logit far above the others: entropy near 0, never NaN."""
    packed = torch.zeros(700, 32, dtype=torch.uint8, device=dev)
    packed[37, 0] = 7  # 6
    w = MXTensor(packed, torch.full((700, 2), 127, dtype=torch.uint8, device=dev))
    x = torch.zeros(3, 64, device=dev, dtype=torch.bfloat16)
    x[1, 0], x[2, 0] = 100.0, -100.0
    t = torch.tensor([37, 37, 37], device=dev, dtype=torch.int32)
    got = mx_score(x, w, t)
    assert abs(got.logprob[0].item() + np.log(700)) < 1e-5 and abs(got.entropy[0].item() - np.log(700)) < 1e-5
    assert got.logprob[1].item() == 0 and got.entropy[1].item() == 0 and got.best[1].item() == 0
    assert abs(got.logprob[2].item() + 600 + np.log(699)) < 1e-3


def test_targets_outside_and_bad_rows(dev):
    rng = np.random.default_rng(0)
    w, wv = head(rng, 900, 96, dev)
    for m in (6, 70):
        x = torch.from_numpy(rng.standard_normal((m, 96))).to(dev).to(torch.bfloat16)
        t = torch.from_numpy(rng.integers(0, 900, m)).to(dev).int()
        clean = mx_score(x, w, t)
        t2, x2 = t.clone(), x.clone()
        t2[0], t2[1] = -1, 900
        x2[3, 5], x2[4, 95] = float("nan"), float("inf")
        got = mx_score(x2, w, t2)
        assert got.logprob[:2].isnan().all()
        assert torch.equal(got.entropy[:3], clean.entropy[:3]) and torch.equal(got.best[:3], clean.best[:3])
        assert got.logprob[3:5].isnan().all() and got.entropy[3:5].isnan().all() and got.best[3:5].isnan().all()
        assert torch.equal(got.logprob[5:], clean.logprob[5:])


@pytest.mark.parametrize("m", [9, 150])
def test_agrees_with_product_and_logprobs(dev, m):
    rng = np.random.default_rng(m)
    w, _ = head(rng, 3333, 1024, dev)
    x = torch.from_numpy(rng.standard_normal((m, 1024)) / 4).to(dev).to(torch.float16)
    t = torch.from_numpy(rng.integers(0, 3333, m)).to(dev).int()
    a = mx_score(x.view(1, m, 1024), w, t.view(1, m))
    b = token_logprobs(mx_linear(x, w, out_dtype=torch.float32), t, top=1)
    size = (x.double().abs() @ w.dequantize().double().abs().T).amax(-1)
    tol = 4 * 1024 * 2.0 ** -23 * size + 1e-4
    assert ((a.logprob[0] - b.logprob).abs() <= tol).all()
    assert ((a.best[0] - b.top_logprobs[:, 0]).abs() <= tol).all()
    assert ((a.entropy[0] - b.entropy).abs() <= 20 * tol).all()


def test_no_rows_and_refusals(dev):
    rng = np.random.default_rng(0)
    w, _ = head(rng, 90, 64, dev)
    x = torch.zeros(3, 64, device=dev, dtype=torch.float16)
    t = torch.zeros(3, device=dev, dtype=torch.int32)
    assert mx_score(x[:0], w, t[:0]).logprob.shape == (0,)
    for bad in (lambda: mx_score(x.float(), w, t), lambda: mx_score(x, w, t.long()), lambda: mx_score(x, w, t[:2]),
                lambda: mx_score(x[:, :32], w, t), lambda: mx_score(x, w, t.cpu()), lambda: mx_score(x.cpu(), w, t)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("m,n", [(6, 300), (100, 300), (100, 1025), (6, 49152), (20, 49200)])  # each kernel, ragged tiles
def test_logits_of_minus_inf_and_far_apart(dev, m, n):
    """-Inf has the probability 0, nothing but -Inf is NaN, and what is finite counts however large.  Every logit is
    one product of powers of two and short numbers, so that the bound is the softmax's alone (2^-17: 2^-22 of 1 + |log
    probability|, which is below 24 here)."""
    rng = np.random.default_rng(n)
    codes = np.zeros((n, 64), dtype=np.uint8)
    codes[37, 0] = 15                        # -6
    codes[:, 1] = rng.integers(0, 16, n)
    codes[:, 2] = 10                         # -1
    codes[:, 3] = 15
    codes[36, 4], codes[38, 4] = 2, 10       # 1, -1
    packed = codes[:, 0::2] | codes[:, 1::2] << 4
    w = MXTensor.from_numpy(packed, np.full((n, 2), 127, dtype=np.uint8), device=dev)
    x = torch.zeros(m, 64, device=dev, dtype=torch.bfloat16)
    x[0, 0], x[0, 1] = 2.0 ** 127, 1.0       # token 37: -Inf
    x[1, 1] = 1.0
    x[2, 2] = 2.0 ** 120                     # all alike, far below 0
    x[3, 3] = 2.0 ** 127                     # all -Inf
    x[4, 4] = 2.0 ** 127                     # one far above, one as far below
    t = torch.full((m,), 37, device=dev, dtype=torch.int32)
    got = mx_score(x, w, t)
    z = torch.from_numpy(mx_ref.values(packed, np.full((n, 2), 127))[:, 1])
    for row in (0, 1):
        zr = z.clone()
        if row == 0:
            zr[37] = -float("inf")
        lp = torch.log_softmax(zr, 0)
        h, best = -(lp.exp() * lp).nansum(), lp.amax()
        lse = (h + 402) * 2.0 ** -23
        assert got.logprob[row].item() == -float("inf") if row == 0 else (got.logprob[row].cpu().double() - lp[37]).abs() <= lse + 2.0 ** -17
        assert (got.best[row].cpu().double() - best).abs() <= lse + 2.0 ** -17
        assert (got.entropy[row].cpu().double() - h).abs() <= lse + 2 * lse * (h - best + 1) + 2.0 ** -17
    even = float(np.log(n))
    lse = (even + 402) * 2.0 ** -23 + 2.0 ** -17
    assert abs(got.logprob[2].item() + even) <= lse and abs(got.best[2].item() + even) <= lse
    assert abs(got.entropy[2].item() - even) <= lse + 2 * lse
    assert all(v[3].isnan() for v in got)
    assert got.logprob[4].item() == -2.0 ** 127 and got.best[4].item() == 0 and got.entropy[4].item() == 0
    far = mx_score(x, w, torch.full_like(t, 38))
    assert far.logprob[4].item() == -float("inf")  # -2^128
    assert (got.logprob[5:] + even).abs().amax() <= lse  # rows of zeros


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 49152, 32), (5, 49153, 96), (16, 50001, 4096), (17, 49200, 2080), (32, 49155, 2048), (32, 60004, 160),
                                   (21, 131001, 1024), (33, 49157, 288), (24, 49151, 128)])
def test_many_tokens(dev, m, n, k, kind):
    rng = np.random.default_rng(n)
    p, s = mx_ref.random_mx(rng, n, k, 121, 125)
    w = MXTensor.from_numpy(p, s, device=dev)
    x = torch.from_numpy(rng.standard_normal((m, k)) / np.sqrt(k) * 8).to(dev).to(kind)
    targets = torch.from_numpy(rng.integers(0, n, m)).to(dev).int()
    targets[0], targets[-1] = 0, n - 1
    check(mx_score(x, w, targets), x, w.dequantize().double(), targets)
