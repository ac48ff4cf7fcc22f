"""q4d_mx_quantize / q4d_mx_dequantize against the format's definition in 64 bits, code for code: rounding
ties, blocks of zeros, subnormals, Inf and NaN, the ends of the exponent's range, both rules, the three
types, row strides, and values back in each type."""

import numpy as np
import pytest
import torch

import mx_ref
from llm_accelerator_amd.mx import MXTensor, mx_quantize

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
RULES = ["floor", "ceil"]


def check(x: torch.Tensor, rule: str):
    """x on the GPU against the definition; returns the tensor."""
    got = mx_quantize(x, rule)
    want_p, want_s = mx_ref.quantize(x.reshape(-1, x.shape[-1]).double().cpu().numpy(), rule)
    p, s = got.numpy()
    np.testing.assert_array_equal(s, want_s)
    # the sign of a zero that was rounded to is no part of the value
    np.testing.assert_array_equal(mx_ref.values(p, s), mx_ref.values(want_p, want_s))
    return got


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (37, 1024), (130, 160), (5, 2080)])
def test_random_rows(dev, rows, cols, dtype, rule):
    g = torch.Generator(device=dev).manual_seed(rows * cols)
    x = torch.randn(rows, cols, generator=g, device=dev) * torch.randn(rows, 1, generator=g, device=dev).exp()
    check(x.to(dtype), rule)


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("dtype", TYPES)
def test_every_half_step_and_its_neighbours(dev, dtype, rule):
    """All multiples of 1/8 up to 8 in blocks whose largest is fixed, so that every tie is met."""
    grid = torch.arange(0, 64, device=dev) / 8.0
    rows = [torch.cat([grid[i:i + 31], torch.tensor([top], device=dev)]) for i in (0, 31, 33) for top in (6.0, 4.0, 7.875)]
    x = torch.stack(rows)
    check(torch.cat([x, -x, x * 2.0 ** -9, x * 2.0 ** 7]).to(dtype), rule)


@pytest.mark.parametrize("rule", RULES)
def test_range_ends_fp32(dev, rule):
    tiny, big = 2.0 ** -149, 3.4e38
    rows = []
    for most in (0.0, tiny, 3 * tiny, 2.0 ** -127, 2.0 ** -126, 1.75 * 2.0 ** -126, 2.0 ** -125, 1.9 * 2.0 ** -125, 2.0 ** -124, 1e-30, 1.0, 2e38, big):
        f = torch.linspace(-1, 1, 32, dtype=torch.float64)
        rows.append((f * most).float())
    x = torch.stack(rows).to(dev)
    got = check(x, rule)
    assert got.scale[0].item() == 0  # zeros


@pytest.mark.parametrize("dtype,value", [(torch.float16, 2.0 ** -24), (torch.float16, 65504.0), (torch.bfloat16, 2.0 ** -133),
                                         (torch.bfloat16, 3.3895e38)])
@pytest.mark.parametrize("rule", RULES)
def test_range_ends_16_bits(dev, dtype, value, rule):
    x = (torch.linspace(-1, 1, 64, dtype=torch.float64) * value).to(dtype).reshape(2, 32).to(dev)
    check(x, rule)


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("dtype", TYPES)
def test_inf_and_nan_make_their_block_nan_alone(dev, dtype, rule):
    x = torch.randn(6, 128, device=dev).to(dtype)
    x[0, 0], x[1, 33], x[2, 95], x[3, 127] = float("inf"), float("-inf"), float("nan"), float("nan")
    got = check(x, rule)
    v = got.dequantize()
    assert v.isnan().sum().item() == 4 * 32
    for i, j in ((0, 0), (1, 1), (2, 2), (3, 3)):
        assert v[i, 32 * j:32 * j + 32].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_leading_dims(dev, dtype):
    wide = torch.randn(9, 256, device=dev).to(dtype)
    want = check(wide[:, 32:128].contiguous(), "floor")
    for view in (wide[:, 32:128],                                  # rows read in place
                 torch.cat([wide, wide[:, :8]], 1)[:, 32:128],     # another pitch
                 torch.cat([wide, wide[:, :1]], 1)[:, 32:128],     # rows that are not 16-byte aligned: copied
                 torch.cat([wide[:, :1], wide], 1)[:, 33:129],     # a base that is not
                 wide.t().contiguous().t()[:, 32:128]):            # columns side by side
        got = mx_quantize(view)
        assert torch.equal(got.packed, want.packed) and torch.equal(got.scale, want.scale)
    got = mx_quantize(wide[:, 32:128].reshape(3, 3, 96))
    assert got.shape == (9, 96) and torch.equal(got.packed, want.packed)
    got = mx_quantize(wide[4, 32:128])
    assert got.shape == (1, 96) and torch.equal(got.packed[0], want.packed[4])
    same = mx_quantize(wide[0:1, 32:64].expand(5, 32))  # one row five times
    assert (same.packed == same.packed[0]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_every_code_and_scale_comes_back(dev, dtype):
    """256 bytes x 256 scales: exact in fp32 and bf16, rounded once in fp16."""
    packed = np.tile(np.arange(256, dtype=np.uint8).reshape(16, 16), (256, 1))
    scale = np.repeat(np.arange(256, dtype=np.uint8), 16).reshape(-1, 1)
    got = MXTensor.from_numpy(packed, scale, device=dev).dequantize(dtype)
    want = torch.from_numpy(mx_ref.values(packed, scale)).to(dtype)  # one rounding
    assert got.dtype == dtype
    np.testing.assert_array_equal(got.float().cpu().numpy(), want.float().numpy())


@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 96), (33, 160), (70, 288), (1000, 1056)])
def test_pack_on_the_device_is_the_hosts(dev, rows, cols):
    p, s = mx_ref.random_mx(np.random.default_rng(cols), rows, cols)
    host, here = MXTensor.from_numpy(p, s), MXTensor.from_numpy(p, s, device=dev)
    p2, s2 = here.numpy()
    assert (p2 == p).all() and (s2 == s).all()
    back = here.to("cpu")
    assert all((a == b).all() for a, b in zip(back.numpy(), (p, s)))
    v = host.to(dev).dequantize().cpu().numpy()
    np.testing.assert_array_equal(v, mx_ref.values(p, s))


def test_pads_are_zeros_whatever_was_there(dev):
    """Columns past the last, which products read, in memory that held NaN scales."""
    junk = torch.full((1 << 20,), 255, dtype=torch.uint8, device=dev)
    del junk
    x = torch.randn(40, 160, device=dev)
    got = mx_quantize(x)
    rows = torch.arange(40, device=dev)
    sc = got.scales.view(2, 2, 32, 4).permute(0, 2, 1, 3).reshape(64, 8)[rows]
    codes = got.codes.view(2, 2, 4, 32, 16).permute(0, 3, 1, 2, 4).reshape(64, 8, 16)[rows]
    assert not sc[:, 5:].any() and not codes[:, 5:].any()


def test_a_large_matrix_and_its_last_rows(dev):
    """More groups than the grid has threads in a round."""
    x = torch.randn(40001, 1056, device=dev, dtype=torch.bfloat16)
    got = mx_quantize(x)
    for i in (0, 7943, 31776, 40000):
        p, s = mx_ref.quantize(x[i:i + 1].double().cpu().numpy())
        np.testing.assert_array_equal(got.scale[i].cpu().numpy(), s[0])
        np.testing.assert_array_equal(mx_ref.values(got.packed[i:i + 1].cpu().numpy(), s), mx_ref.values(p, s))
    v = got.dequantize(torch.bfloat16)
    err = (v.float() - x.float()).abs().view(40001, 33, 32)
    top = x.float().abs().view(40001, 33, 32).amax(-1, keepdim=True)
    # floor rule: 2^e >= top / 8, steps of 2^(e + 1) at most: off by 2^e <= top / 4, or by what lies past 6 2^e (< 2 2^e)
    assert (err <= top / 2).all()
