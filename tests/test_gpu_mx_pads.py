"""What quantisation and packing write of a matrix's memory, over memory that holds 255 (NaN scales) everywhere: every
column of the rows that there are, zeros past the last, nothing outside."""

import numpy as np
import pytest
import torch

import mx_ref
from llm_accelerator_amd._lib import Q4D_BF16, Q4D_F16, Q4D_F32
from llm_accelerator_amd.model import call_on
from llm_accelerator_amd.mx import MXTensor, mx_linear, mx_score

pytestmark = pytest.mark.gpu
GUARD = 4096


def over_junk(rows, cols, dev):
    """(MXTensor over memory of 255, the memory with room on both sides)."""
    size = -(-rows // 32) * -(-cols // 128) * 2176
    room = torch.full((size + 2 * GUARD,), 255, dtype=torch.uint8, device=dev)
    return MXTensor.__new__(MXTensor)._setup(room[GUARD:GUARD + size], rows, cols), room


def check(t, room, packed, scale):
    rows, cols = t.shape
    rt, kt, n = -(-rows // 32), -(-cols // 128), cols // 32
    assert (room[:GUARD] == 255).all() and (room[-GUARD:] == 255).all()
    codes = t.codes.view(rt, kt, 4, 32, 16).permute(0, 3, 1, 2, 4).reshape(rt * 32, 4 * kt, 16)
    scales = t.scales.view(rt, kt, 32, 4).permute(0, 2, 1, 3).reshape(rt * 32, 4 * kt)
    assert not codes[:rows, n:].any() and not scales[:rows, n:].any()
    got = codes[:rows, :n].reshape(rows, cols // 2).cpu().numpy()
    assert (scales[:rows, :n].cpu().numpy() == scale).all()
    assert (mx_ref.values(got, scale) == mx_ref.values(packed, scale)).all()


SIZES = [(1, 32), (31, 96), (33, 160), (40, 160), (64, 256), (70, 288), (1, 1056)]


@pytest.mark.parametrize("dtype,code", [(torch.float32, Q4D_F32), (torch.float16, Q4D_F16), (torch.bfloat16, Q4D_BF16)])
@pytest.mark.parametrize("rule", [0, 1])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantise(dev, rows, cols, dtype, code, rule):
    x = torch.from_numpy(np.random.default_rng(cols).standard_normal((rows, cols))).to(dev).to(dtype)
    t, room = over_junk(rows, cols, dev)
    call_on(0, "q4d_mx_quantize", x.data_ptr(), code, cols, rule, t._ref)
    check(t, room, *mx_ref.quantize(x.double().cpu().numpy(), ("floor", "ceil")[rule]))


@pytest.mark.parametrize("rows,cols", SIZES)
def test_pack(dev, rows, cols):
    p, s = mx_ref.random_mx(np.random.default_rng(cols), rows, cols)
    t, room = over_junk(rows, cols, dev)
    packed, scale = torch.from_numpy(p).to(dev), torch.from_numpy(s).to(dev)
    call_on(0, "q4d_mx_pack", packed.data_ptr(), scale.data_ptr(), t._ref)
    check(t, room, p, s)


@pytest.mark.parametrize("m,n,k", [(3, 70, 160), (61, 4101, 1056), (300, 4105, 288), (1001, 6147, 224), (2161, 8201, 416), (17, 50001, 96)])
def test_products_of_matrices_over_junk(dev, m, n, k):
    """Rows past the last stay NaN: no product and no score takes anything from there."""
    rng = np.random.default_rng(n)
    pw, sw = mx_ref.random_mx(rng, n, k)
    px, sx = mx_ref.random_mx(rng, m, k, 122, 130)
    w, room_w = over_junk(n, k, dev)
    x, room_x = over_junk(m, k, dev)
    for t, p, s in ((w, pw, sw), (x, px, sx)):
        packed, scale = torch.from_numpy(p).to(dev), torch.from_numpy(s).to(dev)
        call_on(0, "q4d_mx_pack", packed.data_ptr(), scale.data_ptr(), t._ref)
    clean_w, clean_x = MXTensor.from_numpy(pw, sw, device=dev), MXTensor.from_numpy(px, sx, device=dev)
    for kind in (torch.bfloat16, torch.float16):
        wide = clean_x.dequantize(kind)
        targets = torch.from_numpy(rng.integers(0, n, m)).to(dev).int()
        for a, b in ((mx_linear(x, w, out_dtype=torch.float32), mx_linear(clean_x, clean_w, out_dtype=torch.float32)),
                     (mx_linear(wide, w), mx_linear(wide, clean_w)), *zip(mx_score(wide / 64, w, targets), mx_score(wide / 64, clean_w, targets))):
            assert torch.equal(a, b) and a.isfinite().all()
