"""Every form of the product kernels at ragged sizes against products in 64 bits: the sizes are chosen by the rules that
choose the kernel, and a test without a device says that no form is left out.  Bounds: see test_gpu_mx_linear."""

import numpy as np
import pytest
import torch

import mx_ref
import mx_shim
from llm_accelerator_amd.mx import MXTensor, mx_linear, mx_score

# (m, n, k): the form that x in 16 bits takes / in 4 bits
R, H, T = "rows", "head", "tiles"
SHAPES = {
    (5, 300, 96): [(R, 1, 1, 4)] * 2,
    (3, 511, 1056): [(R, 1, 1, 8)] * 2,
    (16, 1000, 2080): [(R, 1, 1, 8)] * 2,
    (5, 6147, 1024): [(R, 1, 2, 4)] * 2,
    (15, 8200, 160): [(R, 1, 2, 4)] * 2,
    (5, 6147, 1056): [(R, 1, 2, 8)] * 2,
    (2, 32770, 2080): [(R, 1, 2, 8)] * 2,
    (7, 33001, 160): [(R, 1, 4, 4)] * 2,
    (15, 49157, 224): [(R, 1, 4, 4)] * 2,
    (20, 4203, 224): [(R, 2, 2, 4)] * 2,
    (30, 8195, 1056): [(R, 2, 2, 8)] * 2,
    (22, 33003, 1056): [(R, 2, 2, 8)] * 2,
    (21, 33002, 96): [(R, 2, 4, 4)] * 2,
    (61, 8195, 1024): [(R, 4, 2, 4)] * 2,
    (150, 4100, 160): [(R, 4, 2, 4)] * 2,
    (61, 8195, 2080): [(R, 4, 2, 8)] * 2,
    (150, 4101, 1056): [(R, 4, 2, 8)] * 2,
    (16, 50003, 1056): [(H, 1, 2, 8), (R, 1, 2, 8)],
    (27, 60001, 224): [(H, 2, 2, 8), (T, 2, 1, 4)],
    (21, 151931, 96): [(H, 2, 2, 10), (T, 4, 2, 4)],
    (300, 4104, 416): [(T, 2, 1, 4)] * 2,           # (n: pieces of 16 bytes in every type)
    (259, 4102, 32): [(T, 2, 1, 4)] * 2,            # a stage of 32 columns alone
    (300, 4105, 1056): [(T, 2, 1, 4)] * 2,
    (1001, 6147, 224): [(T, 2, 2, 4)] * 2,
    (1000, 6152, 96): [(T, 2, 2, 4)] * 2,
    (1025, 6148, 160): [(T, 2, 2, 4)] * 2,          # of 16 bytes in fp32, of 8 in 16 bits
    (1000, 6150, 1056): [(T, 2, 2, 4)] * 2,
    (1100, 6144, 32): [(T, 2, 2, 4)] * 2,
    (1037, 6400, 128): [(T, 2, 2, 4)] * 2,
    (129, 131100, 160): [(T, 2, 2, 4), (T, 4, 2, 4)],
    (4100, 4200, 288): [(T, 2, 2, 4), (T, 4, 2, 4)],
    (2161, 8201, 416): [(T, 2, 2, 4), (T, 4, 2, 4)],
    (2049, 8196, 32): [(T, 2, 2, 4), (T, 4, 2, 4)],
}
SCORES = {
    (5, 301, 96): (R, 1, 4, 4), (16, 33001, 4128): (R, 1, 4, 4), (31, 20003, 1056): (R, 2, 4, 4), (32, 34000, 32): (R, 2, 4, 4),
    (33, 33331, 160): (R, 4, 2, 4), (64, 8195, 2080): (R, 4, 2, 4), (9, 49153, 1056): (H, 1, 2, 8), (31, 50007, 288): (H, 2, 2, 8),
    (65, 257, 96): (T, 2, 2, 4), (40, 60001, 32): (T, 2, 2, 4), (1001, 6147, 224): (T, 2, 2, 4), (190, 50001, 1056): (T, 2, 2, 4),
}
# every form that a launch can have
PRODUCTS = {(R, 1, 1, 4), (R, 1, 1, 8), (R, 1, 2, 4), (R, 1, 2, 8), (R, 1, 4, 4), (R, 2, 2, 4), (R, 2, 2, 8), (R, 2, 4, 4), (R, 4, 2, 4),
            (R, 4, 2, 8), (T, 2, 1, 4), (T, 2, 2, 4)}


def without_waves(forms):
    """The head kernel is one for all waves."""
    return {f[:3] if f[0] == H else f for f in forms}


def test_sizes_take_the_forms_that_they_stand_for():
    for size, (wide, codes) in SHAPES.items():
        assert mx_shim.form(*size, False) == wide and mx_shim.form(*size, True) == codes, size
    for size, want in SCORES.items():
        assert mx_shim.score_form(*size) == want, size


def test_no_form_is_left_out():
    """The forms of sizes of all kinds are those above, and each is among the sizes tested."""
    rng = np.random.default_rng(0)
    seen = {False: set(), True: set()}
    scored = set()
    edges = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000, 4096, 65536]
    for m in edges + [int(2 ** v) for v in rng.uniform(0, 18, 60)]:
        for n in [1, 16, 4096, 4097, 32767, 32768, 49151, 49152, 151936, 1 << 20] + [int(2 ** v) for v in rng.uniform(0, 21, 60)]:
            for k in (32, 1024, 1056, 4096, 8192):
                for codes in (False, True):
                    seen[codes].add(mx_shim.form(m, n, k, codes))
                scored.add(mx_shim.score_form(m, n, k))
    assert without_waves(seen[False]) == PRODUCTS | {(H, 1, 2), (H, 2, 2)}
    assert without_waves(seen[True]) == PRODUCTS | {(T, 4, 2, 4)}
    assert without_waves(seen[False]) == without_waves(f[0] for f in SHAPES.values())
    assert without_waves(seen[True]) == without_waves(f[1] for f in SHAPES.values())
    assert without_waves(scored) == without_waves(SCORES.values())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, "mx"])
@pytest.mark.parametrize("m,n,k", list(SHAPES))
def test_products(dev, m, n, k, kind):
    from test_gpu_mx_linear import compare, make
    rng = np.random.default_rng(3 * m + 5 * n + 11 * k)
    w, wv = make(rng, n, k, dev)
    if kind == "mx":
        x, xv = make(rng, m, k, dev, 122, 130)
    else:
        x = torch.from_numpy(rng.standard_normal((m, k))).to(dev).to(kind)
        xv = x.double()
    for out in (torch.float32, torch.float16, torch.bfloat16):
        # a result with room around it, which stays as it was
        room = torch.full((m * n + 512,), 7.0, device=dev, dtype=out)
        y = room[256:256 + m * n].view(m, n)
        mx_linear(x, w, out=y)
        compare(y, xv, wv)
        assert (room[:256] == 7).all() and (room[256 + m * n:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", list(SCORES))
def test_scores(dev, m, n, k, kind):
    from test_gpu_mx_score import check
    rng = np.random.default_rng(m + n + k)
    p, s = mx_ref.random_mx(rng, n, k, 121, 125)
    w = MXTensor.from_numpy(p, s, device=dev)
    x = torch.from_numpy(rng.standard_normal((m, k)) / np.sqrt(k) * 8).to(dev).to(kind)
    targets = torch.from_numpy(rng.integers(0, n, m)).to(dev).int()
    targets[0], targets[-1] = 0, n - 1
    check(mx_score(x, w, targets), x, w.dequantize().double(), targets)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(61, 8195, 1056), (1001, 6147, 224), (4100, 4200, 288), (150, 4100, 160)])
def test_nan_stays_in_its_rows_and_outputs(dev, m, n, k):
    """A NaN block of x and one of the weights in each form of many rows: their row and output alone, also where tiles
    hold rows past the last."""
    rng = np.random.default_rng(k)
    ps, ss = mx_ref.random_mx(rng, n, k)
    px, sx = mx_ref.random_mx(rng, m, k, 122, 130)
    clean = {}
    for kind in ("mx", torch.bfloat16):
        for bad in (False, True):
            if bad:
                ss[n - 1, -1] = sx[m - 1, 0] = 255
            else:
                ss[n - 1, -1] = sx[m - 1, 0] = 125
            w = MXTensor.from_numpy(ps, ss, device=dev)
            x = MXTensor.from_numpy(px, sx, device=dev)
            y = mx_linear(x if kind == "mx" else x.dequantize(kind), w, out_dtype=torch.float32)
            if not bad:
                clean[kind] = y
                assert y.isfinite().all()
            else:
                assert y[m - 1].isnan().all() and y[:, n - 1].isnan().all()
                assert torch.equal(y[:m - 1, :n - 1], clean[kind][:m - 1, :n - 1])
