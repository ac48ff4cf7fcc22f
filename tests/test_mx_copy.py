"""MXTensors are copied and pickled as Q4 tensors are: the copy has memory of its own, and a descriptor of that memory."""

import copy
import io
import pickle

import numpy as np
import pytest
import torch

import mx_ref
from llm_accelerator_amd.mx import MXTensor, mx_linear, mx_quantize, mx_score


def pickled(t):
    return pickle.loads(pickle.dumps(t))


def saved(t):
    f = io.BytesIO()
    torch.save(t, f)
    f.seek(0)
    return torch.load(f, weights_only=False)  # (of this test's own making)


def own(t):
    """The descriptor points into the tensor's memory: codes, then scales."""
    return (t._desc.w == t.codes.data_ptr() and t._desc.s == t.scales.data_ptr() and (t._desc.rows, t._desc.cols) == tuple(t.shape)
            and t._ref._obj is t._desc)


@pytest.mark.parametrize("way", [copy.deepcopy, pickled, saved])
def test_copies_on_the_host(way):
    p, s = mx_ref.random_mx(np.random.default_rng(0), 37, 160)
    a = MXTensor.from_numpy(p, s)
    b = way(a)
    assert type(b) is MXTensor and b.shape == (37, 160) and own(a) and own(b) and b._desc.w != a._desc.w
    assert b._index == -1 and all((u == v).all() for u, v in zip(b.numpy(), (p, s)))
    b._memory.zero_()
    assert all((u == v).all() for u, v in zip(a.numpy(), (p, s)))


def test_a_shallow_copy_shares_the_memory():
    a = MXTensor.from_numpy(*mx_ref.random_mx(np.random.default_rng(1), 5, 32))
    b = copy.copy(a)
    assert b is not a and b._memory is a._memory and own(b)


def test_one_tensor_in_two_places_stays_one():
    a = MXTensor.from_numpy(*mx_ref.random_mx(np.random.default_rng(2), 5, 32))
    both = copy.deepcopy({"head": a, "table": a})
    assert both["head"] is both["table"] and both["head"] is not a


@pytest.mark.gpu
@pytest.mark.parametrize("way", [copy.deepcopy, pickled, saved])
def test_copies_on_the_device(dev, way):
    rng = np.random.default_rng(3)
    a = mx_quantize(torch.from_numpy(rng.standard_normal((300, 96))).to(dev).float())
    x = torch.from_numpy(rng.standard_normal((7, 96))).to(dev).to(torch.bfloat16)
    t = torch.from_numpy(rng.integers(0, 300, 7)).to(dev).int()

    def results(w):
        return [mx_linear(x, w), mx_linear(mx_quantize(x), w), *mx_score(x, w, t), w.dequantize(), w.packed, w.scale]
    want = [v.clone() for v in results(a)]
    b = way(a)
    assert b.device == a.device and own(b) and b._desc.w != a._desc.w
    a._memory.zero_()
    assert all(torch.equal(u, v) for u, v in zip(results(b), want))
