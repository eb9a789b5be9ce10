"""GPU: what the 4-bit and distillation operators read and write, as other parts of a program see it: copies of
packed rows, outputs that autograd has saved, shared memory, streams, modules' state."""
import copy
import io
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def saved(t):
    f = io.BytesIO()
    torch.save(t, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("how", [copy.deepcopy, lambda t: pickle.loads(pickle.dumps(t)), saved])
def test_copies_outlive_their_original(how):
    from lira_amd import IndexMX4, mx4_linear, mx4_matmul, mx4_quantize
    x, q = torch.randn(70, 300, generator=gen(1), device="cuda"), torch.randn(20, 300, generator=gen(2), device="cuda")
    t = mx4_quantize(x)
    want = [t.dequantize(), mx4_linear(q, t), mx4_matmul(mx4_quantize(q), t), t[5:9].dequantize()]
    c, part = how(t), how(t[5:9])
    t.codes.zero_()  # (what the original's memory may hold once it is gone)
    t.scales.zero_()
    del t
    got = [c.dequantize(), mx4_linear(q, c), mx4_matmul(mx4_quantize(q), c), part.dequantize()]
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    idx = IndexMX4(300)
    idx.add(x)
    D, I = idx.search(q, 5)
    other = how(idx)
    idx._packed().codes.zero_()
    idx._packed().scales.zero_()
    D2, I2 = other.search(q, 5)
    assert torch.equal(D, D2) and torch.equal(I, I2)
