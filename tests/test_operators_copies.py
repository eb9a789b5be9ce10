"""CPU: packed rows that are copied, pickled or saved hold the addresses of their own memory."""
import copy
import io
import pickle

import pytest
import torch

from lira_amd import MX4Tensor, mx4_dequantize


def packed(n=5, k=300):
    """Packed rows over a host buffer (as mx4_quantize makes them over one on the GPU): never given to a kernel."""
    buf = (torch.arange((k + 127) // 128 * n * 68) % 251).to(torch.uint8)
    return MX4Tensor._of(buf, n, k)


def saved(t):
    f = io.BytesIO()
    torch.save(t, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


HOW = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda t: pickle.loads(pickle.dumps(t)), "save": saved,
       "pickle2": lambda t: pickle.loads(pickle.dumps(t, 2))}


@pytest.mark.parametrize("how", list(HOW))
@pytest.mark.parametrize("n,k", [(5, 300), (1, 128), (3, 1), (0, 129)])
@pytest.mark.parametrize("looked_at", [False, True])
def test_copies_point_at_their_own_memory(how, n, k, looked_at):
    t = packed(n, k)
    if looked_at:  # (the two views of the buffer are made when they are asked for)
        t.codes, t.scales
    c = HOW[how](t)
    assert c.codes_ptr == c.codes.data_ptr() and (n == 0 or c.scales_ptr == c.scales.data_ptr())
    assert (c.n, c.k, c.shape, c.plane_rows, c.device) == (t.n, t.k, t.shape, t.plane_rows, t.device)
    assert torch.equal(c.codes, t.codes) and torch.equal(c.scales, t.scales)
    if n and how != "copy":
        assert c.codes_ptr != t.codes_ptr and c.scales_ptr != t.scales_ptr
        was = t.codes.clone()
        c.codes.zero_()
        assert torch.equal(t.codes, was)


@pytest.mark.parametrize("how", list(HOW))
def test_copies_of_a_range_of_rows(how):
    t = packed(9, 300)
    v = MX4Tensor.__getitem__(t, slice(2, 6))
    c = HOW[how](v)
    assert v.codes_ptr == t.codes_ptr + 2 * 64 and v.scales_ptr == t.scales_ptr + 2 * 4 and v.plane_rows == 9
    assert c.codes_ptr == c.codes.data_ptr() and c.scales_ptr == c.scales.data_ptr()
    assert torch.equal(c.codes, v.codes) and torch.equal(c.scales, v.scales) and c.shape == (4, 300)
    assert c.plane_rows >= 4 and c.codes.stride(0) == c.plane_rows * 64 and c.scales.stride(0) == c.plane_rows * 4


def test_addresses_follow_their_tensors():
    t = packed()
    other = torch.ones_like(t.codes)
    t.codes.set_(other)
    assert t.codes_ptr == other.data_ptr()


def test_rows_in_host_memory_reach_no_kernel():
    """As torch.load(map_location="cpu") leaves them."""
    t = packed()
    with pytest.raises(ValueError, match="on the GPU"):
        mx4_dequantize(t)
    with pytest.raises(ValueError, match="on the GPU"):
        t.dequantize()
