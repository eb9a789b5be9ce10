"""CPU: the 4-bit and distillation entry points refuse bad calls before they touch the GPU."""
import ctypes

import pytest
import torch

import lira_amd
from lira_amd import _lib

P = ctypes.c_void_p
A = 4096  # an aligned address that is never read: every call below ends before a launch


def lib():
    return _lib.load()


def why() -> str:
    return lib().lira_last_error().decode()


@pytest.mark.parametrize("change,code,text", [
    ({"dtype": 9}, -1, "dtype"), ({"n": -1}, -1, "rows"), ({"k": 0}, -1, "k >= 1"), ({"ld": 99}, -1, "ld must"),
    ({"plane_rows": 7}, -1, "plane_rows"), ({"codes": None}, -1, "NULL"), ({"scales": None}, -1, "NULL"),
    ({"x": None}, -1, "NULL"), ({"codes": A + 8}, -1, "aligned"), ({"scales": A + 2}, -1, "aligned"),
    ({"k": 65535 * 128 + 1, "ld": 1 << 40}, -6, "k must"), ({"n": 1 << 60, "plane_rows": 1 << 60}, -6, "too many rows"),
])
def test_pack_refusals(change, code, text):
    a = dict(x=A, dtype=0, n=8, k=100, ld=100, codes=A, scales=A, plane_rows=8) | change
    assert lib().lira_mx4_quantize(a["x"], a["dtype"], a["n"], a["k"], a["ld"], a["codes"], a["scales"], a["plane_rows"], None) == code
    assert text in why()
    assert lib().lira_mx4_dequantize(a["codes"], a["scales"], a["plane_rows"], a["n"], a["k"], a["x"], a["dtype"], a["ld"], None) == code
    assert text in why()


@pytest.mark.parametrize("change,code,text", [
    ({"dtype": -1}, -1, "dtype"), ({"out_dtype": 3}, -1, "dtype"), ({"act": 5}, -1, "activation"), ({"ldx": 63}, -1, "ldx"),
    ({"ldo": 31}, -1, "ldo"), ({"out": None}, -1, "NULL"), ({"x": None}, -1, "NULL"), ({"codes": None}, -1, "NULL"),
    ({"m": -1}, -1, "shape"), ({"n": -1}, -1, "rows"), ({"b_rows": 5}, -1, "plane_rows"), ({"k": 0}, -1, "k >= 1"),
    ({"m": 1 << 40}, -6, "too many rows"), ({"n": 1 << 40, "b_rows": 1 << 40, "ldo": 1 << 40}, -6, "too many rows"),
    ({"m": 200, "ws": None}, -1, "workspace"), ({"m": 200, "wsb": 16}, -1, "workspace"), ({"m": 200, "ws": A + 4}, -1, "workspace"),
])
def test_linear_refusals(change, code, text):
    a = dict(x=A, dtype=0, m=16, k=64, ldx=64, codes=A, scales=A, b_rows=32, n=32, act=0, out=A, out_dtype=0, ldo=32, ws=A,
             wsb=1 << 40) | change
    assert lib().lira_mx4_linear(a["x"], a["dtype"], a["m"], a["k"], a["ldx"], a["codes"], a["scales"], a["b_rows"], a["n"], 1.0,
                                 None, a["act"], a["out"], a["out_dtype"], a["ldo"], a["ws"], a["wsb"], None) == code
    assert text in why()


def test_matmul_refusals_and_empty_calls():
    f = lib().lira_mx4_matmul
    assert f(A, A, 4, 8, A, A, 32, 32, 64, 1.0, None, 0, A, 0, 32, None) == -1 and "plane_rows" in why()
    assert f(A, A, 8, 8, A, A, 32, 32, 64, 1.0, None, 0, A, 0, 31, None) == -1 and "ldo" in why()
    assert f(A, A, 8, 8, A, A, 32, 32, 64, 1.0, None, 9, A, 0, 32, None) == -1 and "activation" in why()
    assert f(None, None, 0, 0, A, A, 32, 32, 64, 1.0, None, 0, None, 0, 32, None) == 0
    assert f(A, A, 8, 8, None, None, 0, 0, 64, 1.0, None, 0, None, 0, 0, None) == 0
    n = ctypes.c_size_t(1)
    assert lib().lira_mx4_linear_workspace_size(0, 10, 64, ctypes.byref(n)) == 0 and n.value == 0
    assert lib().lira_mx4_linear_workspace_size(1000, 10, 129, ctypes.byref(n)) == 0 and n.value == 2 * 1000 * 68
    assert lib().lira_mx4_linear_workspace_size(10, 10, 0, ctypes.byref(n)) == -1
    assert lib().lira_mx4_linear_workspace_size(10, 10, 64, None) == -1


@pytest.mark.parametrize("change,code,text", [
    ({"dtype": 4}, -1, "dtype"), ({"bits": 16}, -1, "ids_bits"), ({"rows": -1}, -1, "rows"), ({"vocab": 0}, -1, "vocab"),
    ({"top": 0}, -1, "top"), ({"top": -3}, -1, "top"), ({"top": 1025}, -6, "top"), ({"ldz": 99}, -1, "strides"),
    ({"ldd": 99}, -1, "strides"), ({"t": 0.0}, -1, "temperature"), ({"t": float("inf")}, -1, "temperature"),
    ({"t": float("nan")}, -1, "temperature"), ({"stride": 2}, -1, "scale_stride"), ({"rows": 1 << 31}, -6, "too many rows"),
    ({"z": None}, -1, "NULL"), ({"ids": None}, -1, "NULL"), ({"tv": None}, -1, "NULL"), ({"out": None}, -1, "NULL"),
])
def test_distill_refusals(change, code, text):
    a = dict(z=A, dtype=0, rows=4, vocab=100, ldz=100, ids=A, bits=32, tv=A, top=5, t=1.0, out=A, stride=1, ldd=100) | change
    head = (a["z"], a["dtype"], a["rows"], a["vocab"], a["ldz"], a["ids"], a["bits"], a["tv"], a["top"], a["t"], None)
    assert lib().lira_distill_topk(*head, a["out"], None, A, a["stride"], A, a["ldd"], A, 1 << 40, None) == code
    assert text in why()
    assert lib().lira_distill_topk_backward(*head, a["out"], A, a["stride"], A, a["ldd"], None) == code
    assert text in why()


def test_distill_empty_and_reduce():
    head = (None, 0, 0, 100, 100, None, 32, None, 5, 1.0, None)
    assert lib().lira_distill_topk(*head, None, None, None, 0, None, 0, None, 0, None) == 0
    assert lib().lira_distill_topk_backward(*head, None, None, 0, A, 100, None) == 0
    few = (A, 1, 2, 100000, 100000, A, 32, A, 5, 1.0, None, A, None, None, 0, A, 100000)  # (split over the chip)
    need = ctypes.c_size_t()
    assert lib().lira_distill_workspace_size(2, 100000, 5, 1, ctypes.byref(need)) == 0 and need.value > 0
    for ws, n in ((None, 1 << 40), (A, need.value - 1), (A + 4, 1 << 40)):
        assert lib().lira_distill_topk(*few, ws, n, None) == -1 and "workspace" in why()
    assert lib().lira_distill_workspace_size(2, 0, 5, 1, ctypes.byref(need)) == -1
    assert lib().lira_distill_workspace_size(2, 10, 5, 7, ctypes.byref(need)) == -1
    assert lib().lira_distill_workspace_size(2, 10, 5, 0, None) == -1
    assert lib().lira_distill_topk(A, 0, 4, 10, 10, A, 32, A, 5, 1.0, None, A, A + 8, None, 0, A, 10, None, 0, None) == -1
    assert "stats" in why()
    assert lib().lira_distill_reduce(A, A, -1, 0, A, None) == -1
    assert lib().lira_distill_reduce(None, A, 3, 0, A, None) == -1
    assert lib().lira_distill_reduce(A, A, 3, 0, None, None) == -1


def test_python_refuses_host_tensors():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="on the GPU"):
        lira_amd.mx4_quantize(x)
    with pytest.raises(ValueError, match="on the GPU"):
        lira_amd.MX4Tensor(torch.zeros(1, 4, 64, dtype=torch.uint8), torch.zeros(1, 4, 4, dtype=torch.uint8), 64)
    with pytest.raises(ValueError, match="MX4Tensor"):
        lira_amd.mx4_linear(x, x)
    with pytest.raises(ValueError, match="MX4Tensor"):
        lira_amd.mx4_matmul(x, x)
    with pytest.raises(ValueError, match="MX4Tensor"):
        lira_amd.mx4_dequantize(x)
    ids = torch.zeros(4, 2, dtype=torch.int64)
    for f in (lira_amd.distill_topk_loss, lira_amd.distill_topk_loss_and_grad):
        with pytest.raises(ValueError, match="on the GPU"):
            f(x, ids, torch.zeros(4, 2))
    with pytest.raises(ValueError, match="reduction"):
        lira_amd.distill_topk_loss(x, ids, torch.zeros(4, 2), reduction="max")
