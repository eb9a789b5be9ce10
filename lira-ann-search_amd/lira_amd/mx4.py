"""Microscaled 4-bit floats: packed rows, and their products on the matrix cores.

Stored vectors and the probing model's layers in 4.25 bits an element: 32 elements share a
power-of-two scale (include/lira_hip.h has the layout and the rounding).  A row of d = 128
takes 68 bytes, where the reference's fp32 copy (search.cpp:387-403) takes 512.

* ``mx4_quantize`` / ``MX4Tensor.dequantize``   pack rows and read them back
* ``mx4_matmul``   act(alpha * A B^T + bias) of two packed arrays
* ``mx4_linear``   the same with fp32 / bf16 / fp16 rows that are packed on the way

All of them run on the current stream (or ``stream=``: what they read must be ready there; inputs may
be dropped after the call, results belong to that stream), allocate nothing that outlives the call but
their results, and can be captured into a graph.  They have no gradient: an input that asks
for one is refused.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools

import torch
from torch.autograd.graph import increment_version

from . import _lib

DTYPES = {torch.float32: _lib.LIRA_DTYPE_F32, torch.bfloat16: _lib.LIRA_DTYPE_BF16,
          torch.float16: _lib.LIRA_DTYPE_F16}
ACTIVATIONS = {None: _lib.LIRA_ACT_NONE, "relu": _lib.LIRA_ACT_RELU, "sigmoid": _lib.LIRA_ACT_SIGMOID}


# the current stream of a device as an address, without a torch.cuda.Stream object for it (3 us a call)
raw_stream = torch._C._cuda_getCurrentRawStream
_HERE = contextlib.nullcontext()


def on(device: torch.device, stream=None):
    """The context a call runs in: the tensors' device, and ``stream`` as the current one, so that
    whatever the call allocates belongs to the stream that uses it."""
    if device.type != "cuda":
        raise ValueError(f"the tensors must be on the GPU, not on {device}")
    if stream is not None:
        if stream.device != device:
            raise ValueError(f"stream is on {stream.device}, the tensors are on {device}")
        return torch.cuda.stream(stream)
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def keep_for(stream, *tensors) -> None:
    """A call on a stream of its own: the memory that it reads or writes belongs to other streams, which must not give
    it out again before the call is through."""
    for t in tensors:
        if isinstance(t, MX4Tensor):
            keep_for(stream, t._buf, t._codes, t._scales)
        elif t is not None:
            t.record_stream(stream)


def check_rows(x, name: str, device=None) -> torch.Tensor:
    """A 2-D device tensor of a float type the kernels read; copied only if its rows are not runs of
    consecutive elements."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{name} must be a tensor on the GPU")
    if x.dtype not in DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {x.dtype}")
    if x.dim() != 2:
        raise ValueError(f"{name} must have 2 dimensions, not {x.dim()}")
    if device is not None and x.device != device:
        raise ValueError(f"{name} is on {x.device}, not on {device}")
    return x


def _rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """x with consecutive elements in its rows, and its row stride."""
    n, k = x.shape
    s0, s1 = x.stride()
    if s1 == 1 and (s0 >= k or n <= 1):
        return x, k if n <= 1 else s0
    x = x.contiguous()
    return x, k


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The addresses from t's first element to past its last one."""
    at = t.data_ptr()
    if t.is_contiguous():  # (an empty one is)
        return at, at + t.nbytes
    return at, at + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def refuse_shared(out: torch.Tensor, name: str, *inputs) -> None:
    """An output may not lie over an input (a tensor or None), which other workgroups still read."""
    lo, hi = _span(out)
    for t in inputs:
        if t is not None:
            a, b = _span(t)
            if lo < b and a < hi:
                raise ValueError(f"{name} must not share memory with an input")


def _no_grad(t) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("the 4-bit operators have no gradient: call them under torch.no_grad() or on detached tensors")


class MX4Tensor:
    """Packed rows: ``codes`` (P, n, 64) uint8, ``scales`` (P, n, 4) uint8, P = ceil(k / 128)
    planes of 128 elements (include/lira_hip.h).  Row ranges ``t[lo:hi]`` are views.  Copies (``copy``,
    ``pickle``, ``torch.save``) are of the two tensors and k."""

    # (what mx4_quantize packs is one buffer, whose two views are made when they are asked for; addresses are
    # read from the tensors at each call, never kept beside them)
    __slots__ = ("_codes", "_scales", "_buf", "k", "n", "plane_rows", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, k: int):
        for t, w, name in ((codes, 64, "codes"), (scales, 4, "scales")):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise ValueError(f"{name} must be a (P, n, {w}) uint8 tensor on the GPU")
        self._set(codes, scales, int(k))

    def _set(self, codes: torch.Tensor, scales: torch.Tensor, k: int) -> None:
        for t, w, name in ((codes, 64, "codes"), (scales, 4, "scales")):
            if t.dtype != torch.uint8 or t.dim() != 3 or t.shape[2] != w:
                raise ValueError(f"{name} must be a (P, n, {w}) uint8 tensor on the GPU")
        p, n, _ = codes.shape
        if k < 1 or p != (k + 127) // 128:
            raise ValueError(f"k = {k} needs {(max(k, 1) + 127) // 128} planes, codes have {p}")
        if scales.shape[0] != p or scales.shape[1] != n or codes.device != scales.device:
            raise ValueError("codes and scales must have the same planes and rows, on one device")
        rows = self._plane_rows(codes)
        if rows is None or rows != self._plane_rows(scales) or codes.data_ptr() % 16 or scales.data_ptr() % 4:
            codes, scales = codes.clone(memory_format=torch.contiguous_format), \
                scales.clone(memory_format=torch.contiguous_format)
            rows = n
        self._codes, self._scales, self._buf = codes, scales, None
        self.k, self.n, self.plane_rows, self.device = k, n, rows, codes.device

    @classmethod
    def _of(cls, buf: torch.Tensor, n: int, k: int) -> "MX4Tensor":
        """Of one buffer: the codes, then the scales."""
        t = object.__new__(cls)
        t._codes = t._scales = None
        t._buf, t.k, t.n, t.plane_rows, t.device = buf, k, n, n, buf.device
        return t

    def __reduce__(self):
        return _restored, (self.codes, self.scales, self.k)

    def addresses(self) -> tuple[int, int]:
        """Of the codes and of the scales."""
        codes, scales = self._codes, self._scales
        at = (self._buf if codes is None else codes).data_ptr()
        if scales is not None:
            return at, scales.data_ptr()
        return at, (at if codes is None else self._buf.data_ptr()) + (self.k + 127) // 128 * self.n * 64

    @property
    def codes_ptr(self) -> int:
        return self.addresses()[0]

    @property
    def scales_ptr(self) -> int:
        return self.addresses()[1]

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            p = (self.k + 127) // 128
            self._codes = self._buf[:p * self.n * 64].view(p, self.n, 64)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            p = (self.k + 127) // 128
            self._scales = self._buf[p * self.n * 64:].view(p, self.n, 4)
        return self._scales

    @staticmethod
    def _plane_rows(t: torch.Tensor):
        p, n, w = t.shape
        if t.is_contiguous():
            return n
        if t.stride(2) != 1 or (n > 1 and t.stride(1) != w):
            return None
        if p == 1:
            return n
        return t.stride(0) // w if t.stride(0) % w == 0 and t.stride(0) >= n * w else None

    @property
    def shape(self) -> tuple[int, int]:
        return self.n, self.k

    def nbytes(self) -> int:
        return (self.k + 127) // 128 * self.n * 68

    def __len__(self) -> int:
        return self.n

    def __getitem__(self, rows: slice) -> "MX4Tensor":
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise TypeError("an MX4Tensor is cut by a range of rows, t[lo:hi]")
        return _restored(self.codes[:, rows], self.scales[:, rows], self.k)

    def dequantize(self, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
                   stream=None) -> torch.Tensor:
        """The rows as numbers, (n, k): exact in float32, rounded once to the 16-bit types."""
        return mx4_dequantize(self, dtype, out, stream)


def _restored(codes: torch.Tensor, scales: torch.Tensor, k: int) -> MX4Tensor:
    """What copies, and views of rows, are made by: on whatever device the tensors are (torch.load may have put them
    into host memory, where no operator takes them)."""
    t = object.__new__(MX4Tensor)
    t._set(codes, scales, k)
    return t


def mx4_quantize(x: torch.Tensor, stream=None) -> MX4Tensor:
    """Pack the rows of x (n, k), float32 / bfloat16 / float16 (lira_mx4_quantize)."""
    x = check_rows(x, "x")
    _no_grad(x)
    n, k = x.shape
    if k < 1:
        raise ValueError("x must have at least one column")
    p = (k + 127) // 128
    dev = x.device
    with on(dev, stream):
        if stream is not None:
            keep_for(stream, x)
        x, ld = _rows(x)
        t = MX4Tensor._of(torch.empty(p * n * 68, dtype=torch.uint8, device=dev), n, k)
        _lib.run("lira_mx4_quantize", x.data_ptr(), DTYPES[x.dtype], n, k, ld, *t.addresses(), n,
                 raw_stream(dev.index))
    return t


def _out(out, shape, dtype, device, *inputs) -> tuple[torch.Tensor, int]:
    """Where the result goes, and its row stride; not over an input, which other workgroups still read."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device), max(1, shape[1])
    if not isinstance(out, torch.Tensor) or out.device != device or out.dtype != dtype or tuple(out.shape) != shape:
        raise ValueError(f"out must be a {shape} {dtype} tensor on {device}")
    if shape[1] > 1 and out.stride(1) != 1 or shape[0] > 1 and out.stride(0) < shape[1]:
        raise ValueError("out must have rows of consecutive elements that do not overlap")
    refuse_shared(out, "out", *(v for i in inputs for v in ((i.codes, i.scales) if isinstance(i, MX4Tensor) else (i,))))
    _no_grad(out)
    increment_version(out)  # (autograd may have saved it)
    return out, out.stride(0) if shape[0] > 1 else max(1, shape[1])


def mx4_dequantize(t: MX4Tensor, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
                   stream=None) -> torch.Tensor:
    """The rows of t as numbers (lira_mx4_dequantize)."""
    if not isinstance(t, MX4Tensor):
        raise ValueError("t must be an MX4Tensor")
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    dev, n = t.device, t.n
    with on(dev, stream):
        out, ld = _out(out, (n, t.k), dtype, dev, t)
        if stream is not None:
            keep_for(stream, t, out)
        _lib.run("lira_mx4_dequantize", *t.addresses(), t.plane_rows, n, t.k, out.data_ptr(), DTYPES[dtype], ld,
                 raw_stream(dev.index))
    return out


def _epilogue(w, bias, activation):
    if not isinstance(w, MX4Tensor):
        raise ValueError("the right operand must be an MX4Tensor (mx4_quantize packs one)")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, not {activation!r}")
    if bias is None:
        return None, ACTIVATIONS[activation]
    if not isinstance(bias, torch.Tensor) or bias.device != w.device or tuple(bias.shape) != (w.n,) \
            or not bias.is_floating_point():
        raise ValueError(f"bias must be a ({w.n},) float tensor on {w.device}")
    _no_grad(bias)
    return bias, ACTIVATIONS[activation]


def mx4_matmul(a: MX4Tensor, b: MX4Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
               alpha: float = 1.0, out_dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
               stream=None) -> torch.Tensor:
    """activation(alpha * a @ b.T + bias), (a rows, b rows) in out_dtype, sums in fp32
    (lira_mx4_matmul).  activation: None, "relu" or "sigmoid"; bias (b rows,)."""
    if not isinstance(a, MX4Tensor):
        raise ValueError("the left operand must be an MX4Tensor (mx4_linear packs plain rows on the way)")
    bias, act = _epilogue(b, bias, activation)
    if a.k != b.k or a.device != b.device:
        raise ValueError(f"a has {a.k} columns on {a.device}, b has {b.k} on {b.device}")
    if out_dtype not in DTYPES:
        raise ValueError(f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
    m, n = a.n, b.n
    dev = a.device
    with on(dev, stream):
        if stream is not None:
            keep_for(stream, a, b, bias)
        bias = None if bias is None else bias.to(torch.float32).contiguous()
        out, ldo = _out(out, (m, n), out_dtype, dev, a, b, bias)
        if stream is not None:
            keep_for(stream, out)
        _lib.run("lira_mx4_matmul", *a.addresses(), a.plane_rows, m, *b.addresses(), b.plane_rows, n, a.k, alpha, _lib.ptr(bias), act, out.data_ptr(),
                 DTYPES[out_dtype], ldo, raw_stream(dev.index))
    return out


@functools.lru_cache(maxsize=1024)
def _linear_workspace(m: int, n: int, k: int) -> int:
    need = ctypes.c_size_t()
    _lib.run("lira_mx4_linear_workspace_size", m, n, k, ctypes.byref(need))
    return need.value


def mx4_linear(x: torch.Tensor, w: MX4Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
               alpha: float = 1.0, out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
               stream=None) -> torch.Tensor:
    """activation(alpha * Q(x) @ w.T + bias): the rows of x (m, k) are packed on the way, exactly as
    mx4_quantize packs them (lira_mx4_linear).  The result has x's type unless out_dtype says otherwise."""
    bias, act = _epilogue(w, bias, activation)
    x = check_rows(x, "x", w.device)
    _no_grad(x)
    if x.shape[1] != w.k:
        raise ValueError(f"x has {x.shape[1]} columns, w has {w.k}")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in DTYPES:
        raise ValueError(f"out_dtype must be float32, bfloat16 or float16, not {out_dtype}")
    m, n, k, dev = x.shape[0], w.n, w.k, x.device
    need = _linear_workspace(m, n, k)
    with on(dev, stream):
        if stream is not None:
            keep_for(stream, x, w, bias)
        x, ld = _rows(x)
        bias = None if bias is None else bias.to(torch.float32).contiguous()
        out, ldo = _out(out, (m, n), out_dtype, dev, x, w, bias)
        if stream is not None:
            keep_for(stream, out)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.run("lira_mx4_linear", x.data_ptr(), DTYPES[x.dtype], m, k, ld, *w.addresses(), w.plane_rows, n, alpha, _lib.ptr(bias), act, out.data_ptr(), DTYPES[out_dtype], ldo, _lib.ptr(ws), need,
                 raw_stream(dev.index))
    return out
