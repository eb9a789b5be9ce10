"""Distillation from a teacher's top outputs: loss and gradient in one or two passes over the student's logits.

The probing model learns which partitions a query needs (model_probing.py:41-54); its teacher
here is whatever ranks them better -- the exact centroid ranking, kNN counts, a larger model --
of which only the top entries of each row are kept.  include/lira_hip.h has the formulas.

* ``distill_topk_loss``            differentiable: the forward pass reads the logits once, the
                                   backward pass reads them again and writes their gradient
* ``distill_topk_loss_and_grad``   both in one call, for a training step whose row weights are
                                   known beforehand: the logits are read from memory once

A captured graph should hold ``distill_topk_loss_and_grad``, or a whole forward and backward pass
whose leaves no eager autograd graph still uses.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .mx4 import DTYPES, check_rows, keep_for, on, raw_stream, refuse_shared, _rows


def check_device(logits) -> None:
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError("logits must be a tensor on the GPU")


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    return t if t.dim() == 2 else t.reshape(-1, t.shape[-1])


def _fp32(t: torch.Tensor) -> torch.Tensor:
    """A constant of the kernels: detached, float32, contiguous."""
    if t.requires_grad:
        t = t.detach()
    return (t if t.dtype == torch.float32 else t.to(torch.float32)).contiguous()


def _row_values(t, name: str, lead, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.device != device or t.shape != lead or not t.is_floating_point():
        raise ValueError(f"{name} must be a {tuple(lead)} float tensor on {device}")
    return _fp32(t if len(lead) == 1 else t.reshape(-1))


def _entries(logits, top_ids, top_logits, temperature, teacher_lse):
    """(logits (rows, vocab), the logits' leading dimensions, ids, teacher's logits, its logsumexp), checked and as
    the kernels read them (the teacher is constant)."""
    shape, dev = logits.shape, logits.device
    if not shape or not shape[-1]:
        raise ValueError("logits must have at least one dimension and one output")
    lead = shape[:-1]
    z = check_rows(_rows_of(logits), "logits")
    for t, name in ((top_ids, "top_ids"), (top_logits, "top_logits")):
        if not isinstance(t, torch.Tensor) or t.device != dev:
            raise ValueError(f"{name} must be a tensor on {dev}")
        if t.dim() != len(shape) or t.shape[:-1] != lead:
            raise ValueError(f"{name} must have the logits' leading dimensions {tuple(lead)}, not {tuple(t.shape[:-1])}")
    if top_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"top_ids must be int32 or int64, not {top_ids.dtype}")
    if top_logits.dtype not in DTYPES:
        raise ValueError(f"top_logits must be float32, bfloat16 or float16, not {top_logits.dtype}")
    if top_logits.shape != top_ids.shape or not top_ids.shape[-1]:
        raise ValueError(f"top_ids {tuple(top_ids.shape)} and top_logits {tuple(top_logits.shape)} must have the same "
                         "shape, at least one entry a row")
    if not 0.0 < temperature < float("inf"):
        raise ValueError("temperature must be positive and finite")
    return (z, lead, _rows_of(top_ids).contiguous(), _fp32(_rows_of(top_logits)),
            _row_values(teacher_lse, "teacher_lse", lead, dev))


def _head(z, ids, tv, lse, t):
    """The arguments that the forward and the backward entry begin with (z: rows of consecutive elements)."""
    rows, vocab = z.shape
    return (z.data_ptr(), DTYPES[z.dtype], rows, vocab, z.stride(0) if rows > 1 else vocab, ids.data_ptr(),
            64 if ids.dtype == torch.int64 else 32, tv.data_ptr(), ids.shape[1], t, None if lse is None else lse.data_ptr())


@functools.lru_cache(maxsize=1024)
def _workspace_size(rows: int, vocab: int, top: int, dtype: int) -> int:
    need = ctypes.c_size_t()
    _lib.run("lira_distill_workspace_size", rows, vocab, top, dtype, ctypes.byref(need))
    return need.value


def _forward(head, dev, stats, row_weight, dz):
    rows, vocab = head[2], head[3]
    loss = torch.empty(rows, dtype=torch.float32, device=dev)
    need = _workspace_size(rows, vocab, head[8], head[1])
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _lib.run("lira_distill_topk", *head, loss.data_ptr(), _lib.ptr(stats), _lib.ptr(row_weight), 1, _lib.ptr(dz), vocab,
             _lib.ptr(ws), need, raw_stream(dev.index))
    return loss


_KINDS = {**DTYPES, torch.int32: 32, torch.int64: 64}


def _same(t: torch.Tensor, shape: tuple, kind: int, device: torch.device) -> torch.Tensor:
    """A tensor that the backward pass reads by address: as it was saved, but for its layout."""
    if t.shape != shape or _KINDS.get(t.dtype) != kind or t.device != device:
        raise RuntimeError(f"distill_topk_loss: a saved tensor came back as {tuple(t.shape)} {t.dtype} on {t.device}")
    return t.contiguous()


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, ids, tv, lse, t, reduction):
        dev = z.device
        z = _rows(z)[0]
        head = _head(z, ids, tv, lse, t)
        stats = torch.empty((head[2], 4), dtype=torch.float32, device=dev)
        loss = _forward(head, dev, stats, None, None)
        ctx.save_for_backward(z, ids, tv, lse, stats)
        ctx.sizes, ctx.factor = (head[1], head[2], head[3], head[4], head[6], head[8], t), None
        if reduction == "none":
            return loss
        out = torch.empty(2, dtype=torch.float32, device=dev)
        _lib.run("lira_distill_reduce", loss.data_ptr(), stats.data_ptr(), head[2], reduction == "mean", out.data_ptr(),
                 raw_stream(dev.index))
        if reduction == "mean":
            ctx.factor = out[1]  # (of a sum it is 1)
        return out[0].clone()

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():
            raise RuntimeError("distill_topk_loss has no second derivative (create_graph=True)")
        # (not always the tensors of the forward pass: hooks may have moved them, or laid them out otherwise.  The engine
        # has made their device and the forward pass's stream the current ones.)
        z, ids, tv, lse, stats = ctx.saved_tensors
        dtype, rows, vocab, ld, bits, top, t = ctx.sizes
        dev = z.device
        if z.shape != (rows, vocab) or DTYPES.get(z.dtype) != dtype or dev != g.device:
            raise RuntimeError(f"distill_topk_loss: the logits came back as {tuple(z.shape)} {z.dtype} on {z.device}")
        ids = _same(ids, (rows, top), bits, dev)
        tv, stats = _same(tv, (rows, top), _lib.LIRA_DTYPE_F32, dev), _same(stats, (rows, 4), _lib.LIRA_DTYPE_F32, dev)
        if lse is not None:
            lse = _same(lse, (rows,), _lib.LIRA_DTYPE_F32, dev)
        if z.stride() != (ld, 1):
            z, ld = _rows(z)
        if ctx.factor is not None:
            g = g * ctx.factor
        whole = g.dim() == 0 or (rows > 1 and g.stride(0) == 0)  # one factor for all rows
        if not whole:
            g = g.contiguous()
        dz = torch.empty((rows, vocab), dtype=z.dtype, device=dev)
        _lib.run("lira_distill_topk_backward", z.data_ptr(), dtype, rows, vocab, ld, ids.data_ptr(), bits, tv.data_ptr(), top, t,
                 None if lse is None else lse.data_ptr(), stats.data_ptr(), g.data_ptr(), 0 if whole else 1, dz.data_ptr(),
                 vocab, raw_stream(dev.index))
        return dz, None, None, None, None, None


def distill_topk_loss(logits: torch.Tensor, top_ids: torch.Tensor, top_logits: torch.Tensor,
                      temperature: float = 1.0, teacher_lse: torch.Tensor | None = None,
                      reduction: str = "mean") -> torch.Tensor:
    """T^2 KL(teacher's top entries || student) of every row of logits (..., vocab).

    top_ids (..., top) int32 / int64, -1 = unused; top_logits (..., top): the teacher's logits
    there.  teacher_lse (...): the teacher's logsumexp of all its logits / temperature -- its
    probabilities are then taken as they are; without it they are normalised over the entries.
    reduction: "none" (one loss a row), "sum", or "mean" over the rows with an entry that counts
    (0 where none has).  The teacher is constant: no gradient reaches it.  A masked output is a
    logit of -inf.  Losses are float32, the gradient has the logits' type.
    """
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', not {reduction!r}")
    check_device(logits)
    with on(logits.device):
        z, lead, ids, tv, lse = _entries(logits, top_ids, top_logits, temperature, teacher_lse)
        loss = _Loss.apply(z, ids, tv, lse, temperature, reduction)
    return loss.view(lead) if reduction == "none" and len(lead) != 1 else loss


def distill_topk_loss_and_grad(logits: torch.Tensor, top_ids: torch.Tensor, top_logits: torch.Tensor,
                               temperature: float = 1.0, teacher_lse: torch.Tensor | None = None,
                               row_weight: torch.Tensor | None = None, grad_out: torch.Tensor | None = None,
                               stream=None):
    """(loss (...), grad (..., vocab)): every row's loss as distill_topk_loss(reduction="none")
    gives it, and the gradient of sum(row_weight * loss) with respect to the logits, for
    ``logits.backward(grad)``.  row_weight (...): None = 1.  grad_out: where the gradient goes, a
    contiguous tensor like the logits, which must not share memory with an input; the logits
    themselves are allowed (an in-place change to autograd: the backward pass of an operation that
    saved them, as tanh does, is then refused by torch)."""
    check_device(logits)
    dev = logits.device
    with on(dev, stream):
        z, lead, ids, tv, lse = _entries(logits, top_ids, top_logits, temperature, teacher_lse)
        w = _row_values(row_weight, "row_weight", lead, dev)
        if stream is not None:
            keep_for(stream, logits, top_ids, top_logits, teacher_lse, row_weight)
        z = _rows(z)[0]  # (perhaps a copy: held until the launch, the head has its address alone)
        if grad_out is None:
            dz = torch.empty(logits.shape, dtype=z.dtype, device=dev)
        elif not isinstance(grad_out, torch.Tensor) or grad_out.shape != logits.shape or grad_out.dtype != z.dtype \
                or grad_out.device != dev or not grad_out.is_contiguous():
            raise ValueError("grad_out must be a contiguous tensor of the logits' shape, type and device")
        else:
            dz = grad_out
            same = dz.data_ptr() == z.data_ptr() and z.is_contiguous()  # (the logits' own places)
            refuse_shared(dz, "grad_out (but for the logits themselves)", None if same else z, ids, tv, lse, w)
            if stream is not None:
                keep_for(stream, dz)
            increment_version(dz)  # (autograd may have saved it: the logits' own operation, where it is the logits)
        loss = _forward(_head(z, ids, tv, lse, temperature), dev, None, w, dz)
    return loss if len(lead) == 1 else loss.view(lead), dz
