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

import torch

from . import _lib
from .mx4 import DTYPES, check_rows, on, _rows


def check_device(logits) -> None:
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError("logits must be a tensor on the GPU")


def _entries(logits, top_ids, top_logits, temperature, teacher_lse):
    """The checked arguments, as (rows, vocab) logits and (rows, top) entries."""
    check_device(logits)
    if logits.dim() < 1:
        raise ValueError("logits must have at least one dimension")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    z = check_rows(logits.reshape(-1, vocab) if vocab else logits.reshape(lead.numel(), 0), "logits")
    if vocab < 1:
        raise ValueError("logits must have at least one output")
    for t, name in ((top_ids, "top_ids"), (top_logits, "top_logits")):
        if not isinstance(t, torch.Tensor) or t.device != z.device:
            raise ValueError(f"{name} must be a tensor on {z.device}")
        if t.dim() != logits.dim() or t.shape[:-1] != lead:
            raise ValueError(f"{name} must have the logits' leading dimensions {tuple(lead)}, not {tuple(t.shape[:-1])}")
    if top_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"top_ids must be int32 or int64, not {top_ids.dtype}")
    if top_logits.dtype not in DTYPES:
        raise ValueError(f"top_logits must be float32, bfloat16 or float16, not {top_logits.dtype}")
    top = top_ids.shape[-1]
    if top < 1 or top_logits.shape != top_ids.shape:
        raise ValueError(f"top_ids {tuple(top_ids.shape)} and top_logits {tuple(top_logits.shape)} must have the same "
                         "shape, at least one entry a row")
    if not 0.0 < float(temperature) < float("inf"):
        raise ValueError("temperature must be positive and finite")
    if teacher_lse is not None and (not isinstance(teacher_lse, torch.Tensor) or teacher_lse.device != z.device
                                    or teacher_lse.shape != lead or not teacher_lse.is_floating_point()):
        raise ValueError(f"teacher_lse must be a {tuple(lead)} float tensor on {z.device}")
    return z, lead, top


def _plain(top_ids, top_logits, teacher_lse, top):
    """The entries as the kernels read them (constants: the teacher gets no gradient)."""
    ids = top_ids.reshape(-1, top).contiguous()
    tv = top_logits.detach().reshape(-1, top).to(torch.float32).contiguous()
    lse = None if teacher_lse is None else teacher_lse.detach().reshape(-1).to(torch.float32).contiguous()
    return ids, tv, lse


def _head(z, ld, ids, tv, lse, t):
    rows, vocab = z.shape
    return (z.data_ptr(), DTYPES[z.dtype], rows, vocab, ld, ids.data_ptr(), 64 if ids.dtype == torch.int64 else 32,
            tv.data_ptr(), ids.shape[1], t, _lib.ptr(lse))


def _workspace(z, ids):
    need = ctypes.c_size_t()
    _lib.call("lira_distill_workspace_size", *z.shape, ids.shape[1], DTYPES[z.dtype], ctypes.byref(need))
    return torch.empty(need.value, dtype=torch.uint8, device=z.device) if need.value else None


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, ids, tv, lse, t, reduction):
        z, ld = _rows(z)
        rows = z.shape[0]
        loss = torch.empty(rows, dtype=torch.float32, device=z.device)
        stats = torch.empty((rows, 4), dtype=torch.float32, device=z.device)
        ws = _workspace(z, ids)
        _lib.call("lira_distill_topk", *_head(z, ld, ids, tv, lse, t), loss.data_ptr(), stats.data_ptr(), None, 0, None,
                  0, _lib.ptr(ws), 0 if ws is None else ws.numel(), _lib.stream_ptr())
        ctx.save_for_backward(z, ids, tv, lse, stats)
        ctx.t, ctx.factor = t, None
        if reduction == "none":
            return loss
        out = torch.empty(2, dtype=torch.float32, device=z.device)
        _lib.call("lira_distill_reduce", loss.data_ptr(), stats.data_ptr(), rows, reduction == "mean", out.data_ptr(),
                  _lib.stream_ptr())
        ctx.factor = out[1]
        return out[0].clone()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        z, ids, tv, lse, stats = ctx.saved_tensors
        rows, vocab = z.shape
        with on(z.device):
            g = (g if ctx.factor is None else g * ctx.factor).to(torch.float32)
            whole = g.dim() == 0 or (rows > 1 and g.stride(0) == 0)  # one factor for all rows
            g = g if whole else g.contiguous()
            z, ld = _rows(z)
            dz = torch.empty((rows, vocab), dtype=z.dtype, device=z.device)
            _lib.call("lira_distill_topk_backward", *_head(z, ld, ids, tv, lse, ctx.t), stats.data_ptr(), g.data_ptr(),
                      0 if whole else 1, dz.data_ptr(), vocab, _lib.stream_ptr())
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
    z, lead, top = _entries(logits, top_ids, top_logits, temperature, teacher_lse)
    with on(z.device):
        loss = _Loss.apply(z, *_plain(top_ids, top_logits, teacher_lse, top), float(temperature), reduction)
    return loss.view(lead) if reduction == "none" else loss


@torch.no_grad()
def distill_topk_loss_and_grad(logits: torch.Tensor, top_ids: torch.Tensor, top_logits: torch.Tensor,
                               temperature: float = 1.0, teacher_lse: torch.Tensor | None = None,
                               row_weight: torch.Tensor | None = None, grad_out: torch.Tensor | None = None,
                               stream=None):
    """(loss (...), grad (..., vocab)): every row's loss as distill_topk_loss(reduction="none")
    gives it, and the gradient of sum(row_weight * loss) with respect to the logits, for
    ``logits.backward(grad)``.  row_weight (...): None = 1.  grad_out: where the gradient goes, a
    contiguous tensor like the logits; the logits themselves are allowed."""
    check_device(logits)
    with on(logits.device, stream):
        z, lead, top = _entries(logits, top_ids, top_logits, temperature, teacher_lse)
        if row_weight is not None and (not isinstance(row_weight, torch.Tensor) or row_weight.device != z.device
                                       or row_weight.shape != lead or not row_weight.is_floating_point()):
            raise ValueError(f"row_weight must be a {tuple(lead)} float tensor on {z.device}")
        if grad_out is not None and (not isinstance(grad_out, torch.Tensor) or grad_out.shape != logits.shape
                                     or grad_out.dtype != logits.dtype or grad_out.device != z.device
                                     or not grad_out.is_contiguous()):
            raise ValueError("grad_out must be a contiguous tensor of the logits' shape, type and device")
        z, ld = _rows(z.detach())
        rows, vocab = z.shape
        ids, tv, lse = _plain(top_ids, top_logits, teacher_lse, top)
        w = None if row_weight is None else row_weight.detach().reshape(-1).to(torch.float32).contiguous()
        loss = torch.empty(rows, dtype=torch.float32, device=z.device)
        dz = torch.empty((rows, vocab), dtype=z.dtype, device=z.device) if grad_out is None else grad_out
        ws = _workspace(z, ids)
        _lib.call("lira_distill_topk", *_head(z, ld, ids, tv, lse, float(temperature)), loss.data_ptr(), None,
                  _lib.ptr(w), 1, dz.data_ptr(), vocab, _lib.ptr(ws), 0 if ws is None else ws.numel(),
                  _lib.stream_ptr())
    return loss.view(lead), dz.view(logits.shape)
