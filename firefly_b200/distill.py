"""Distillation from a teacher's top logits: the loss that trains a quantised student.

The reference ships no loss; this stands beside the decoder's cross-entropy.  The teacher is given
by its k largest logits per position, which is what a teacher run can afford to store.  Forward with
a reduction reads the student's logits once and writes their gradient in the same pass, for an
upstream gradient of 1; backward hands it out, or, when the upstream gradient on the device is
another, recomputes it (no host synchronisation either way).  In CUDA graphs that holds where one graph has both; a
backward captured without its forward, or run on a captured one, computes the gradient in a buffer of its own.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _capi


class DistillationLossFn(torch.autograd.Function):
    """Rows of ``distillation_loss``: operands 2-D with unit column stride."""

    @staticmethod
    def forward(ctx, logits, ids, teacher_logits, labels, teacher_lse, temperature, alpha, ignore_index, reduction, grad):
        grad = grad and ctx.needs_input_grad[0]
        ctx.args = (temperature, alpha, ignore_index)
        ctx.reduction = reduction
        rows = _capi.distill_rows(logits, ids, teacher_logits, labels, teacher_lse, *ctx.args)
        row, loss, g, held, counts = _capi.distill_loss(rows, logits, reduction, grad)
        if grad:
            ctx.save_for_backward(logits, ids, teacher_logits, labels, teacher_lse, counts)
            ctx.ready = None if g is None else (g, held, _capi.capture_id(logits.device))
        return row if reduction == "none" else loss

    @staticmethod
    @once_differentiable
    def backward(ctx, up):
        logits, ids, teacher_logits, labels, teacher_lse, counts = ctx.saved_tensors
        rows = _capi.distill_rows(logits, ids, teacher_logits, labels, teacher_lse, *ctx.args)
        up = up.to(torch.float32).contiguous()
        g, held, made_in = ctx.ready or (None, None, 0)
        ctx.ready = None  # the buffer is handed out: a second backward makes its own
        capture = _capi.capture_id(logits.device)
        if made_in != capture:
            # a forward and a backward that are not replayed together: the one's buffer would be rewritten under, or
            # handed out a second time to, the other's caller
            g = held = None
        g = _capi.distill_grad(rows, logits, ctx.reduction, up, counts, g, held, replayed=capture != 0)
        return (g,) + (None,) * 9


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """[..., width] as a matrix with unit column stride."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    return t if t.stride(1) == 1 and t.stride(0) >= width else t.contiguous()


def distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor,
                      labels: torch.Tensor | None = None, *, teacher_lse: torch.Tensor | None = None,
                      temperature: float = 1.0, alpha: float = 1.0, ignore_index: int = -100,
                      reduction: str = "mean") -> torch.Tensor:
    """``alpha · T² · KL(p ‖ q) + (1 - alpha) · cross-entropy``, in fp32.

    logits [..., V] (bf16, fp16 or fp32; the gradient has their type): the student's; q = softmax(logits / T).
    teacher_ids, teacher_logits [..., k]: the teacher's top tokens and logits; an entry with a negative id or
    a logit of -inf is absent, a token given twice counts with both entries.  p = softmax(teacher_logits / T)
    over the entries; with ``teacher_lse`` [...], the teacher's ``logsumexp(logits / T)`` over its whole
    vocabulary, p are its true probabilities and the rest of the mass is one bucket for all other tokens (none if the
    entries cover the vocabulary; infinitely far from a student that has every other token at -inf).
    labels [...]: hard labels; a row with ``ignore_index`` counts nothing.  Without labels only the first
    term is left, and a row without entries counts nothing.
    reduction: "mean" over the rows that count (0 if none does), "sum", or "none" (a loss per row).

    A token or label at or beyond V is treated as absent or ignored and reported by ``device_status()``.
    """
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1 or logits.dtype not in (
            torch.float32, torch.bfloat16, torch.float16):
        raise ValueError("logits must be a float32, bfloat16 or float16 tensor [..., V]")
    lead, V = tuple(logits.shape[:-1]), logits.shape[-1]
    k = teacher_ids.shape[-1] if teacher_ids.dim() else 0
    if V < 1 or k < 1 or tuple(teacher_ids.shape) != lead + (k,) or tuple(teacher_logits.shape) != lead + (k,):
        raise ValueError(f"distillation shapes: logits {tuple(logits.shape)}, teacher_ids {tuple(teacher_ids.shape)}, "
                         f"teacher_logits {tuple(teacher_logits.shape)} (the same leading dims, k >= 1 entries)")
    if teacher_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"teacher_ids must be int32 or int64, got {teacher_ids.dtype}")
    if teacher_logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"unsupported teacher_logits dtype {teacher_logits.dtype}")
    if labels is not None and (tuple(labels.shape) != lead or labels.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"labels must be int32 or int64 of shape {lead}, got {labels.dtype} {tuple(labels.shape)}")
    if teacher_lse is not None and tuple(teacher_lse.shape) != lead:
        raise ValueError(f"teacher_lse must have shape {lead}, got {tuple(teacher_lse.shape)}")
    if reduction not in _capi.FF_REDUCE:
        raise ValueError(f"reduction must be one of {sorted(_capi.FF_REDUCE)}, got {reduction!r}")
    temperature, alpha = float(temperature), float(alpha)
    if not 0.0 < temperature < float("inf") or not 0.0 <= alpha <= 1.0:
        raise ValueError(f"temperature must be positive and alpha in [0, 1], got {temperature} and {alpha}")
    if teacher_logits.requires_grad or (teacher_lse is not None and teacher_lse.requires_grad):
        raise ValueError("the teacher's logits get no gradient: detach them")
    _capi._require_cuda(logits, teacher_ids, teacher_logits, labels, teacher_lse)
    lab = None if labels is None else labels.reshape(-1).contiguous()
    lse = None if teacher_lse is None else teacher_lse.reshape(-1).to(torch.float32).contiguous()
    args = (_rows(logits, V), _rows(teacher_ids, k), _rows(teacher_logits, k), lab, lse, temperature, alpha, int(ignore_index))
    grad = torch.is_grad_enabled() and logits.requires_grad
    if grad or _capi.has_tangent(logits, teacher_logits, teacher_lse):  # (a tangent is refused there)
        out = DistillationLossFn.apply(*args, reduction, grad)
    else:
        row, loss, *_ = _capi.distill_loss(_capi.distill_rows(*args), args[0], reduction, False)
        out = row if reduction == "none" else loss
    return out.view(lead) if reduction == "none" and len(lead) != 1 else out


__all__ = ["DistillationLossFn", "distillation_loss"]
