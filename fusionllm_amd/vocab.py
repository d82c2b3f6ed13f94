"""The two ends of a model on the kernels: ``embedding`` / ``Embedding`` in front of
the blocks, and the losses behind them that take the hidden states and the
vocabulary's weight, ``linear_cross_entropy`` and ``linear_distillation``.

``embedding(ids, weight, scale)`` is ``scale * weight[ids]``.  Its backward adds each
id's rows in fp32 in a fixed order (above 64 tokens they are sorted by id first): the same
bits every run, no atomics.

The losses are those of the logits ``s = logit_scale * hidden @ weight.T``,
which are not kept (a distillation with long lists forms them a piece of 256 MB
at a time).  A loss of one value (mean, sum) that needs gradients forms them in
its forward, a piece of the rows at a time (up to 2 GiB), and its backward scales
them by the loss's gradient (rounded to their dtype a second time, unless that is
a power of two).  A loss per row (none), and one of up to 64 rows or of a
vocabulary too large for such pieces, reduces the logits tile by tile in the
forward and forms them again in the backward.  Rows without a target
(``ignore_index``) are left out of every product.

    linear_cross_entropy   -log softmax(s)[target]
    linear_distillation    temperature^2 * sum_k q_k (log q_k - log p_k), with q the
                           softmax of a teacher's listed logits over the temperature
                           and p = softmax(s / temperature) over the whole vocabulary

hidden and weight are both bf16 (bf16 products, fp32 sums) or both fp32 (fp32 precision throughout);
under bf16 autocast either may be either, and both are taken as bf16.  Losses
are fp32, gradients have their operand's dtype.  fp32 operands that hold infinities may give NaN
where sums of infinities would be infinite.  ROCm tensors only.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _kernels as K
from .norm import _on_device, _rows, refuse_tangents

_FLOATS = (torch.bfloat16, torch.float32)
_INTS = (torch.int32, torch.int64)


def _check_weight(what, weight):
    if not weight.is_cuda:
        raise RuntimeError(f"{what} runs on a ROCm device only (got a {weight.device.type} weight)")
    if weight.dim() != 2 or weight.shape[0] == 0:
        raise ValueError(f"{what}: weight must be [vocab, dim] (got {tuple(weight.shape)})")
    if not 1 <= weight.shape[1] <= K.VOCAB_MAX_DIM:
        raise NotImplementedError(f"{what} takes 1 to {K.VOCAB_MAX_DIM} columns (got {weight.shape[1]})")
    if weight.dtype not in _FLOATS:
        raise NotImplementedError(f"{what} supports bf16 and fp32 weights (got {weight.dtype})")


def _check_index(what, name, t, device):
    if t.dtype not in _INTS:
        raise ValueError(f"{what}: {name} must be int32 or int64 (got {t.dtype})")
    if t.device != device:
        raise RuntimeError(f"{what}: {name} must be on the weight's device")


# ---- embedding ------------------------------------------------------------------


class _EmbeddingFunction(torch.autograd.Function):
    """The embedding through the Python wrappers (the native form, csrc/block_host.cpp, runs the same entry points)."""

    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        with _on_device(weight):
            y = K.embedding_fwd(ids, _rows(weight), scale)
        ctx.save_for_backward(ids)
        ctx.args = (weight.shape[0], scale, padding_idx, weight.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        with _on_device(dy):
            return None, K.embedding_bwd(ids, _rows(dy), *ctx.args), None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[ids]`` in weight's dtype, for ids of any shape.  The row of padding_idx
    receives no gradient; an id outside the vocabulary gives a row of NaN and adds to no gradient."""
    what = "fusionllm_amd.embedding"
    _check_weight(what, weight)
    _check_index(what, "ids", ids, weight.device)
    V, dim = weight.shape
    pad = -1
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"{what}: padding_idx must be within the vocabulary (got {padding_idx} of {V})")
        pad = padding_idx % V
    scale = float(scale)
    flat = ids if ids.dim() == 1 and ids.is_contiguous() else ids.reshape(-1).contiguous()
    if torch.compiler.is_compiling():
        y = torch.ops.fusionllm.embedding_fwd(flat, weight, scale, pad)
    else:
        refuse_tangents(what, weight)
        grad = torch.is_grad_enabled() and weight.requires_grad
        host = K.block_host()
        if host is not None:
            y = host.embedding(flat, weight, scale, pad, grad)
        elif grad:
            y = _EmbeddingFunction.apply(flat, weight, scale, pad)
        else:
            with _on_device(weight):
                y = K.embedding_fwd(flat, _rows(weight), scale)
    return y if ids.dim() == 1 else y.view(*ids.shape, dim)


class Embedding(nn.Embedding):
    """``torch.nn.Embedding`` on the kernels: the same constructor (less max_norm, scale_grad_by_freq and
    sparse, which are refused), parameters and state dict, and a factor ``scale`` for its rows."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, max_norm=None, norm_type=2.0,
                 scale_grad_by_freq=False, sparse=False, *args, scale: float = 1.0, **kwargs):
        if max_norm is not None or scale_grad_by_freq or sparse:
            raise NotImplementedError("fusionllm_amd.Embedding has no max_norm, scale_grad_by_freq or sparse gradients")
        super().__init__(num_embeddings, embedding_dim, padding_idx, None, norm_type, False, False, *args, **kwargs)
        self.scale = float(scale)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return embedding(input, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return super().extra_repr() + (f", scale={self.scale}" if self.scale != 1.0 else "")


# ---- losses -----------------------------------------------------------------------


class _VocabLossFunction(torch.autograd.Function):
    """A loss over the vocabulary (teacher None: cross entropy) through the Python wrappers (the native form,
    csrc/block_host.cpp, runs the same entry points)."""

    @staticmethod
    def forward(ctx, hidden, weight, index, teacher, ignore_index, logit_scale, temperature, planes, reduction):
        w = _rows(weight)
        with _on_device(weight):
            loss, state = K.vocab_loss_fwd(_rows(hidden), w, index, teacher, ignore_index, logit_scale, temperature,
                                           planes, reduction)
        ctx.save_for_backward(w, state)
        ctx.args = (hidden.shape[0], index.shape[1], teacher is not None, logit_scale, temperature, planes, reduction)
        ctx.dtypes = (hidden.dtype, weight.dtype)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss):
        w, state = ctx.saved_tensors
        need_h, need_w = ctx.needs_input_grad[:2]
        with _on_device(w):
            dh, dw = K.vocab_loss_bwd(d_loss.contiguous(), w, state, *ctx.args, ctx.dtypes[0] if need_h else None,
                                      ctx.dtypes[1] if need_w else None)
        return dh, dw, None, None, None, None, None, None, None


class _VocabLossGradFunction(torch.autograd.Function):
    """A loss of one value whose gradients are formed in the forward, through the Python wrappers."""

    @staticmethod
    def forward(ctx, hidden, weight, index, teacher, ignore_index, logit_scale, temperature, planes, reduction):
        with _on_device(weight):
            loss, dh, dw = K.vocab_loss_fwd_grad(_rows(hidden), _rows(weight), index, teacher, ignore_index, logit_scale,
                                                 temperature, planes, reduction, *ctx.needs_input_grad[:2])
        ctx.save_for_backward(dh, dw)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss):
        grads = [g if need else None for g, need in zip(ctx.saved_tensors, ctx.needs_input_grad)]
        with _on_device(d_loss):
            grads = K.scale(d_loss.contiguous(), grads)
        return *grads, None, None, None, None, None, None, None


def _gradients_at_once(flat, weight, planes, reduction):
    """Whether the forward forms the gradients.  A contiguous copy of a weight that is none starts at an aligned
    address."""
    return reduction != "none" and K.vocab_loss_takes_gradients(
        flat.shape[0], flat.shape[1], weight.shape[0], planes, K.vocab_loss_packs(_rows(weight), planes))


def _check_loss(what, hidden, weight, reduction, logit_scale):
    """Checks the operands; the planes of the products (1: bf16, 3: fp32)."""
    _check_weight(what, weight)
    if hidden.device != weight.device:
        raise RuntimeError(f"{what}: hidden must be on the weight's device")
    if hidden.dim() == 0 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: hidden must have {weight.shape[1]} columns (got {tuple(hidden.shape)})")
    if hidden.dtype not in _FLOATS:
        raise NotImplementedError(f"{what} supports bf16 and fp32 hidden states (got {hidden.dtype})")
    if reduction not in K.REDUCTIONS:
        raise ValueError(f"{what}: reduction must be 'none', 'mean' or 'sum' (got {reduction!r})")
    if not math.isfinite(logit_scale):
        raise ValueError(f"{what}: logit_scale must be finite (got {logit_scale})")
    if torch.is_autocast_enabled("cuda"):
        if torch.get_autocast_dtype("cuda") != torch.bfloat16:
            raise NotImplementedError(f"{what} supports bf16 autocast only")
        return 1
    if hidden.dtype != weight.dtype:
        raise RuntimeError(f"{what}: hidden and weight must have one dtype outside autocast "
                           f"(got {hidden.dtype} and {weight.dtype})")
    return 1 if weight.dtype == torch.bfloat16 else 3


def _vocab_loss(what, hidden, weight, index, teacher, ignore_index, logit_scale, temperature, planes, reduction):
    """index and teacher: hidden's leading shape and the list."""
    logit_scale, temperature = float(logit_scale), float(temperature)
    if not (2.0 ** -63 <= temperature <= 2.0 ** 63 and
            abs(logit_scale) * max(temperature, 1.0 / temperature) < 2.0 ** 126):
        raise ValueError(f"{what}: logit_scale {logit_scale} and temperature {temperature} leave the range of fp32")
    shape = hidden.shape[:-1]
    flat = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
    index = index.reshape(-1, index.shape[-1]).contiguous()
    if teacher is not None:
        teacher = teacher.detach().reshape(index.shape).contiguous()
    args = (flat, weight, index, teacher, int(ignore_index), logit_scale, temperature, planes, reduction)
    if torch.compiler.is_compiling():
        # (the traced form sees no addresses: a weight as it lies in a module)
        packs = planes != 1 or weight.dtype != torch.bfloat16 or weight.shape[1] % 64 != 0 or not weight.is_contiguous()
        if (torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad) and reduction != "none" and
                K.vocab_loss_takes_gradients(flat.shape[0], flat.shape[1], weight.shape[0], planes, packs)):
            loss = torch.ops.fusionllm.vocab_loss_fwd_grad(*args, hidden.requires_grad, weight.requires_grad)[0]
        else:
            loss = torch.ops.fusionllm.vocab_loss_fwd(*args)[0]
    else:
        refuse_tangents(what, hidden, weight)
        grad = torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)
        host = K.block_host()
        if host is not None:
            loss = host.vocab_loss(*args[:-1], K.REDUCTIONS[reduction], grad)
        elif grad:
            with _on_device(weight):
                at_once = _gradients_at_once(flat, weight, planes, reduction)
            loss = (_VocabLossGradFunction if at_once else _VocabLossFunction).apply(*args)
        else:
            with _on_device(weight):
                loss = K.vocab_loss_fwd(_rows(flat), _rows(weight), *args[2:])[0]
    return loss.view(shape) if reduction == "none" and len(shape) != 1 else loss


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *,
                         ignore_index: int = -100, reduction: str = "mean", logit_scale: float = 1.0) -> torch.Tensor:
    """Cross entropy of the logits ``logit_scale * hidden @ weight.T`` and target, as
    ``torch.nn.functional.cross_entropy`` gives it (mean: over the targets that are not ignore_index;
    NaN if there are none), with an fp32 result and without the logits.  A target outside the
    vocabulary makes its loss NaN."""
    what = "fusionllm_amd.linear_cross_entropy"
    planes = _check_loss(what, hidden, weight, reduction, float(logit_scale))
    _check_index(what, "target", target, weight.device)
    if target.shape != hidden.shape[:-1]:
        raise ValueError(f"{what}: target must have shape {tuple(hidden.shape[:-1])} (got {tuple(target.shape)})")
    return _vocab_loss(what, hidden, weight, target.unsqueeze(-1), None, ignore_index, logit_scale, 1.0, planes,
                       reduction)


def linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_index: torch.Tensor,
                        teacher_logits: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100,
                        reduction: str = "mean", logit_scale: float = 1.0) -> torch.Tensor:
    """Divergence of the student's softmax over the vocabulary from a teacher's softmax over its listed
    logits (teacher_index, teacher_logits: hidden's leading shape and a list of up to 1024), at a temperature,
    times its square.  List entries whose index is ignore_index or whose logit is -infinity are none; a row
    without entries has no loss (mean: over the rows with entries).  An index listed twice counts twice; any
    other index outside the vocabulary makes the row's loss NaN.  The teacher receives no gradient."""
    what = "fusionllm_amd.linear_distillation"
    planes = _check_loss(what, hidden, weight, reduction, float(logit_scale))
    _check_index(what, "teacher_index", teacher_index, weight.device)
    if teacher_index.shape[:-1] != hidden.shape[:-1] or teacher_index.dim() != hidden.dim():
        raise ValueError(f"{what}: teacher_index must have shape {(*hidden.shape[:-1], 'top')} "
                         f"(got {tuple(teacher_index.shape)})")
    if not 1 <= teacher_index.shape[-1] <= K.VOCAB_MAX_TOP:
        raise NotImplementedError(f"{what} takes lists of 1 to {K.VOCAB_MAX_TOP} logits (got {teacher_index.shape[-1]})")
    if teacher_logits.shape != teacher_index.shape or teacher_logits.device != weight.device:
        raise ValueError(f"{what}: teacher_logits must have teacher_index's shape and device")
    if teacher_logits.dtype not in _FLOATS:
        raise NotImplementedError(f"{what} supports bf16 and fp32 teacher logits (got {teacher_logits.dtype})")
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{what} has no gradient for the teacher: pass teacher_logits.detach()")
    temperature = float(temperature)
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"{what}: temperature must be positive and finite (got {temperature})")
    return _vocab_loss(what, hidden, weight, teacher_index, teacher_logits, ignore_index, logit_scale, temperature,
                       planes, reduction)
