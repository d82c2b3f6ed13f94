"""DeepSeekMoE block (and the dense SwiGLU) as torch.library operators, for
torch.compile and graph capture.

``fusionllm::moe_fwd`` and ``fusionllm::moe_bwd`` run the same kernels as
the module's eager path (models/moe.py:44-87 forward, its autograd backward)
but are opaque to the tracer: ``register_fake`` gives their outputs' static
shapes (no data-dependent shape anywhere: rows = T*k routed + T shared), and
``register_autograd`` connects them.  ``DeepSeekMoE.forward`` routes through
them while ``torch.compiler.is_compiling()``, so ``torch.compile(model,
fullgraph=True)`` (training/trainer.py:39 compiles the whole model that way)
traces the block as two nodes.  The one difference from the eager module:
nothing here reads the expert counts on the host, so experts that received
no tokens get zero gradients instead of None.

moe_fwd outputs: y [T,d] (out_dtype), indices [T,k] int64, weights [T,k]
fp32, counts [E] int32, then the tensors the backward reads: idx32 [T,k],
topv [T,k] fp32, offsets [E+1], perm [T*k], pos_of_slot [T*k], x_perm
[T*k,d] bf16 (0 rows when the routed rows are read from x through perm),
ab [rows,2I] bf16, h [rows,I] bf16, o [rows,d] bf16.
moe_bwd returns [dx, d_gate_w, d_gate_b, *d_weights] in the inputs' dtypes.

``fusionllm::swiglu_fwd`` / ``swiglu_bwd`` do the same for the dense SwiGLU
(models/moe.py:11-21 used alone, the DenseFFN of models/fusionllm.py:17-27):
outputs y [T,d] bf16, ab [T,2I] bf16, h [T,I] bf16; gradients [dx, dw1,
dw3, dw2] in the inputs' dtypes.

``fusionllm::layer_norm_fwd`` / ``layer_norm_bwd`` do the same for ``layer_norm``:
outputs y [T,d] (out_dtype), mean [T] and rstd [T] fp32; gradients [dx, dw, db],
without those of a weight or bias that is not there.

``fusionllm::embedding_fwd`` / ``embedding_bwd`` and the losses over a vocabulary:
``vocab_loss_fwd`` (loss, the state for the backward) / ``vocab_loss_bwd`` (d_hidden, d_weight, those that are wanted),
and ``vocab_loss_fwd_grad`` (loss, and the gradients that are wanted, formed at once) with ``scale``.
"""
from __future__ import annotations

import types

import torch
from torch import Tensor

from . import _kernels as K
from . import norm as _norm
from .moe import _backward_pass, _bf16_operands, _dense_backward, _dense_offsets, _forward_pass, gathers_rows


def _meta(gate_w: Tensor, weights: list[Tensor], k: int, route_scale: float, has_shared: bool,
          out_dtype: torch.dtype):
    return (gate_w.shape[0], k, weights[0].shape[0], float(route_scale), bool(has_shared), out_dtype)


@torch.library.custom_op("fusionllm::moe_fwd", mutates_args=())
def moe_fwd(x: Tensor, gate_w: Tensor, gate_b: Tensor, weights: list[Tensor], k: int, route_scale: float,
            has_shared: bool, out_dtype: torch.dtype) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor,
                                                                Tensor, Tensor, Tensor, Tensor, Tensor, Tensor,
                                                                Tensor]:
    meta = _meta(gate_w, weights, k, route_scale, has_shared, out_dtype)
    fw = _forward_pass(meta, x, gate_w, gate_b, weights)
    xb, gwb, wb, idx, idx64, w, v, counts, offsets, perm, pos, x_perm, ab, h, o, y = fw
    if x_perm is None:  # routed rows read through perm: no gathered copy (0 rows)
        x_perm = xb.new_empty((0, xb.shape[1]))
    return y, idx64, w, counts, idx, v, offsets, perm, pos, x_perm, ab, h, o


@moe_fwd.register_fake
def _(x, gate_w, gate_b, weights, k, route_scale, has_shared, out_dtype):
    T, d = x.shape
    E, inter = gate_w.shape[0], weights[0].shape[0]
    rows = T * k + (T if has_shared else 0)
    i32, f32, bf = torch.int32, torch.float32, torch.bfloat16
    e = lambda *shape, dtype: x.new_empty(shape, dtype=dtype)
    xp_rows = 0 if gathers_rows(T, k, has_shared) else T * k
    return (e(T, d, dtype=out_dtype), e(T, k, dtype=torch.int64), e(T, k, dtype=f32), e(E, dtype=i32),
            e(T, k, dtype=i32), e(T, k, dtype=f32), e(E + 1, dtype=i32), e(T * k, dtype=i32),
            e(T * k, dtype=i32), e(xp_rows, d, dtype=bf), e(rows, 2 * inter, dtype=bf), e(rows, inter, dtype=bf),
            e(rows, d, dtype=bf))


@torch.library.custom_op("fusionllm::moe_bwd", mutates_args=())
def moe_bwd(dy: Tensor, x: Tensor, gate_w: Tensor, gate_b: Tensor, weights: list[Tensor], idx: Tensor,
            w: Tensor, v: Tensor, offsets: Tensor, perm: Tensor, pos: Tensor, x_perm: Tensor, ab: Tensor,
            h: Tensor, o: Tensor, k: int, route_scale: float, has_shared: bool) -> list[Tensor]:
    meta = _meta(gate_w, weights, k, route_scale, has_shared, dy.dtype)
    xb, gwb, *wb = _bf16_operands([x, gate_w, *weights])
    ctx = types.SimpleNamespace(meta=meta, param_dtypes=(gate_w.dtype, gate_b.dtype, [t.dtype for t in weights]))
    saved = (xb, gwb, idx, w, v, offsets, perm, pos, x_perm, ab, h, o, *wb)
    dx_rows, d_logits, dgw, dgb, grads_w = _backward_pass(ctx, saved, dy.contiguous())
    dx = K.dx_reduce(dx_rows, pos, idx, d_logits, gwb, idx.shape[0] * k, has_shared, x.dtype)
    return [dx, dgw, dgb, *grads_w]


@moe_bwd.register_fake
def _(dy, x, gate_w, gate_b, weights, idx, w, v, offsets, perm, pos, x_perm, ab, h, o, k, route_scale,
      has_shared):
    return [torch.empty_like(x), torch.empty_like(gate_w), torch.empty_like(gate_b),
            *[torch.empty_like(t) for t in weights]]


def _setup_context(ctx, inputs, output):
    x, gate_w, gate_b, weights, k, route_scale, has_shared, out_dtype = inputs
    y, idx64, w, counts, idx, v, offsets, perm, pos, x_perm, ab, h, o = output
    ctx.n_w = len(weights)
    ctx.args = (k, route_scale, has_shared)
    ctx.save_for_backward(x, gate_w, gate_b, idx, w, v, offsets, perm, pos, x_perm, ab, h, o, *weights)


def _backward(ctx, dy, *unused):
    x, gate_w, gate_b, idx, w, v, offsets, perm, pos, x_perm, ab, h, o, *weights = ctx.saved_tensors
    if dy is None:
        return None, None, None, [None] * ctx.n_w, None, None, None, None
    k, route_scale, has_shared = ctx.args
    g = torch.ops.fusionllm.moe_bwd(dy, x, gate_w, gate_b, weights, idx, w, v, offsets, perm, pos, x_perm,
                                    ab, h, o, k, route_scale, has_shared)
    return g[0], g[1], g[2], list(g[3:]), None, None, None, None


moe_fwd.register_autograd(_backward, setup_context=_setup_context)


@torch.library.custom_op("fusionllm::swiglu_fwd", mutates_args=())
def swiglu_fwd(x: Tensor, w1: Tensor, w3: Tensor, w2: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    T, d = x.shape
    inter = w1.shape[0]
    xb, w1b, w3b, w2b = _bf16_operands([x, w1, w3, w2])
    off = _dense_offsets(T, x.device)
    ab, h = K.gateup_fwd(xb, None, off, 1, [w1b], [w3b], inter)
    y = K.down_fwd(h, off, 1, T, 0, [w2b], d)
    return y, ab, h


@swiglu_fwd.register_fake
def _(x, w1, w3, w2):
    T, inter = x.shape[0], w1.shape[0]
    bf = torch.bfloat16
    return (x.new_empty((T, w2.shape[0]), dtype=bf), x.new_empty((T, 2 * inter), dtype=bf),
            x.new_empty((T, inter), dtype=bf))


@torch.library.custom_op("fusionllm::swiglu_bwd", mutates_args=())
def swiglu_bwd(dy: Tensor, x: Tensor, w1: Tensor, w3: Tensor, w2: Tensor, ab: Tensor, h: Tensor) -> list[Tensor]:
    xb, w1b, w3b, w2b = _bf16_operands([x, w1, w3, w2])
    off = _dense_offsets(x.shape[0], x.device)
    dx, dw1, dw3, dw2 = _dense_backward(dy, xb, ab, h, w1b, w3b, w2b, off,
                                        (x.dtype, w1.dtype, w3.dtype, w2.dtype), True)
    return [dx, dw1, dw3, dw2]


@swiglu_bwd.register_fake
def _(dy, x, w1, w3, w2, ab, h):
    return [torch.empty_like(x), torch.empty_like(w1), torch.empty_like(w3), torch.empty_like(w2)]


def _swiglu_setup(ctx, inputs, output):
    x, w1, w3, w2 = inputs
    y, ab, h = output
    ctx.save_for_backward(x, w1, w3, w2, ab, h)


def _swiglu_backward(ctx, dy, *unused):
    x, w1, w3, w2, ab, h = ctx.saved_tensors
    if dy is None:
        return None, None, None, None
    dx, dw1, dw3, dw2 = torch.ops.fusionllm.swiglu_bwd(dy, x, w1, w3, w2, ab, h)
    return dx, dw1, dw3, dw2


swiglu_fwd.register_autograd(_swiglu_backward, setup_context=_swiglu_setup)


@torch.library.custom_op("fusionllm::layer_norm_fwd", mutates_args=())
def layer_norm_fwd(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float,
                   out_dtype: torch.dtype) -> tuple[Tensor, Tensor, Tensor]:
    _norm.refuse_tangents("fusionllm::layer_norm_fwd", x, weight, bias)
    with _norm._on_device(x):
        return _norm._forward(x, weight, bias, eps, out_dtype, True)[2:]


@layer_norm_fwd.register_fake
def _(x, weight, bias, eps, out_dtype):
    T = x.shape[0]
    return (x.new_empty(x.shape, dtype=out_dtype), x.new_empty((T,), dtype=torch.float32),
            x.new_empty((T,), dtype=torch.float32))


@torch.library.custom_op("fusionllm::layer_norm_bwd", mutates_args=())
def layer_norm_bwd(dy: Tensor, x: Tensor, mean: Tensor, rstd: Tensor, weight: Tensor | None,
                   bias: Tensor | None) -> list[Tensor]:
    with _norm._on_device(x):
        grads = _norm._backward(dy, _norm._rows(x), None if weight is None else weight.contiguous(), mean, rstd, None,
                                True, None if weight is None else weight.dtype, None if bias is None else bias.dtype)
    return [g for g in grads if g is not None]


@layer_norm_bwd.register_fake
def _(dy, x, mean, rstd, weight, bias):
    return [x.new_empty(x.shape), *[p.new_empty(p.shape) for p in (weight, bias) if p is not None]]


def _layer_norm_setup(ctx, inputs, output):
    x, weight, bias, eps, out_dtype = inputs
    y, mean, rstd = output
    ctx.save_for_backward(x, weight, bias, mean, rstd)


def _layer_norm_backward(ctx, dy, *unused):
    x, weight, bias, mean, rstd = ctx.saved_tensors
    if dy is None:
        return None, None, None, None, None
    grads = iter(torch.ops.fusionllm.layer_norm_bwd(dy, x, mean, rstd, weight, bias))
    dx = next(grads)
    return (dx, None if weight is None else next(grads), None if bias is None else next(grads), None, None)


layer_norm_fwd.register_autograd(_layer_norm_backward, setup_context=_layer_norm_setup)


@torch.library.custom_op("fusionllm::embedding_fwd", mutates_args=())
def embedding_fwd(ids: Tensor, weight: Tensor, scale: float, padding_idx: int) -> Tensor:
    _norm.refuse_tangents("fusionllm::embedding_fwd", weight)
    with _norm._on_device(weight):
        return K.embedding_fwd(ids, _norm._rows(weight), scale)


@embedding_fwd.register_fake
def _(ids, weight, scale, padding_idx):
    return weight.new_empty((ids.shape[0], weight.shape[1]))


@torch.library.custom_op("fusionllm::embedding_bwd", mutates_args=())
def embedding_bwd(ids: Tensor, dy: Tensor, vocab: int, scale: float, padding_idx: int) -> Tensor:
    with _norm._on_device(dy):
        return K.embedding_bwd(ids, _norm._rows(dy), vocab, scale, padding_idx, dy.dtype)


@embedding_bwd.register_fake
def _(ids, dy, vocab, scale, padding_idx):
    return dy.new_empty((vocab, dy.shape[1]))


def _embedding_setup(ctx, inputs, output):
    ids, weight, scale, padding_idx = inputs
    ctx.save_for_backward(ids)
    ctx.args = (weight.shape[0], scale, padding_idx)


def _embedding_backward(ctx, dy):
    ids, = ctx.saved_tensors
    if dy is None:
        return None, None, None, None
    return None, torch.ops.fusionllm.embedding_bwd(ids, dy, *ctx.args), None, None


embedding_fwd.register_autograd(_embedding_backward, setup_context=_embedding_setup)


@torch.library.custom_op("fusionllm::vocab_loss_fwd", mutates_args=())
def vocab_loss_fwd(hidden: Tensor, weight: Tensor, index: Tensor, teacher: Tensor | None, ignore_index: int,
                   logit_scale: float, temperature: float, planes: int, reduction: str) -> tuple[Tensor, Tensor]:
    _norm.refuse_tangents("fusionllm::vocab_loss_fwd", hidden, weight)
    with _norm._on_device(weight):
        return K.vocab_loss_fwd(_norm._rows(hidden), _norm._rows(weight), index, teacher, ignore_index, logit_scale,
                                temperature, planes, reduction)


@vocab_loss_fwd.register_fake
def _(hidden, weight, index, teacher, ignore_index, logit_scale, temperature, planes, reduction):
    T, top = index.shape
    return (hidden.new_empty((T,) if reduction == "none" else (), dtype=torch.float32),
            hidden.new_empty((K.vocab_loss_state_bytes(T, hidden.shape[1], top, planes),), dtype=torch.uint8))


@torch.library.custom_op("fusionllm::vocab_loss_bwd", mutates_args=())
def vocab_loss_bwd(d_loss: Tensor, hidden: Tensor, weight: Tensor, state: Tensor, top: int, distill: bool,
                   logit_scale: float, temperature: float, planes: int, reduction: str, need_h: bool = True,
                   need_w: bool = True) -> list[Tensor]:
    """The gradients that are wanted; hidden gives its rows and dtype alone (any columns)."""
    with _norm._on_device(weight):
        out = K.vocab_loss_bwd(d_loss.contiguous(), _norm._rows(weight), state, hidden.shape[0], top, distill, logit_scale,
                               temperature, planes, reduction, hidden.dtype if need_h else None,
                               weight.dtype if need_w else None)
    return [t for t in out if t is not None]


@vocab_loss_bwd.register_fake
def _(d_loss, hidden, weight, state, top, distill, logit_scale, temperature, planes, reduction, need_h=True, need_w=True):
    return ([hidden.new_empty((hidden.shape[0], weight.shape[1]))] if need_h else []) + (
        [weight.new_empty(weight.shape)] if need_w else [])


def _vocab_loss_setup(ctx, inputs, output):
    hidden, weight, index, teacher, _, logit_scale, temperature, planes, reduction = inputs
    ctx.save_for_backward(weight, output[1])  # (the state holds the hidden states)
    ctx.hidden = (hidden.shape[0], hidden.dtype)
    ctx.args = (index.shape[1], teacher is not None, logit_scale, temperature, planes, reduction)


def _vocab_loss_backward(ctx, d_loss, *unused):
    weight, state = ctx.saved_tensors
    need = ctx.needs_input_grad[:2]
    if d_loss is None or not any(need):
        return (None,) * 9
    rows, dtype = ctx.hidden
    grads = iter(torch.ops.fusionllm.vocab_loss_bwd(d_loss, weight.new_empty((rows, 0), dtype=dtype), weight, state,
                                                    *ctx.args, *need))
    dh, dw = (next(grads) if n else None for n in need)
    return dh, dw, None, None, None, None, None, None, None


vocab_loss_fwd.register_autograd(_vocab_loss_backward, setup_context=_vocab_loss_setup)


@torch.library.custom_op("fusionllm::vocab_loss_fwd_grad", mutates_args=())
def vocab_loss_fwd_grad(hidden: Tensor, weight: Tensor, index: Tensor, teacher: Tensor | None, ignore_index: int,
                        logit_scale: float, temperature: float, planes: int, reduction: str, need_h: bool,
                        need_w: bool) -> list[Tensor]:
    _norm.refuse_tangents("fusionllm::vocab_loss_fwd_grad", hidden, weight)
    with _norm._on_device(weight):
        w = _norm._rows(weight)
        if not K.vocab_loss_takes_gradients(*hidden.shape, w.shape[0], planes, K.vocab_loss_packs(w, planes)):
            # chosen for a weight as it lies in a module; this one's address or stride needs a copy of its rows, which is more
            # than this form takes
            w = w.clone(memory_format=torch.contiguous_format)
        out = K.vocab_loss_fwd_grad(_norm._rows(hidden), w, index, teacher, ignore_index, logit_scale,
                                    temperature, planes, reduction, need_h, need_w)
    return [t for t in out if t is not None]


@vocab_loss_fwd_grad.register_fake
def _(hidden, weight, index, teacher, ignore_index, logit_scale, temperature, planes, reduction, need_h, need_w):
    out = [hidden.new_empty((), dtype=torch.float32)]
    return out + ([hidden.new_empty(hidden.shape)] if need_h else []) + ([weight.new_empty(weight.shape)] if need_w else [])


@torch.library.custom_op("fusionllm::scale", mutates_args=())
def scale(factor: Tensor, tensors: list[Tensor]) -> list[Tensor]:
    with _norm._on_device(factor):
        return K.scale(factor.contiguous(), tensors)


@scale.register_fake
def _(factor, tensors):
    return [torch.empty_like(t) for t in tensors]


def _vocab_loss_grad_setup(ctx, inputs, output):
    ctx.need = inputs[-2:]
    ctx.save_for_backward(*output[1:])


def _vocab_loss_grad_backward(ctx, d_outs):
    d_loss = d_outs[0]
    if d_loss is None:
        return (None,) * 11
    grads = iter(torch.ops.fusionllm.scale(d_loss, list(ctx.saved_tensors)))
    dh, dw = (next(grads) if need else None for need in ctx.need)
    return dh, dw, *(None,) * 9


vocab_loss_fwd_grad.register_autograd(_vocab_loss_grad_backward, setup_context=_vocab_loss_grad_setup)
