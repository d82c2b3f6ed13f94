"""Layer norm on the kernels: ``layer_norm`` and the module ``LayerNorm``, beside
the RMSNorm that ``moe_residual`` fuses around the block.

``layer_norm(x, weight, bias, eps)`` is

    mean = sum(x) / D,  r = 1 / sqrt(sum((x - mean)^2) / D + eps)
    y = ((x - mean) * r) * weight + bias

over the last dimension, one read of x and one write of y, with fp32
arithmetic and one rounding, to the result's dtype.  The backward reads x and
dy once, writes dx, and reduces the weight's and bias's gradients in a fixed
order (the same bits every run).  x is bf16 or fp32, weight and bias share one
of these dtypes (not necessarily x's); the result has x's dtype, and fp32 under
autocast, where torch's layer norm returns fp32.  Rows may lie apart (a slice
of wider rows); the normalised dimension is at most 16384.  ROCm tensors only.
"""
from __future__ import annotations

import contextlib

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _kernels as K


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [T, D] as the kernels take it: elements of a row adjacent, rows that do not overlap."""
    T, dim = x.shape
    if x.is_contiguous() or (dim > 1 and x.stride(1) == 1 and (T <= 1 or x.stride(0) >= dim)):
        return x
    return x.contiguous()


def _on_device(t: torch.Tensor):
    # Switch devices only when needed (the context manager costs host time).
    switch = t.device.index != torch._C._cuda_getDevice()
    return torch.cuda.device(t.device) if switch else contextlib.nullcontext()


def _forward(x, weight, bias, eps, out_dtype, stats):
    xr = _rows(x)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    return xr, w, *K.layer_norm_fwd(xr, w, b, eps, out_dtype, stats)


def _backward(dy, x, w, mean, rstd, d_residual, need_dx, w_dtype, b_dtype):
    """(dx, dw, db), each None where it is not wanted (a dtype of None: no such gradient)."""
    return K.layer_norm_bwd(_rows(dy), x, mean, rstd, w, d_residual, need_dx, w_dtype, b_dtype)


class _LayerNormFunction(torch.autograd.Function):
    """The layer norm through the Python wrappers (the native form, csrc/block_host.cpp, runs the same entry points)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        with _on_device(x):
            xr, w, y, mean, rstd = _forward(x, weight, bias, eps, out_dtype, True)
        ctx.save_for_backward(xr, w, mean, rstd)
        ctx.dtypes = (None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, mean, rstd = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        with _on_device(x):
            dx, dw, db = _backward(dy, x, w, mean, rstd, None, need_x, ctx.dtypes[0] if need_w else None,
                                   ctx.dtypes[1] if need_b else None)
        return dx, dw, db, None, None


def refuse_tangents(what, *tensors):
    """A tensor with a tangent (forward-mode derivatives) need not require a gradient: without this
    the result would come without one."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def check_norm_operands(x, weight, bias):
    what = "fusionllm_amd.layer_norm"
    if not x.is_cuda:
        raise RuntimeError(f"{what} runs on a ROCm device only (got a {x.device.type} tensor)")
    if x.dim() == 0:
        raise ValueError(f"{what} needs at least one dimension")
    dim = x.shape[-1]
    if not 1 <= dim <= K.LAYER_NORM_MAX_DIM:
        raise NotImplementedError(f"{what} takes a last dimension of 1 to {K.LAYER_NORM_MAX_DIM} (got {dim})")
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError(f"{what} supports bf16 and fp32 tensors (got {x.dtype})")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (dim,):
            raise ValueError(f"{what}: {name} must have shape ({dim},) (got {tuple(p.shape)})")
        if p.device != x.device:
            raise RuntimeError(f"{what}: {name} must be on the input's device")
        if p.dtype not in (torch.bfloat16, torch.float32):
            raise NotImplementedError(f"{what} supports bf16 and fp32 parameters (got {p.dtype})")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise NotImplementedError(f"{what}: weight and bias must have one dtype")


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of x over its last dimension (any leading shape)."""
    check_norm_operands(x, weight, bias)
    out_dtype = torch.float32 if torch.is_autocast_enabled("cuda") else x.dtype
    flat = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if torch.compiler.is_compiling():
        # traced (torch.compile): the fusionllm::layer_norm_fwd operator
        y = torch.ops.fusionllm.layer_norm_fwd(flat, weight, bias, float(eps), out_dtype)[0]
    else:
        refuse_tangents("fusionllm_amd.layer_norm", x, weight, bias)
        grad = torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                            or (bias is not None and bias.requires_grad))
        host = K.block_host()
        if host is not None:
            y = host.layer_norm(flat, weight, bias, eps, out_dtype, grad)
        elif grad:  # through the wrappers, which time their calls
            y = _LayerNormFunction.apply(flat, weight, bias, float(eps), out_dtype)
        else:
            with _on_device(flat):
                y = _forward(flat, weight, bias, float(eps), out_dtype, False)[2]
    return y if x.dim() == 2 else y.view(x.shape)


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm`` on the kernels: the same constructor, parameters and
    state dict.  After it, ``moe_residual`` runs the norm, the block and the
    residual add fused."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        k = len(self.normalized_shape)
        if tuple(input.shape[input.dim() - k:]) != tuple(self.normalized_shape):
            raise RuntimeError(f"expected an input of shape [*, {', '.join(map(str, self.normalized_shape))}] "
                               f"(got {tuple(input.shape)})")
        if k == 1:
            return layer_norm(input, self.weight, self.bias, self.eps)
        flat = lambda p: None if p is None else p.flatten()
        return layer_norm(input.flatten(-k), flat(self.weight), flat(self.bias), self.eps).view(input.shape)
