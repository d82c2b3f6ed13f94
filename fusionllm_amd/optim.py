"""Optimizers of the weight matrices: NorMuon, Muon and the orthogonalisation it uses.

``NorMuon``: drop-in for the reference's (training/optimizer.py:11-58).  Same constructor (params, lr, betas, eps, weight_decay, cautious_wd), the
same per-parameter state ("step", "exp_avg", "exp_avg_sq", so optimizer
checkpoints (training/checkpoint.py:19-40) load either way) and the same
update.  ``step()`` runs the update as fused kernels
(``fmoe_normuon_step``): one launch per 32 tensors of one dtype and step
count reads grad, param, exp_avg and exp_avg_sq once and writes the three
updated tensors once, where the reference issues about fifteen tensor
operations per parameter.  Parameters must be ROCm tensors in bf16 or fp32
with a last dimension that is a multiple of 4 and at most 4096 (every weight
matrix of the reference model); anything else raises.

``orthogonalize`` replaces matrices by their orthogonalised form (an odd
polynomial of the singular values, by Newton-Schulz products), every matrix of
one pair of sides in the same launches.  ``Muon`` is momentum, that form of the
update, decoupled weight decay and the parameter's update in the same launches,
with the constructor and state of ``torch.optim.Muon``.  Matrices are bf16 or
fp32; the products of bf16 matrices run on fp16 operands with fp32 sums, those of
fp32 matrices on pairs of fp16 operands (22 bits).
"""
from __future__ import annotations

import bisect
import math

import torch
from torch.optim import Optimizer

from . import _kernels as K
from .norm import refuse_tangents


class NorMuon(Optimizer):
    """NorMuon: Adam moments, per-row RMS normalisation of the update and
    cautious weight decay (reference: training/optimizer.py:11-58)."""

    def __init__(self, params, lr: float = 0.02, betas: tuple[float, float] = (0.9, 0.95), eps: float = 1e-8,
                 weight_decay: float = 0.1, cautious_wd: bool = True):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, cautious_wd=cautious_wd)
        super().__init__(params, defaults)

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        for group in self.param_groups:
            lr, (beta1, beta2) = group["lr"], group["betas"]
            eps, wd, cautious = group["eps"], group["weight_decay"], group["cautious_wd"]
            batches: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                grad = p.grad
                if not p.is_cuda:
                    raise RuntimeError("fusionllm_amd.optim.NorMuon runs on a ROCm device only")
                if p.dtype not in (torch.bfloat16, torch.float32) or grad.dtype != p.dtype:
                    raise NotImplementedError(f"NorMuon step for {p.dtype} parameters with {grad.dtype} grads")
                if not (p.is_contiguous() and grad.is_contiguous()):
                    raise NotImplementedError("NorMuon step needs contiguous parameters and gradients")
                c = p.shape[-1] if p.dim() >= 1 else 1
                if c % 4 != 0 or c > 4096:
                    raise NotImplementedError(f"NorMuon step for last dimension {c} (needs a multiple of 4, <= 4096)")
                state = self.state[p]
                if len(state) == 0:
                    state["step"] = 0
                    state["exp_avg"] = torch.zeros_like(grad)
                    state["exp_avg_sq"] = torch.zeros_like(grad)
                state["step"] += 1
                key = (p.device, p.dtype, state["step"])
                batches.setdefault(key, []).append((p, grad, state["exp_avg"], state["exp_avg_sq"]))
            for (dev, _dtype, step), items in batches.items():
                bias_corr1 = 1.0 - beta1 ** step
                bias_corr2 = 1.0 - beta2 ** step
                with torch.cuda.device(dev):
                    for i in range(0, len(items), K.NORMUON_MAX_TENSORS):
                        chunk = items[i:i + K.NORMUON_MAX_TENSORS]
                        K.normuon_step([t[0] for t in chunk], [t[1] for t in chunk], [t[2] for t in chunk],
                                       [t[3] for t in chunk], lr, beta1, beta2, eps, wd, cautious,
                                       bias_corr1, bias_corr2)
        return loss


NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


# Elements of one launch's matrices, at most (one matrix may have more): its workspace takes 5 to 8 bytes
# for each and as much again for square ones, and this many fill the chip many times over.
LAUNCH_ELEMENTS = 1 << 28


def _sides(t):
    r, c = t.shape
    return (r, c) if r <= c else (c, r)


class _Spans:
    """Ranges of addresses, kept sorted and disjoint (those that meet become one)."""

    def __init__(self):
        self.lo, self.hi = [], []

    def _meeting(self, lo, hi):
        return bisect.bisect_right(self.hi, lo), bisect.bisect_left(self.lo, hi)

    def meets(self, lo, hi):
        i, j = self._meeting(lo, hi)
        return i < j

    def add(self, lo, hi):
        i, j = self._meeting(lo, hi)
        if i < j:
            lo, hi = min(lo, self.lo[i]), max(hi, self.hi[j - 1])
        self.lo[i:j], self.hi[i:j] = [lo], [hi]


def _span(t):
    """Addresses from a tensor's first element to the end of its last."""
    n = t.numel() if t.is_contiguous() else 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    lo = t.data_ptr()
    return lo, lo + n * t.element_size()


class _Launch:
    def __init__(self):
        self.items, self.written, self.read = [], _Spans(), _Spans()

    def conflicts(self, written, read):
        return (any(self.written.meets(*s) or self.read.meets(*s) for s in written)
                or any(self.written.meets(*s) for s in read))

    def add(self, written, read):
        for s in written:
            self.written.add(*s)
        for s in read:
            self.read.add(*s)


def _apart(written, read):
    """Whether no written span meets another one (read spans may meet each other)."""
    spans = sorted([(lo, hi, True) for w in written for lo, hi in w] + [(lo, hi, False) for r in read for lo, hi in r])
    end = end_written = 0
    for lo, hi, w in spans:
        if lo < (end if w else end_written):
            return False
        if hi > end:
            end = hi
        if w and hi > end_written:
            end_written = hi
    return True


def _launches(items, written=lambda it: (), read=lambda it: ()):
    """Lists of items (tuples whose first tensor is the matrix) for one launch each: one device, dtype and
    pair of sides, at most MUON_MAX_TENSORS and LAUNCH_ELEMENTS, and no two of which one writes
    memory that the other writes or reads (written(item), read(item): tensors).  Two such items, of whatever
    sides, are in launches of their order: an item joins its sides' last launch only if it conflicts
    neither with that nor with any launch behind it."""
    w, r = [[_span(x) for x in written(it)] for it in items], [[_span(x) for x in read(it)] for it in items]
    apart = _apart(w, r)  # as ever, but for tied and overlapping parameters
    last: dict = {}  # place of the last launch of each device, dtype and sides
    out: list = []
    for i, it in enumerate(items):
        t = it[0]
        key = (t.device, t.dtype, _sides(t))
        at = last.get(key)
        if (at is None or len(out[at].items) >= min(K.MUON_MAX_TENSORS, max(1, LAUNCH_ELEMENTS // t.numel()))
                or (not apart and any(c.conflicts(w[i], r[i]) for c in out[at:]))):
            at = last[key] = len(out)
            out.append(_Launch())
        out[at].items.append(it)
        if not apart:
            out[at].add(w[i], r[i])
    return [c.items for c in out]


def _check_ns(steps, coefficients, eps):
    if len(coefficients) != 3:
        raise ValueError(f"three coefficients are needed (got {len(coefficients)})")
    if not 1 <= steps <= K.MUON_MAX_STEPS:
        raise ValueError(f"the number of Newton-Schulz steps must be 1 to {K.MUON_MAX_STEPS} (got {steps})")
    if not eps > 0:
        raise ValueError(f"eps must be positive (got {eps})")


def _check_matrix(what, t):
    if not t.is_cuda:
        raise RuntimeError(f"{what} runs on a ROCm device only (got a {t.device.type} tensor)")
    if t.dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError(f"{what} supports bf16 and fp32 matrices (got {t.dtype})")
    if max(t.shape[-2:]) > K.MUON_MAX_SIDE:
        raise NotImplementedError(f"{what} takes sides up to {K.MUON_MAX_SIDE} (got {tuple(t.shape)})")
    r, c = (-(-s // 64) * 64 for s in t.shape[-2:])
    if r * c > K.MUON_MAX_ELEMENTS:
        raise NotImplementedError(f"{what} takes matrices of up to {K.MUON_MAX_ELEMENTS} elements (got "
                                  f"{tuple(t.shape)})")


def orthogonalize(mats, steps: int = 5, coefficients=NS_COEFFICIENTS, eps: float = 1e-7):
    """Orthogonalised matrices: X = G / max(|G|_F, eps), then ``steps`` times X = a X + (b A + c A^2) X
    with A = X X^T, on the shorter side.

    mats: a tensor [..., rows, cols] (every matrix of the stack), or a list of such tensors; the result
    has the same structure, shapes and dtypes.  No backward pass.  The coefficients must keep the
    singular values below 2.8 (the defaults do).  The result of a matrix whose norm is far below eps is
    nearly zero; beside its relative error, an element of any result is off by up to about
    steps |a|^steps 2^-38 (2^-27 with the defaults)."""
    single = isinstance(mats, torch.Tensor)
    stacks = [mats] if single else list(mats)
    _check_ns(steps, coefficients, eps)
    for t in stacks:
        if t.dim() < 2:
            raise ValueError(f"orthogonalize takes matrices (got shape {tuple(t.shape)})")
        _check_matrix("orthogonalize", t)
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("orthogonalize has no backward pass: call it under no_grad or on detached matrices")
        refuse_tangents("orthogonalize", t)
    outs, items = [], []
    for t in stacks:
        t = t.detach().contiguous()
        out = torch.empty_like(t)
        outs.append(out)
        if t.numel():
            items += zip(t.view(-1, *t.shape[-2:]), out.view(-1, *t.shape[-2:]))
    for chunk in _launches(items):  # (the results' memory is new)
        with torch.cuda.device(chunk[0][0].device):
            K.orthogonalize([c[0] for c in chunk], [c[1] for c in chunk], steps, coefficients, eps)
    return outs[0] if single else outs


class Muon(Optimizer):
    """Muon: momentum, the update orthogonalised by Newton-Schulz products, decoupled weight decay.

        buf = momentum buf + (1 - momentum) grad
        u   = (1 - momentum) grad + momentum buf  if nesterov else buf
        p   = p (1 - lr weight_decay) - lr' orthogonalize(u)

    with lr' = lr sqrt(max(1, rows / cols)) (adjust_lr_fn None or "original") or
    lr 0.2 sqrt(max(rows, cols)) ("match_rms_adamw").  The constructor and the
    state ("momentum_buffer") are those of ``torch.optim.Muon``.  Parameters are
    matrices on a ROCm device, bf16 or fp32, with gradients of their own dtype;
    every matrix of one dtype and pair of sides is updated in the same launches.
    What a step refuses it refuses before anything is updated.  A step can be captured into a
    graph once every matrix has its momentum; the graph keeps the step sizes of the capture."""

    def __init__(self, params, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95,
                 nesterov: bool = True, ns_coefficients=NS_COEFFICIENTS, eps: float = 1e-7, ns_steps: int = 5,
                 adjust_lr_fn: str | None = None):
        if lr < 0:
            raise ValueError(f"the learning rate must not be negative (got {lr})")
        if weight_decay < 0:
            raise ValueError(f"the weight decay must not be negative (got {weight_decay})")
        if not 0 <= momentum < 1:
            raise ValueError(f"the momentum must be in [0, 1) (got {momentum})")
        if adjust_lr_fn not in (None, "original", "match_rms_adamw"):
            raise ValueError(f"unknown learning rate adjustment {adjust_lr_fn!r}")
        _check_ns(ns_steps, ns_coefficients, eps)
        defaults = dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                        ns_coefficients=tuple(ns_coefficients), eps=eps, ns_steps=ns_steps,
                        adjust_lr_fn=adjust_lr_fn)
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        ps = group["params"]
        try:
            if len(set(ps)) != len(ps):
                raise ValueError("a parameter is given twice")
            for p in ps:
                if p.dim() != 2:
                    raise ValueError(f"Muon takes matrices (got a parameter of shape {tuple(p.shape)})")
            self._check_group(group)
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(group):
        _check_ns(group["ns_steps"], group["ns_coefficients"], group["eps"])
        K.check_newton_schulz(group["ns_steps"], group["ns_coefficients"])

    def _group_items(self, group):
        """(parameter, gradient, momentum or None) of a group's matrices that have something to do, checked."""
        self._check_group(group)
        items = []
        for p in group["params"]:
            g = p.grad
            if g is None or p.numel() == 0:
                continue
            _check_matrix("fusionllm_amd.optim.Muon", p)
            if g.dtype != p.dtype or g.layout != torch.strided or g.device != p.device:
                raise NotImplementedError(f"Muon step for a {p.dtype} parameter on {p.device} with a {g.dtype} {g.layout} "
                                          f"grad on {g.device}")
            if not p.is_contiguous():
                raise NotImplementedError("Muon step needs contiguous parameters")
            state = self.state.get(p)
            buf = state.get("momentum_buffer") if state else None
            if buf is not None and (buf.shape != p.shape or buf.dtype != p.dtype or buf.device != p.device
                                    or not buf.is_contiguous()):
                raise RuntimeError("the momentum buffer must be contiguous, with its parameter's shape, dtype and device "
                                   f"(got {tuple(buf.shape)}, {buf.dtype}, {buf.device})")
            items.append((p, g, buf))
        return items

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # every group is checked before any is updated: a step that is refused has changed nothing
        todo = [(group, float(group["lr"]), float(group["weight_decay"]), float(group["momentum"]),
                 self._group_items(group)) for group in self.param_groups]
        if any(it[2] is None for t in todo for it in t[-1]) and torch.cuda.is_current_stream_capturing():
            # the zeros would be part of the graph and clear the momentum in every replay
            raise RuntimeError("Muon: a step that creates momentum buffers cannot be captured into a graph; run one "
                               "before the capture")
        for group, lr, wd, momentum, items in todo:
            for i, (p, g, buf) in enumerate(items):
                if buf is None:
                    state = self.state[p]
                    if state.get("momentum_buffer") is None:
                        state["momentum_buffer"] = torch.zeros_like(p)
                    items[i] = (p, g, state["momentum_buffer"])
            for chunk in _launches(items, lambda it: (it[0], it[2]), lambda it: (it[1],)):
                small, large = _sides(chunk[0][0])
                if group["adjust_lr_fn"] == "match_rms_adamw":
                    tall = wide = lr * 0.2 * math.sqrt(large)
                else:
                    tall, wide = lr * math.sqrt(large / small), lr
                with torch.cuda.device(chunk[0][0].device):
                    K.muon_step([c[0] for c in chunk], [c[1].contiguous() for c in chunk], [c[2] for c in chunk],
                                tall, wide, 1.0 - lr * wd, momentum, group["nesterov"], group["ns_steps"],
                                group["ns_coefficients"], group["eps"])
        return loss
