"""The embedding and the vocabulary losses on the GPU against their definitions in 64 bits.

Tolerances are error bounds, element by element, from the arithmetic that the kernels do:
u = 2^-24 is half a step of fp32 and h half a step of the operands' and results' type (bf16 2^-8, fp32 u).

* A dot product of K terms in fp32 is off by at most (K + 2) u sum |a b|; of operands in three planes (six products a
  term, products below 2^-23 of a term left out) by (6 K + 8) u sum |a b|.
* A logit of size up to A in sums of |h w| is off by e = dot u A (plus two roundings of the logit itself).  A
  maximum and a logsumexp are off by no more than that, plus the relative error of the sum of exponentials: 32 terms in a
  lane, 6 joins, then one per 128 columns, each with up to 4 roundings.
* p = exp(s - lse) has the relative error of both, d; G = up (p - q) the error d up p, and half a step h of its own.
* dH = G W and dW = G^T H: what G is off by times |W| or |H|, the dot product's own error and the result's rounding.
"""
import math

import pytest
import torch

import fusionllm_amd
from fusionllm_amd import embedding, linear_cross_entropy, linear_distillation

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}
DTYPES = [torch.bfloat16, torch.float32]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _within(got, want, bound, what):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                                 f"{float((err / bound.clamp_min(1e-300))[bad].max()):.3g} of the bound")


# ---- embedding --------------------------------------------------------------------


def _embed_bound(ids, dy, w, scale, pad):
    """d_weight in 64 bits and its bound."""
    keep = (ids >= 0) & (ids < w.shape[0])
    if pad is not None:
        keep &= ids != pad
    ids, dy = ids[keep].long(), dy.double()[keep]
    zeros = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    want = zeros.clone().index_add_(0, ids, dy) * scale
    size = zeros.clone().index_add_(0, ids, dy.abs()) * abs(scale)
    count = torch.bincount(ids, minlength=w.shape[0]).double()[:, None]
    return want, (count + 2) * U * size + HALF[w.dtype] * want.abs()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,D,scale", [(1, 1, 1, 1.0), (1, 32768, 768, 1.0), (7, 3, 5, 2.5), (64, 512, 512, 1.0),
                                         (601, 513, 2048, 45.25), (1000, 1024, 513, -0.5), (4099, 50021, 1000, 1.0),
                                         (3000, 7, 768, 1.0), (40000, 2, 64, 27.75), (9000, 1, 520, 1.0)])
def test_embedding_and_its_gradient(gpu_device, T, V, D, scale, dtype):
    g = _gen(T + V)
    w = torch.randn(V, D, generator=g).to(gpu_device, dtype).requires_grad_(True)
    ids = (V * torch.rand(T, generator=g) ** 3).long().clamp(max=V - 1).to(gpu_device)
    dy = torch.randn(T, D, generator=g).to(gpu_device, dtype)
    for index in (ids, ids.int()):
        y = embedding(index, w, scale)
        assert torch.equal(y, (w.detach().float()[ids] * scale).to(dtype))
        dw, = torch.autograd.grad(y, [w], dy)
        _within(dw, *_embed_bound(ids, dy, w.detach(), scale, None), "d_weight")
    again, = torch.autograd.grad(embedding(ids, w, scale), [w], dy)
    assert torch.equal(dw, again)


@pytest.mark.parametrize("pad", [0, 5, -1])
def test_embedding_padding_invalid_ids_and_strides(gpu_device, pad):
    g = _gen(pad + 2)
    V, D = 700, 96
    w = torch.randn(V, 2 * D, generator=g).to(gpu_device)[:, :D].requires_grad_(True)  # rows that lie apart
    ids = torch.randint(0, V, (50, 41), generator=g)
    ids[torch.rand(ids.shape, generator=g) < 0.3] = pad % V
    ids[3, 4], ids[5, 6], ids[7, 8] = -1, V, 2 ** 40
    ids = ids.to(gpu_device)
    dy = torch.randn(50, 41, 2 * D, generator=g).to(gpu_device)[..., D:]
    y = embedding(ids.t().contiguous().t(), w, 1.5, padding_idx=pad)
    good = (ids >= 0) & (ids < V)
    assert torch.equal(y[good], w.detach()[ids[good]] * 1.5) and bool(y[~good].isnan().all())
    dw, = torch.autograd.grad(y, [w], dy)
    want, bound = _embed_bound(ids.flatten(), dy.reshape(-1, D), w.detach(), 1.5, pad % V)
    _within(dw, want, bound, "d_weight")
    assert not dw[pad % V].any()


def test_embedding_module_and_empty_batches(gpu_device):
    torch.manual_seed(0)
    m = fusionllm_amd.Embedding(100, 64, padding_idx=3, scale=8.0).to(gpu_device)
    ref = torch.nn.Embedding(100, 64, padding_idx=3).to(gpu_device)
    ref.load_state_dict(m.state_dict())
    ids = torch.randint(0, 100, (6, 9), device=gpu_device)
    dy = torch.randn(6, 9, 64, device=gpu_device)
    a, b = m(ids), ref(ids) * 8.0
    assert torch.equal(a, b)
    a.backward(dy)
    b.backward(dy)
    torch.testing.assert_close(m.weight.grad, ref.weight.grad, rtol=56 * U, atol=56 * U * 8 * 54)
    m.weight.grad = None
    e = m(ids[:0])
    assert e.shape == (0, 9, 64)
    e.sum().backward()
    assert not m.weight.grad.any()


# ---- losses ---------------------------------------------------------------------------


def _reference(hidden, weight, lists, teacher, ignore, scale, tau, reduction, up):
    """Loss, gradients and their bounds (see above) of one call, in 64 bits; up: the loss's gradient."""
    dtype = weight.dtype
    planes = 3 if dtype == torch.float32 and hidden.dtype == torch.float32 else 1
    H, W = hidden.detach().double(), weight.detach().double()
    (T, D), V = H.shape, W.shape[0]
    dot = lambda k: (6 * k + 8 if planes == 3 else k + 2) * U
    there = lists != ignore
    if teacher is not None:
        there &= teacher != -math.inf
    rows = there.any(1)
    n = int(rows.sum())
    H = torch.where(rows[:, None], H, 0.0)
    f = scale / tau
    s = (H @ W.T) * f
    size = (H.abs() @ W.abs().T) * abs(f)
    e = size.amax(1, keepdim=True) * (dot(D) + 6 * U)  # of a logit, and of the maximum
    lse = torch.logsumexp(s, 1, keepdim=True)
    d = 4 * e + (64 + 4 * (V / 128 + 8)) * U + 6 * U * (s - lse).abs()  # of p, relative; of log p, absolute
    p = torch.exp(s - lse)
    idx = torch.where(there, lists, 0).long()
    if teacher is None:
        q, log_q = there.double(), torch.zeros_like(there, dtype=torch.float64)
    else:
        z = torch.where(there, teacher.double() / tau, -math.inf)
        z = torch.where(rows[:, None], z, 0.0)
        log_q = torch.log_softmax(z, 1)
        q = torch.where(there, log_q.exp(), 0.0)
        log_q = torch.where(there & (q > 0), log_q, 0.0)
        log_q = torch.where(log_q == -math.inf, 0.0, log_q)
    log_p = (s - lse).gather(1, idx)
    per_row = tau ** 2 * (q * (log_q - log_p)).sum(1)
    # q and ln q: the logits over the temperature, their maximum, a sum of K terms, an exponential
    K = lists.shape[1]
    zsize = 0.0 if teacher is None else torch.where(there, (teacher.double() / tau).abs(), 0.0).amax(1)
    dq = (4 * zsize + K + 40) * U if teacher is not None else 0.0
    row_bound = tau ** 2 * (d.amax(1) + dq * (1 + (q * (log_q.abs() + log_p.abs())).sum(1)) +
                            (K + 16) * U * (q * (log_q.abs() + log_p.abs())).sum(1)) + 4 * U * per_row.abs()
    row_bound = torch.where(rows, row_bound, 0.0)
    per_row = torch.where(rows, per_row, 0.0)
    if reduction == "none":
        loss, bound, share = per_row, row_bound, up.double()
    elif reduction == "mean":
        loss, bound = per_row.sum() / n, row_bound.mean() * T / n + U * per_row.sum().abs() / n
        share = torch.full((T,), float(up) / n, dtype=torch.float64, device=H.device)
    else:
        loss, bound = per_row.sum(), row_bound.sum() + U * per_row.sum().abs()
        share = torch.full((T,), float(up), dtype=torch.float64, device=H.device)
    c = (torch.where(rows, share, 0.0) * tau * scale)[:, None]
    target = torch.zeros_like(p).scatter_add_(1, idx, q)
    G = c * (p - target)
    g_half = HALF[torch.bfloat16] if planes == 1 else 4 * U
    dG = c.abs() * ((d + 8 * U) * p + (dq if teacher is None else dq[:, None]) * target + 4 * U * (p + target)) + g_half * G.abs()
    out_h, out_w = HALF[hidden.dtype], HALF[weight.dtype]
    dH, dW = G @ W, G.T @ H
    bH = dG @ W.abs() + (dot(V) + 80 * U) * (G.abs() @ W.abs()) + out_h * dH.abs()
    bW = dG.T @ H.abs() + dot(T) * (G.abs().T @ H.abs()) + out_w * dW.abs()
    return (loss, bound * 1.0001 + 1e-30), (dH, bH * 1.01 + 1e-30), (dW, bW * 1.01 + 1e-30)


def _operands(g, T, V, D, dtype, device, pull=True):
    w = (torch.randn(V, D, generator=g) / math.sqrt(D)).to(dtype)
    t = (V * torch.rand(T, generator=g) ** 2).long().clamp(max=V - 1)
    h = torch.randn(T, D, generator=g)
    if pull:  # some rows are sure of their target
        h = h + 14 * torch.rand(T, 1, generator=g) * w[t].float()
    return h.to(device, dtype).requires_grad_(True), w.to(device).requires_grad_(True), t.to(device)


def _check(loss, h, w, up, want):
    (l, bl), (dh, bh), (dw, bw) = want
    _within(loss.detach(), l, bl, "loss")
    gh, gw = torch.autograd.grad(loss, [h, w], up)
    assert gh.dtype == h.dtype and gw.dtype == w.dtype
    _within(gh, dh, bh, "d_hidden")
    _within(gw, dw, bw, "d_weight")
    return gh, gw


SIZES = [(1, 2, 8), (1, 300, 64), (1, 32768, 768), (37, 5003, 768), (64, 64, 48), (65, 257, 128), (300, 777, 1001),
         (513, 4096, 256), (700, 10007, 192), (1030, 1000, 320)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("T,V,D", SIZES)
def test_cross_entropy(gpu_device, T, V, D, reduction, dtype):
    g = _gen(T + V + D)
    h, w, t = _operands(g, T, V, D, dtype, gpu_device)
    if T > 1:
        t[torch.randperm(T, generator=g)[:T // 3].to(gpu_device)] = -100
    scale = 0.75 if T % 2 else 1.0
    up = torch.rand(T, generator=g).to(gpu_device) if reduction == "none" else torch.tensor(0.5, device=gpu_device)
    loss = linear_cross_entropy(h, w, t.int() if T % 3 else t, reduction=reduction, logit_scale=scale)
    assert loss.dtype == torch.float32 and loss.shape == ((T,) if reduction == "none" else ())
    grads = _check(loss, h, w, up, _reference(h, w, t[:, None], None, -100, scale, 1.0, reduction, up))
    assert not grads[0][t == -100].any()
    again = torch.autograd.grad(linear_cross_entropy(h, w, t, reduction=reduction, logit_scale=scale), [h, w], up)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(h, w, t, reduction=reduction, logit_scale=scale), loss)


def _lists(g, T, V, K, device, repeat=False):
    if repeat:
        index = torch.randint(0, V, (T, K), generator=g)
        index[:, K // 2:] = index[:, :K - K // 2]
    else:
        index = torch.rand(T, V, generator=g).argsort(1)[:, :K]
    return index.to(device), (4 * torch.randn(T, K, generator=g)).to(device)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction,tau", [("mean", 1.0), ("none", 2.0), ("sum", 0.5)])
@pytest.mark.parametrize("T,V,D,K", [(1, 40, 64, 1), (3, 1000, 96, 1000), (50, 300, 64, 7), (129, 5003, 768, 64),
                                     (300, 777, 1001, 100)])
def test_distillation(gpu_device, T, V, D, K, reduction, tau, dtype):
    g = _gen(T + V + K)
    h, w, _ = _operands(g, T, V, D, dtype, gpu_device, pull=False)
    index, z = _lists(g, T, V, K, gpu_device)
    if T > 1:  # lists of different lengths, one row in four without entries
        length = torch.randint(0, K + 1, (T, 1), generator=g)
        length[torch.rand(T, 1, generator=g) < 0.25] = 0
        length[0] = K
        index = torch.where((torch.arange(K) < length).to(gpu_device), index, -100)
    z = z.to(dtype)
    up = torch.rand(T, generator=g).to(gpu_device) if reduction == "none" else torch.tensor(2.0, device=gpu_device)
    loss = linear_distillation(h, w, index, z, temperature=tau, reduction=reduction, logit_scale=0.9)
    _check(loss, h, w, up, _reference(h, w, index, z, -100, 0.9, tau, reduction, up))
