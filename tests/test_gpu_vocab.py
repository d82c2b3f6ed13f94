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
* Where a loss of one value forms its gradients at once (more than 64 rows), the rows' factors go into H before
  dW's product: one more rounding of each of its terms, half a step h.
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
                                         (64, 1, 1500, 0.5), (63, 4099, 520, 2.0), (65, 2, 300, 1.0),
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
    # gradients formed in the forward are rounded to their dtype there, as for a loss's gradient of 1, and once more when that
    # gradient, up, multiplies them: (x (1 + a)) up (1 + b) = x up (1 + a + b + a b) with |a|, |b| up to half a step, and b = 0
    # where up is a power of two (the 1.01 below covers a b)
    twice = 2 if reduction != "none" and T > 64 and math.frexp(float(up))[0] != 0.5 else 1
    out_h, out_w = twice * HALF[hidden.dtype], twice * HALF[weight.dtype]
    dH, dW = G @ W, G.T @ H
    bH = dG @ W.abs() + (dot(V) + 80 * U) * (G.abs() @ W.abs()) + out_h * dH.abs()
    again = g_half if reduction != "none" and T > 64 else 0.0
    bW = dG.T @ H.abs() + (dot(T) + again) * (G.abs().T @ H.abs()) + out_w * dW.abs()
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


SIZES = [(1, 2, 8), (1, 300, 64), (1, 32768, 768), (16, 900, 4099), (20, 384, 520), (37, 5003, 768), (64, 64, 48),
         (64, 1281, 1500), (65, 257, 128), (300, 777, 1001),
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
        only = linear_cross_entropy(h, w, t, reduction=reduction, logit_scale=scale)
    if reduction == "none" or T <= 64:
        assert torch.equal(only, loss)
    else:  # (with gradients, the exponentials are relative to another logit: other roundings within the same bound)
        want = _reference(h, w, t[:, None], None, -100, scale, 1.0, reduction, up)[0]
        _within(only, *want, "loss without gradients")


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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("T,V,D,K", [(1500, 60000, 512, 800), (1030, 130, 96, 50)])
def test_long_lists(gpu_device, T, V, D, K, reduction, dtype):
    # lists read from stored logits, the first in two parts of the rows
    g = _gen(T + K)
    h, w, _ = _operands(g, T, V, D, dtype, gpu_device, pull=False)
    index, z = _lists(g, T, V, K, gpu_device, repeat=True)
    index[::6] = -100
    z = z.to(dtype)
    up = torch.rand(T, generator=g).to(gpu_device) if reduction == "none" else torch.tensor(1.0, device=gpu_device)
    loss = linear_distillation(h, w, index, z, temperature=2.0, reduction=reduction)
    _check(loss, h, w, up, _reference(h, w, index, z, -100, 1.0, 2.0, reduction, up))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction,scale", [("mean", -1.5), ("none", 0.0), ("sum", 3.0)])
@pytest.mark.parametrize("T,V,D,K", [(64, 1, 1, 6), (65, 1, 1, 3), (33, 130, 65, 1024), (1024, 2, 9, 1), (1025, 33, 9, 1024),
                                     (2049, 257, 100, 40), (4097, 300, 72, 5)])
def test_smallest_vocabularies_longest_lists_and_signs(gpu_device, T, V, D, K, reduction, scale, dtype):
    g = _gen(T + V + K)
    h, w, t = _operands(g, T, V, D, dtype, gpu_device)
    t[torch.randperm(T, generator=g)[:T // 4].to(gpu_device)] = -100
    up = torch.rand(T, generator=g).to(gpu_device) if reduction == "none" else torch.tensor(1.5, device=gpu_device)
    loss = linear_cross_entropy(h, w, t, reduction=reduction, logit_scale=scale)
    _check(loss, h, w, up, _reference(h, w, t[:, None], None, -100, scale, 1.0, reduction, up))
    index, z = torch.randint(0, V, (T, K), generator=g).to(gpu_device), 3 * torch.randn(T, K, generator=g).to(gpu_device)
    index[::3, : (K + 1) // 2] = -100
    loss = linear_distillation(h, w, index, z, temperature=0.75, reduction=reduction, logit_scale=scale)
    _check(loss, h, w, up, _reference(h, w, index, z, -100, scale, 0.75, reduction, up))


@pytest.mark.parametrize("T", [3, 64, 300])
def test_expanded_operands(gpu_device, T):
    # rows that are one row in memory, and an incoming gradient that is one value
    g = _gen(T)
    row = torch.randn(1, 96, generator=g).to(gpu_device, torch.bfloat16).requires_grad_(True)
    w = torch.randn(500, 96, generator=g).to(gpu_device, torch.bfloat16).requires_grad_(True)
    t = torch.randint(0, 500, (T,), generator=g).to(gpu_device)
    for reduction in ("mean", "none"):
        got = torch.autograd.grad(linear_cross_entropy(row.expand(T, 96), w, t, reduction=reduction).sum(), [row, w])
        want = torch.autograd.grad(linear_cross_entropy(row.repeat(T, 1), w, t, reduction=reduction).sum(), [row, w])
        assert torch.equal(got[1], want[1])
        torch.testing.assert_close(got[0], want[0])
    dw, = torch.autograd.grad(embedding(t, w, 2.0).sum(), [w])
    count = torch.bincount(t, minlength=500).float()[:, None]
    assert torch.equal(dw, (2 * count).to(torch.bfloat16).expand(500, 96))


@pytest.mark.parametrize("T,V,D,K,dtype", [(24000, 46000, 64, 3, torch.bfloat16), (8200, 45000, 96, 2, torch.float32),
                                           (70, 600, 16384, 20, torch.float32), (9, 300, 16384, 20, torch.bfloat16),
                                           (2100, 9000, 640, 1, torch.bfloat16), (5, 1100000, 8, 6, torch.float32),
                                           (40, 2000, 333, 6, torch.float32), (17, 5001, 130, 2, torch.float32)])
def test_several_pieces_wide_rows_and_split_products(gpu_device, T, V, D, K, dtype):
    # the backward in pieces of the vocabulary (the first two), the widest rows, tiles cut along K beside whole ones
    g = _gen(T)
    h, w, t = _operands(g, T, V, D, dtype, gpu_device)
    t[::7] = -100
    up = torch.tensor(3.0, device=gpu_device)
    want = _reference(h, w, t[:, None], None, -100, 1.0, 1.0, "mean", up)
    _check(linear_cross_entropy(h, w, t), h, w, up, want)
    ups = torch.rand(T, generator=g).to(gpu_device)
    want = _reference(h, w, t[:, None], None, -100, 1.0, 1.0, "none", ups)
    _check(linear_cross_entropy(h, w, t, reduction="none"), h, w, ups, want)
    del want
    index = torch.randint(0, V, (T, K), generator=g).to(gpu_device)
    index[::5] = -100
    z = torch.randn(T, K, generator=g).to(gpu_device)
    want = _reference(h, w, index, z, -100, 1.0, 2.0, "sum", up)
    _check(linear_distillation(h, w, index, z, temperature=2.0, reduction="sum"), h, w, up, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K", [(3, 8), (32, 8), (7, 64), (64, 64)])
def test_lists_of_few_rows_in_a_large_vocabulary(gpu_device, T, K, dtype):
    # stored logits of few rows: 1025 tiles of the vocabulary, more than 256 rows of them would fit their bound
    g = _gen(T + K)
    V, D = 262208, 48
    h, w, _ = _operands(g, T, V, D, dtype, gpu_device, pull=False)
    index = torch.randint(0, V, (T, K), generator=g).to(gpu_device)
    index[0, :2] = torch.tensor([V - 1, 0])
    z = 3 * torch.randn(T, K, generator=g).to(gpu_device)
    up = torch.rand(T, generator=g).to(gpu_device)
    want = _reference(h, w, index, z, -100, 1.0, 2.0, "none", up)
    _check(linear_distillation(h, w, index, z, temperature=2.0, reduction="none"), h, w, up, want)
    with torch.no_grad():
        only = linear_distillation(h, w, index, z, temperature=2.0, reduction="none")
    _within(only, *want[0], "loss without gradients")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("far", [60.0, 90.0, 400.0])
def test_rows_far_from_their_targets(gpu_device, far, dtype):
    # targets (and all listed tokens) whose logits lie far below the others': the exponentials relative to them
    # leave the range that stands for probabilities, in one row (90: beyond 2^100; 400: beyond fp32)
    g = _gen(int(far))
    T, V, D = 200, 700, 64
    h, w, t = _operands(g, T, V, D, torch.float32, gpu_device, pull=False)
    with torch.no_grad():
        h[17] = -far * w[t[17]] / w[t[17]].square().sum()
    h, w = (x.detach().to(dtype).requires_grad_(True) for x in (h, w))
    up = torch.tensor(1.0, device=gpu_device)
    for reduction in ("mean", "sum"):
        loss = linear_cross_entropy(h, w, t, reduction=reduction)
        _check(loss, h, w, up, _reference(h, w, t[:, None], None, -100, 1.0, 1.0, reduction, up))
    index = t[:, None].repeat(1, 2)
    z = torch.randn(T, 2, generator=g).to(gpu_device)
    loss = linear_distillation(h, w, index, z)
    _check(loss, h, w, up, _reference(h, w, index, z, -100, 1.0, 1.0, "mean", up))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nats", [27.0, 41.0, 45.0, 68.0])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("hidden,scale", [(-12, -24), (-26, 0)])
def test_rows_of_high_loss_with_small_factors(gpu_device, hidden, scale, nats, reduction, dtype):
    # one row of a high loss, small hidden states (2^hidden) and a small factor of the loss (2^scale) against a large weight: what
    # d_weight's product takes of the row must not end among the subnormal numbers (at 68 nats the row's factor is 2^-98), and
    # d_hidden's stays in range
    g = _gen(int(nats))
    T, V, D = 100, 700, 64
    h, w, t = _operands(g, T, V, D, torch.float32, gpu_device, pull=False)
    t[t == t[17]] = (t[17] + 1) % V
    t[17] = (t[17] - 1) % V
    h, w, scale = h.detach() * 2.0 ** hidden, w.detach() * 2.0 ** (-hidden - scale), 2.0 ** scale
    away = -w[t[17]].double() * (scale / w[t[17]].double().square().sum()) / scale ** 2
    least, most = 0.0, nats
    for _ in range(50):  # the multiple of it that has this loss
        far = (least + most) / 2
        s = w.double() @ (far * away) * scale
        least, most = (far, most) if float(torch.logsumexp(s, 0) - s[t[17]]) < nats else (least, far)
    h[17] = (far * away).float()
    h, w = (x.to(dtype).requires_grad_(True) for x in (h, w))
    up = torch.tensor(1.0, device=gpu_device)
    loss = linear_cross_entropy(h, w, t, reduction=reduction, logit_scale=scale)
    _check(loss, h, w, up, _reference(h, w, t[:, None], None, -100, scale, 1.0, reduction, up))
    index = t[:, None].repeat(1, 2)
    z = torch.randn(T, 2, generator=g).to(gpu_device)
    loss = linear_distillation(h, w, index, z, logit_scale=scale, reduction=reduction)
    _check(loss, h, w, up, _reference(h, w, index, z, -100, scale, 1.0, reduction, up))


@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_rows_of_very_different_scales(gpu_device, reduction):
    # fp32 logits in range, though the hidden states' scale times the products of the scaled rows is not
    g = _gen(8)
    T, V, D, scale = 100, 700, 64, 2.0 ** -72
    h, w, t = _operands(g, T, V, D, torch.float32, gpu_device, pull=False)
    h, w = ((x.detach() * f).requires_grad_(True) for x, f in ((h, 2.0 ** 112), (w, 2.0 ** -40)))
    up = torch.rand(T, generator=g).to(gpu_device) if reduction == "none" else torch.tensor(1.0, device=gpu_device)
    loss = linear_cross_entropy(h, w, t, reduction=reduction, logit_scale=scale)
    _check(loss, h, w, up, _reference(h, w, t[:, None], None, -100, scale, 1.0, reduction, up))


def test_infinite_operands(gpu_device):
    # a vocabulary row of -infinity (a token that is never taken) against positive hidden states: torch's results
    # from bf16 operands; NaN from fp32 operands, whose parts (infinity less infinity) are no numbers
    g = _gen(4)
    T, V, D = 100, 300, 64
    h = torch.rand(T, D, generator=g).to(gpu_device)
    w = torch.randn(V, D, generator=g).to(gpu_device)
    w[7] = -math.inf
    t = torch.randint(8, V, (T,), generator=g).to(gpu_device)
    for rows in (slice(None), slice(0, 50)):  # (up to 64 rows run on fp32 products)
        got = linear_cross_entropy(h[rows], w, t[rows], reduction="none")
        assert bool(got.isnan().all()) or (rows.stop == 50 and bool(got.isfinite().all()))
    hb, wb = h.bfloat16() + 0.25, w.bfloat16()
    for reduction in ("none", "mean"):
        got = linear_cross_entropy(hb.requires_grad_(True), wb, t, reduction=reduction)
        want = torch.nn.functional.cross_entropy(hb.detach().double() @ wb.double().T, t, reduction=reduction)
        torch.testing.assert_close(got.detach().double(), want, rtol=0, atol=(D + 100) * U * 128)
    t[3] = 7
    assert float(linear_cross_entropy(hb, wb, t, reduction="none")[3].detach()) == math.inf
    assert float(linear_cross_entropy(hb, wb, t).detach()) == math.inf


@pytest.mark.parametrize("T", [1, 20, 50, 64])
def test_infinite_rows_of_the_vocabulary_in_fp32(gpu_device, T):
    # up to 64 rows run on fp32 products, so that a row of -infinity against positive hidden states is a token that is never
    # taken: the losses of the vocabulary without it (a dot product of 64 terms below 1 x 4, twice, and the sums behind it)
    g = _gen(T)
    V, D = 300, 64
    h = (0.01 + 0.9 * torch.rand(T, D, generator=g)).to(gpu_device)
    w = torch.randn(V, D, generator=g).clamp(-4, 4).to(gpu_device)
    w[7] = -math.inf
    t = torch.randint(8, V, (T,), generator=g).to(gpu_device)
    rest = torch.cat([w[:7], w[8:]]).double()
    s = h.double() @ rest.T
    size = (h.double() @ rest.abs().T).amax(1)
    want = torch.logsumexp(s, 1) - s.gather(1, t[:, None] - 1)[:, 0]
    _within(linear_cross_entropy(h, w, t, reduction="none"), want,
            (4 * (6 * D + 16) * size + 64 + 4 * (V / 128 + 8)) * U + 8 * U * (want.abs() + size), "loss")
    index = torch.stack([t, t.roll(1)], 1)
    q = torch.softmax(torch.zeros(T, 2, device=gpu_device, dtype=torch.float64), 1)
    log_p = s - torch.logsumexp(s, 1, keepdim=True)
    want = (q * (q.log() - log_p.gather(1, index - 1))).sum(1)
    _within(linear_distillation(h, w, index, torch.zeros(T, 2, device=gpu_device), reduction="none"), want,
            (4 * (6 * D + 16) * size + 128 + 4 * (V / 128 + 8)) * U + 16 * U * (want.abs() + size), "distillation")


@pytest.mark.parametrize("T", [40, 300])
def test_backward_passes_of_a_graph_that_is_kept(gpu_device, T):
    # gradients formed in the forward are handed out scaled; a second pass gets its own
    g = _gen(T)
    h, w, t = _operands(g, T, 500, 96, torch.bfloat16, gpu_device)
    one = torch.autograd.grad(linear_cross_entropy(h, w, t), [h, w])
    loss = linear_cross_entropy(h, w, t)
    first = torch.autograd.grad(loss, [h, w], torch.tensor(0.5, device=gpu_device), retain_graph=True)
    second = torch.autograd.grad(loss, [h, w], torch.tensor(-2.0, device=gpu_device), retain_graph=True)
    third = torch.autograd.grad(loss, [h, w])
    for a, b, c, d in zip(one, first, second, third):  # (powers of two: exact)
        assert torch.equal(b, 0.5 * a) and torch.equal(c, -2 * a) and torch.equal(d, a)
        assert len({x.data_ptr() for x in (b, c, d)}) == 3
    (linear_cross_entropy(h, w, t) * 4).backward()
    (linear_cross_entropy(h, w, t) * 4).backward()
    assert torch.equal(h.grad, 8 * one[0]) and torch.equal(w.grad, 8 * one[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation_lists_with_repeats_infinities_and_lowest_values(gpu_device, dtype):
    g = _gen(5)
    T, V, D, K = 40, 500, 128, 12
    h, w, _ = _operands(g, T, V, D, dtype, gpu_device)
    index, z = _lists(g, T, V, K, gpu_device, repeat=True)
    lowest = torch.finfo(torch.float32).min
    z[1] = lowest                   # equal, so an even distribution
    z[2, 3:] = lowest               # next to ordinary ones: nothing
    z[3, :5] = -math.inf            # none
    z[4] = -math.inf                # a row without entries
    index[5, 1:] = -100
    index[6] = -100
    z[7, 0], index[7, 0] = math.nan, -100  # a value that is not there
    up = torch.rand(T, generator=g).to(gpu_device)
    clean = torch.where(index == -100, 0.0, z)
    loss = linear_distillation(h, w, index, z, reduction="none")
    assert float(loss[4].detach()) == 0 and float(loss[6].detach()) == 0
    gh, _ = _check(loss, h, w, up, _reference(h, w, index, clean, -100, 1.0, 1.0, "none", up))
    assert not gh[4].any() and not gh[6].any()


@pytest.mark.parametrize("T", [50, 300])
def test_what_is_in_rows_without_targets_stays_out(gpu_device, T):
    # NaN and infinities in hidden states whose target is ignored change nothing
    g = _gen(T)
    h, w, t = _operands(g, T, 600, 96, torch.bfloat16, gpu_device)
    drop = torch.rand(T, generator=g).to(gpu_device) < 0.5
    t[drop] = -100
    want = torch.autograd.grad(linear_cross_entropy(h, w, t), [h, w])
    bad = h.detach().clone()
    bad[drop] = math.nan
    bad[int(drop.nonzero()[0])] = math.inf
    bad.requires_grad_(True)
    loss = linear_cross_entropy(bad, w, t)
    got = torch.autograd.grad(loss, [bad, w])
    assert torch.equal(loss, linear_cross_entropy(h, w, t))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not got[0][drop].any()


@pytest.mark.parametrize("T", [3, 100])
def test_no_targets_at_all_and_targets_outside_the_vocabulary(gpu_device, T):
    g = _gen(T)
    h, w, t = _operands(g, T, 300, 64, torch.float32, gpu_device)
    none = torch.full_like(t, -1)
    for reduction, want in (("mean", math.nan), ("sum", 0.0)):
        loss = linear_cross_entropy(h, w, none, ignore_index=-1, reduction=reduction)
        gh, gw = torch.autograd.grad(loss, [h, w])
        assert torch.equal(loss.detach().cpu(), torch.tensor(want)) or (math.isnan(want) and bool(loss.isnan()))
        assert not gh.any() and not gw.any()
    t[1], t[2] = 300, -100
    loss = linear_cross_entropy(h, w, t, reduction="none")
    loss = loss.detach()
    assert bool(loss[1].isnan()) and float(loss[2]) == 0 and not bool(loss[0].isnan())
    t[0] = -7
    assert int(linear_cross_entropy(h, w, t, reduction="none").isnan().sum()) == 2
    assert bool(linear_cross_entropy(h, w, t).isnan())
    lists = t[:, None].repeat(1, 3)
    loss = linear_distillation(h, w, lists, torch.zeros(T, 3, device=gpu_device), reduction="none")
    assert loss.isnan().nonzero().flatten().tolist() == [0, 1]


def test_empty_batch(gpu_device):
    w = torch.randn(100, 64, device=gpu_device, requires_grad=True)
    h = torch.randn(0, 64, device=gpu_device, requires_grad=True)
    t = torch.empty(0, dtype=torch.long, device=gpu_device)
    assert linear_cross_entropy(h, w, t, reduction="none").shape == (0,)
    assert bool(linear_cross_entropy(h, w, t).isnan())
    gh, gw = torch.autograd.grad(linear_cross_entropy(h, w, t, reduction="sum"), [h, w])
    assert gh.shape == (0, 64) and not gw.any()


@pytest.mark.parametrize("K", [1, 2, 30])
def test_empty_batch_of_lists(gpu_device, K):
    w = torch.randn(100, 64, device=gpu_device, requires_grad=True)
    h = torch.randn(2, 0, 64, device=gpu_device, requires_grad=True)
    index = torch.empty(2, 0, K, dtype=torch.long, device=gpu_device)
    z = torch.empty(2, 0, K, device=gpu_device)
    for tau in (1.0, 2.0):
        assert linear_distillation(h, w, index, z, temperature=tau, reduction="none").shape == (2, 0)
        assert bool(linear_distillation(h, w, index, z, temperature=tau).isnan())
        loss = linear_distillation(h, w, index, z, temperature=tau, reduction="sum")
        gh, gw = torch.autograd.grad(loss, [h, w])
        assert float(loss.detach()) == 0 and gh.shape == (2, 0, 64) and not gw.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D", [(48, 192), (200, 192), (200, 101)])
def test_strided_operands_leading_shapes_and_frozen_parts(gpu_device, T, D, dtype):
    # rows inside wider ones at odd addresses, [B, S, D] hidden states, a gradient for one operand only
    g = _gen(T + D)
    V = 700
    h, w, t = _operands(g, T, V, D, dtype, gpu_device)
    wide_h = torch.randn(T, D + 9, generator=g).to(gpu_device, dtype)
    wide_h[:, 5:5 + D] = h.detach()
    wide_w = torch.randn(V, D + 7, generator=g).to(gpu_device, dtype)
    wide_w[:, 3:3 + D] = w.detach()
    hs, ws = wide_h[:, 5:5 + D].requires_grad_(True), wide_w[:, 3:3 + D].requires_grad_(True)
    up = torch.tensor(1.0, device=gpu_device)
    want = _reference(h, w, t[:, None], None, -100, 1.0, 1.0, "mean", up)
    grads = _check(linear_cross_entropy(hs, ws, t), hs, ws, up, want)
    shaped = linear_cross_entropy(hs.view(4, -1, D) if hs.is_contiguous() else hs.unflatten(0, (4, -1)), ws,
                                  t.view(4, -1), reduction="none")
    assert shaped.shape == (4, T // 4)
    only, = torch.autograd.grad(linear_cross_entropy(hs, ws.detach(), t), [hs])
    assert torch.equal(only, grads[0])
    only, = torch.autograd.grad(linear_cross_entropy(hs.detach(), ws, t), [ws])
    assert torch.equal(only, grads[1])
    # a transposed weight: columns adjacent
    turned = w.detach().t().contiguous().t().requires_grad_(True)
    gt = torch.autograd.grad(linear_cross_entropy(h, turned, t), [turned])[0]
    _within(gt, want[2][0], want[2][1], "d_weight of a transposed weight")


@pytest.mark.parametrize("T", [40, 260])
def test_autocast(gpu_device, T):
    # the trainer's setting: fp32 parameters, bf16 products; gradients in each operand's dtype
    g = _gen(T)
    h, w, t = _operands(g, T, 900, 160, torch.float32, gpu_device)
    hb, wb = (x.detach().bfloat16().requires_grad_(True) for x in (h, w))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = linear_cross_entropy(h, w, t)
        mixed = linear_cross_entropy(hb, w, t)
    want = linear_cross_entropy(hb, wb, t)
    assert torch.equal(loss, want) and torch.equal(mixed, want)
    gh, gw = torch.autograd.grad(loss, [h, w])
    bh, bw = torch.autograd.grad(want, [hb, wb])
    assert gh.dtype == gw.dtype == torch.float32
    assert torch.equal(gh.bfloat16(), bh) and torch.equal(gw.bfloat16(), bw)
    mh, mw = torch.autograd.grad(mixed, [hb, w])
    assert mh.dtype == torch.bfloat16 and torch.equal(mh, bh) and torch.equal(mw, gw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradients_against_differences(gpu_device, dtype):
    # the loss's own differences along random directions: a step s changes it by s <grad, dir> up to s^2 and
    # what fp32 sums of it are off by
    g = _gen(3)
    h, w, t = _operands(g, 30, 200, 64, torch.float32, gpu_device)
    index, z = _lists(g, 30, 200, 6, gpu_device)
    for call in (lambda a, b: linear_cross_entropy(a, b, t, reduction="sum"),
                 lambda a, b: linear_distillation(a, b, index, z, temperature=2.0, reduction="sum")):
        if dtype == torch.bfloat16:
            continue  # bf16 operands cannot take a small step; the products are the fp32 path's
        gh, gw = torch.autograd.grad(call(h, w), [h, w])
        for x, grad, place in ((h, gh, 0), (w, gw, 1)):
            d = torch.randn(x.shape, generator=g).to(gpu_device)
            s = 2.0 ** -8 / float(d.norm())
            args = [h.detach(), w.detach()]
            args[place] = x.detach() + s * d
            up = float(call(*args).double())
            args[place] = x.detach() - s * d
            down = float(call(*args).double())
            slope = (up - down) / (2 * s)
            # third-order term of 30 rows whose logits move by s |d_t| |w_v| (at most 2^-8 * 16 here), and fp32 sums
            tol = 30 * (2.0 ** -8 * 16) ** 3 / s + abs(up) * 64 * U / s
            assert abs(slope - float((grad.double() * d.double()).sum())) <= tol


def test_streams_and_two_calls_at_once(gpu_device):
    g = _gen(11)
    cases = []
    for T, V, D in ((300, 2000, 128), (40, 3000, 256)):
        h, w, t = _operands(g, T, V, D, torch.bfloat16, gpu_device)
        cases.append((h, w, t, *torch.autograd.grad(linear_cross_entropy(h, w, t), [h, w])))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = []
    for _ in range(3):
        for s, (h, w, t, _, _) in zip(streams, cases):
            with torch.cuda.stream(s):
                outs.append(torch.autograd.grad(linear_cross_entropy(h, w, t), [h, w]))
    torch.cuda.synchronize()
    for i, (gh, gw) in enumerate(outs):
        assert torch.equal(gh, cases[i % 2][3]) and torch.equal(gw, cases[i % 2][4])


@pytest.mark.parametrize("T", [20, 500])
def test_captured_and_replayed(gpu_device, T):
    # a step of embedding and loss, forward and backward, in a graph; new tokens written into its inputs
    g = _gen(T)
    V, D = 800, 128
    w = torch.randn(V, D, generator=g).to(gpu_device, torch.bfloat16).requires_grad_(True)
    ids = torch.randint(0, V, (T,), generator=g).to(gpu_device)
    t = torch.randint(0, V, (T,), generator=g).to(gpu_device)
    index, z = _lists(g, T, V, 5, gpu_device)

    def step(ids, t, index, z):
        # the weight of this step alone: no graph of an earlier step shares its leaf
        leaf = w.detach().requires_grad_(True)
        x = embedding(ids, leaf, 2.0)
        loss = linear_cross_entropy(x, leaf, t) + linear_distillation(x, leaf, index, z)
        return loss.detach(), *torch.autograd.grad(loss, [leaf])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ids, t, index, z)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(ids, t, index, z)
    for rep in range(4):
        new_ids = torch.randint(0, V, (T,), generator=g).to(gpu_device)
        new_t = torch.randint(0, V, (T,), generator=g).to(gpu_device)
        new_t[:rep * 3] = -100
        ids.copy_(new_ids)
        t.copy_(new_t)
        z.add_(0.5 * torch.randn(z.shape, generator=g).to(gpu_device))
        graph.replay()
        got = [x.clone() for x in out]
        torch.cuda.synchronize()
        want = step(ids, t, index, z)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep


@pytest.mark.parametrize("S", [30, 70])
def test_compiled(gpu_device, S):
    torch.manual_seed(0)
    w = torch.randn(300, 64, device=gpu_device, dtype=torch.bfloat16, requires_grad=True)
    ids = torch.randint(0, 300, (2, S), device=gpu_device)
    z = torch.randn(2, S, 4, device=gpu_device)
    index = torch.randint(0, 300, (2, S, 4), device=gpu_device)

    def step(ids, w):
        x = embedding(ids, w, 3.0, padding_idx=1)
        return linear_cross_entropy(x, w, ids) + linear_distillation(x, w, index, z, reduction="none").sum()

    want = torch.autograd.grad(step(ids, w), [w])[0]
    loss = torch.compile(step, fullgraph=True, backend="aot_eager")(ids, w)
    assert torch.equal(loss, step(ids, w)) and torch.equal(torch.autograd.grad(loss, [w])[0], want)


@pytest.mark.parametrize("S,reduction", [(30, "mean"), (70, "mean"), (70, "none")])
def test_compiled_with_frozen_parts(gpu_device, S, reduction):
    torch._dynamo.reset()
    g = _gen(S)
    h, w, t = _operands(g, S, 300, 64, torch.bfloat16, gpu_device)
    index, z = _lists(g, S, 300, 4, gpu_device)

    def step(h, w):
        return (linear_cross_entropy(h, w, t, reduction=reduction) +
                linear_distillation(h, w, index, z, reduction=reduction)).sum()

    for a, b in ((h, w.detach()), (h.detach(), w), (h, w)):
        leaves = [x for x in (a, b) if x.requires_grad]
        want = torch.autograd.grad(step(a, b), leaves)
        got = torch.autograd.grad(torch.compile(step, fullgraph=True, backend="aot_eager")(a, b), leaves)
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_compiled_with_a_weight_at_an_odd_address(gpu_device):
    # a weight (part of a flat buffer) whose copy would be more than gradients formed in the forward allow for: a traced
    # call, which sees no addresses, has chosen them
    torch._dynamo.reset()
    T, V, D = 65, 131072, 8256
    g = torch.Generator(device=gpu_device).manual_seed(1)
    flat = torch.empty(V * D + 8, device=gpu_device, dtype=torch.bfloat16).normal_(std=0.02, generator=g)
    w = flat[1:1 + V * D].view(V, D)
    h = torch.randn(T, D, device=gpu_device, generator=g).bfloat16().requires_grad_(True)
    t = torch.randint(0, V, (T,), device=gpu_device, generator=g)
    want = linear_cross_entropy(h, w.clone(), t)
    dh, = torch.autograd.grad(want, [h])
    loss = torch.compile(lambda h, w: linear_cross_entropy(h, w, t), fullgraph=True, backend="aot_eager")(h, w)
    assert torch.equal(loss, want) and torch.equal(torch.autograd.grad(loss, [h])[0], dh)


def test_second_derivatives_are_refused(gpu_device):
    h, w, t = _operands(_gen(0), 8, 50, 64, torch.float32, gpu_device)
    gh, = torch.autograd.grad(linear_cross_entropy(h, w, t), [h], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        gh.sum().backward()
    gw, = torch.autograd.grad(embedding(t, w).pow(2).sum(), [w], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        gw.sum().backward()


def test_wrappers_give_the_native_calls_results(gpu_device):
    # the path of per-entry-point timing
    from fusionllm_amd import _kernels as K
    g = _gen(9)
    h, w, t = _operands(g, 70, 300, 96, torch.bfloat16, gpu_device)
    index, z = _lists(g, 70, 300, 9, gpu_device)

    def step():
        loss = linear_cross_entropy(h, w, t) + linear_distillation(h, w, index, z, reduction="none").sum()
        y = embedding(t, w, 2.0)
        return loss, *torch.autograd.grad(loss + y.float().sum(), [h, w])

    want = step()
    times = {}
    K.set_timer(times)
    try:
        got = step()
    finally:
        K.set_timer(None)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert {"embedding_fwd", "embedding_bwd", "vocab_loss_fwd", "vocab_loss_bwd", "vocab_loss_fwd_grad",
            "scale"} <= set(times)


def test_as_many_rows_as_a_call_takes(gpu_device):
    # 2^24 rows: a workgroup for each of their lists is more than one side of a grid holds
    g = torch.Generator(device=gpu_device).manual_seed(6)
    T, V, D = 1 << 24, 3, 4
    h = torch.randn(T, D, device=gpu_device, generator=g).bfloat16()
    w = torch.randn(V, D, device=gpu_device, generator=g).bfloat16()
    index = torch.randint(0, V, (T, 2), device=gpu_device, generator=g, dtype=torch.int32)
    z = torch.randn(T, 2, device=gpu_device, generator=g)
    up = torch.ones(T, device=gpu_device)
    _within(linear_distillation(h, w, index, z, temperature=2.0, reduction="none"),
            *_reference(h, w, index, z, -100, 1.0, 2.0, "none", up)[0], "distillation")
    target = index[:, 0].contiguous()
    _within(linear_cross_entropy(h, w, target, reduction="none"),
            *_reference(h, w, index[:, :1], None, -100, 1.0, 1.0, "none", up)[0], "cross entropy")
    ids = target.long()
    assert torch.equal(embedding(target, w), w[ids])
    leaf = w.clone().requires_grad_(True)
    dw, = torch.autograd.grad(embedding(ids, leaf), [leaf], torch.ones_like(h))
    assert torch.equal(dw, torch.bincount(ids, minlength=V).bfloat16()[:, None].expand(V, D))  # (counts below 2^24: exact sums)


def test_long_offsets(gpu_device):
    # a weight of more than 2^31 elements (rows at offsets beyond 32 bits), few of them used
    V, D = 1 << 20, 2064
    w = torch.zeros(V, D, device=gpu_device, dtype=torch.bfloat16)
    ids = torch.tensor([0, V - 1, V - 2, V // 2, V - 1], device=gpu_device)
    rows = torch.randn(5, D, generator=_gen(1)).to(gpu_device, torch.bfloat16)
    rows[4] = rows[1]
    w[ids] = rows
    assert torch.equal(embedding(ids, w, 1.0), rows)
    w.requires_grad_(True)
    dw, = torch.autograd.grad(embedding(ids, w, 1.0), [w], rows)
    assert torch.equal(dw[V - 1], (2 * rows[1].float()).bfloat16()) and torch.equal(dw[V // 2], rows[3])
    assert int(dw.count_nonzero(dim=1).count_nonzero()) == 4
    # the other rows' logits are zero: lse and its gradients in closed form
    h = (rows * 0.05).detach().requires_grad_(True)
    loss = linear_cross_entropy(h, w, ids, reduction="none")
    s = h.detach().double() @ w.detach()[ids[:4]].double().T
    lse = torch.log(torch.exp(s).sum(1) + (V - 4))
    want = lse - s.gather(1, torch.tensor([[0], [1], [2], [3], [1]], device=gpu_device))[:, 0]
    torch.testing.assert_close(loss.detach().double(), want, rtol=0, atol=(D + V / 128 + 64) * 8 * U * 4)


def test_a_training_step_from_tokens_to_loss(gpu_device):
    # embedding -> norm, block and residual -> norm -> loss, tied weight, in this package's operators; against torch
    # operations around the same block, whose own rounding both sides share
    from fusionllm_amd import DeepSeekMoE, Embedding, configs, layer_norm, moe_residual
    cfg = configs.C2
    torch.manual_seed(2)
    emb = Embedding(1000, cfg.dim, scale=cfg.dim ** 0.5).to(gpu_device, torch.bfloat16)
    torch.nn.init.normal_(emb.weight, std=0.02)
    block = DeepSeekMoE(cfg.moe_config())
    block.load_state_dict({k: v.bfloat16() for k, v in configs.make_block(cfg, seed=1, tokens=8).state_dict().items()})
    block = block.to(device=gpu_device, dtype=torch.bfloat16)
    norm = torch.nn.RMSNorm(cfg.dim, eps=1e-6).to(gpu_device, torch.bfloat16)
    ids = torch.randint(0, 1000, (3, 100), device=gpu_device)
    target = ids.roll(-1, 1)
    target[:, -1] = -100

    x = moe_residual(emb(ids), norm, block)
    hidden = layer_norm(x)
    loss = linear_cross_entropy(hidden, emb.weight, target)
    loss.backward()
    got = emb.weight.grad.clone()
    emb.weight.grad = None

    y = torch.nn.functional.embedding(ids, emb.weight) * cfg.dim ** 0.5
    hidden2 = layer_norm(moe_residual(y.bfloat16(), norm, block))
    logits = hidden2.reshape(-1, cfg.dim).float() @ emb.weight.float().t()
    ref = torch.nn.functional.cross_entropy(logits, target.flatten())
    ref.backward()
    want = emb.weight.grad
    assert torch.equal(hidden, hidden2)
    # both losses in fp32 of the same operands; gradients of bf16 roundings at a few places (G, d_hidden, d_weight)
    assert abs(float(loss) - float(ref)) <= 2 * (cfg.dim + 64) * U * float(logits.abs().max() + 8)
    assert float((got.float() - want.float()).norm()) <= 4 * 2.0 ** -8 * float(want.float().norm())
