"""Layer norm forward and backward against the formulas in 64 bits, and through
the module, autograd, streams, graphs, torch.compile and moe_residual.

Tolerances (u = 2^-24, half of fp32's eps; the kernels compute in fp32 and round
once): a row's sums add at most 16 values per lane, 6 butterfly steps and 15
waves' sums in a chain, so they are within 40 u of sum |terms|; the few
operations after them add a few u each.  N = 64 u covers both.
  xh:  |err| <= E = N (r mean|x| + |xh|)             (mean, r, the subtraction)
  y:   |w| E + N (|xh w| + |b|), plus half a step of the result's type
  dx:  N r (|g| + mean|g| + |xh| mean|g xh|) + r (E mean|g xh| + |xh| mean(|g| E)) + N |dx|,
       plus half a step
  dw:  sum |dy| E + (chain + 2) u sum |dy xh|, db: (chain + 2) u sum |dy|, plus half a step, where
       chain is the number of additions in a column's sum (rows per wave, 4 waves, the
       partial rows in 16 waves, their 16 sums)."""
import copy

import pytest
import torch
import torch.nn as nn

import fusionllm_amd
from fusionllm_amd import LayerNorm, configs, layer_norm, moe_residual
from fusionllm_amd import _kernels as K
from tests.gpu_util import build_module

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
N = 64 * U
BF, F32 = torch.bfloat16, torch.float32
SHAPES = [(1, 768), (1, 1), (3, 1), (5, 7), (2, 8), (3, 9), (17, 63), (4, 64), (33, 100), (129, 511), (7, 512),
          (5, 513), (64, 768), (31, 1023), (16, 1024), (9, 1025), (6, 1032), (5, 2048), (3, 2055), (2, 4099),
          (3, 10240), (2, 16383), (2, 16384)]


def half(t):
    return torch.finfo(t).eps / 2


def inputs(T, dim, xd, wd, dev, seed=0, bias=True, weight=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, dim, generator=g) * (0.2 + 3 * torch.rand(T, 1, generator=g)) + 0.7).to(xd)
    w = (1 + 0.3 * torch.randn(dim, generator=g)).to(wd) if weight else None
    b = (0.5 * torch.randn(dim, generator=g)).to(wd) if bias else None
    dy = torch.randn(T, dim, generator=g)
    to = lambda t: None if t is None else t.to(dev)
    return to(x), to(w), to(b), dy.to(dev)


def truth(x, w, b, dy, eps):
    """The formulas in 64 bits and the bounds above."""
    x, dy = x.double(), dy.double()
    T, D = x.shape
    w = torch.ones(D, device=x.device).double() if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    r = 1 / (((x - mean) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * r
    y = xh * w + b
    E = N * (r * x.abs().mean(-1, keepdim=True) + xh.abs())
    g = dy * w
    m = lambda t: t.mean(-1, keepdim=True)
    dx = r * (g - m(g) - xh * m(g * xh))
    # rows per wave where there are fewer waves than rows (at least 128 workgroups of the longest
    # rows, 512 of four rows), or the fewer additions of a larger launch
    chain = T // 128 + 4 + 1024 // 16 + 16
    tol = {"y": w.abs() * E + N * ((xh * w).abs() + b.abs()),
           "dx": N * r * (g.abs() + m(g.abs()) + xh.abs() * m((g * xh).abs()))
           + r * (E * m((g * xh).abs()) + xh.abs() * m(g.abs() * E)) + N * dx.abs(),
           "dw": (dy.abs() * E).sum(0) + (chain + 2) * U * (dy * xh).abs().sum(0),
           "db": (chain + 2) * U * dy.abs().sum(0)}
    return {"y": y, "dx": dx, "dw": (dy * xh).sum(0), "db": dy.sum(0)}, tol


def check(got, want, tol, name):
    w, t = want[name], tol[name]
    err = (got.double() - w).abs()
    bound = t + (w.abs() + t) * half(got.dtype)
    assert not torch.isnan(got).any(), name
    bad = err > bound
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound).max()):.2f} x "
                           f"the bound at {int((err / bound).argmax())}")


@pytest.mark.parametrize("xd,wd", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)], ids=["bb", "bf", "ff", "fb"])
@pytest.mark.parametrize("T,dim", SHAPES)
def test_forward_and_backward_against_64_bits(gpu_device, T, dim, xd, wd):
    x, w, b, dy = inputs(T, dim, xd, wd, gpu_device, seed=T * 31 + dim)
    eps = 1e-5
    for p in (x, w, b):
        p.requires_grad_(True)
    y = layer_norm(x, w, b, eps)
    dyd = dy.to(y.dtype)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dyd)
    assert (y.dtype, dx.dtype, dw.dtype, db.dtype) == (xd, xd, wd, wd)
    want, tol = truth(x.detach(), w.detach(), b.detach(), dyd, eps)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        check(got.detach(), want, tol, name)
    # without autograd: the same values
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y)


@pytest.mark.parametrize("T,dim,xd", [(5000, 768, BF), (4097, 2048, F32), (9001, 65, BF), (66001, 40, BF),
                                      (65600, 24, F32), (3000, 2051, F32)])
def test_many_rows(gpu_device, T, dim, xd):
    # more rows than the backward's launch has waves (and, for bf16, enough for the larger launch): each adds several
    x, w, b, dy = inputs(T, dim, xd, F32, gpu_device, seed=4)
    BF = xd
    for p in (x, w, b):
        p.requires_grad_(True)
    y = layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy.to(BF))
    again = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy.to(BF))
    want, tol = truth(x.detach(), w.detach(), b.detach(), dy.to(BF), 1e-5)
    for name, got in zip(("y", "dx", "dw", "db"), (y.detach(), *grads)):
        check(got, want, tol, name)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))  # fixed order


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("dim", [5, 64, 1023])
def test_without_weight_or_bias(gpu_device, weight, bias, dim):
    x, w, b, dy = inputs(37, dim, BF, F32, gpu_device, weight=weight, bias=bias)
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = layer_norm(x, w, b, 1e-6)
    grads = dict(zip([n for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None],
                     torch.autograd.grad(y, leaves, dy.to(BF))))
    want, tol = truth(x.detach(), None if w is None else w.detach(), None if b is None else b.detach(), dy.to(BF),
                      1e-6)
    check(y.detach(), want, tol, "y")
    for name, got in grads.items():
        check(got, want, tol, name)


def test_partial_gradients(gpu_device):
    # only what is asked for is computed, with the same bits
    x, w, b, dy = inputs(50, 777, F32, F32, gpu_device)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(layer_norm(*full), full, dy)
    for pick in ((0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
        part = [t.clone().requires_grad_(i in pick) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(layer_norm(*part), [part[i] for i in pick], dy)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, pick)), pick


@pytest.mark.parametrize("dt", [BF, F32])
def test_strides_and_addresses(gpu_device, dt):
    # a slice of wider rows, from an odd element on; its neighbours are not touched; a
    # transposed and an expanded input, an expanded gradient
    T, dim = 19, 203
    base = torch.randn(T, 2 * dim + 3, device=gpu_device).to(dt)
    x = base[:, 3:3 + dim]
    _, w, b, dy = inputs(T, dim, dt, F32, gpu_device)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b), layer_norm(x.contiguous(), w, b))
        xt = torch.randn(dim, T, device=gpu_device).to(dt).t()
        assert torch.equal(layer_norm(xt, w, b), layer_norm(xt.contiguous(), w, b))
        xe = torch.randn(1, dim, device=gpu_device).to(dt).expand(T, dim)
        assert torch.equal(layer_norm(xe, w, b), layer_norm(xe.contiguous(), w, b))
        x3 = torch.randn(3, 5, 2 * dim, device=gpu_device).to(dt)[..., :dim]
        assert torch.equal(layer_norm(x3, w, b), layer_norm(x3.contiguous(), w, b))
    xs = base.clone().requires_grad_(True)
    xc = x.detach().clone().requires_grad_(True)
    layer_norm(xs[:, 3:3 + dim], w, b).backward(dy.to(dt))
    layer_norm(xc, w, b).backward(dy.to(dt))
    assert torch.equal(xs.grad[:, 3:3 + dim], xc.grad)
    assert not xs.grad[:, :3].any() and not xs.grad[:, 3 + dim:].any()
    xc.grad = None
    layer_norm(xc, w, b).sum().backward()  # dy: one value, expanded
    ref = xc.grad
    xc.grad = None
    layer_norm(xc, w, b).backward(torch.ones(T, dim, device=gpu_device, dtype=dt))
    assert torch.equal(ref, xc.grad)


def test_empty_constant_and_non_finite_rows(gpu_device):
    dim = 96
    w = torch.full((dim,), 2.0, device=gpu_device, requires_grad=True)
    b = torch.full((dim,), 0.5, device=gpu_device, requires_grad=True)
    x = torch.empty(0, dim, device=gpu_device, requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == dx.shape == (0, dim) and not dw.any() and not db.any()
    # constant rows: xh = 0 exactly (the mean of equal values is exact here), gradients finite
    x = torch.full((3, dim), 4.0, device=gpu_device, requires_grad=True)
    y = layer_norm(x, w, b)
    assert torch.equal(y, torch.full_like(y, 0.5))
    (dx,) = torch.autograd.grad(y, (x,), torch.randn(3, dim, device=gpu_device))
    assert torch.isfinite(dx).all()
    # rows with infinities or NaN give NaN rows and leave the others alone
    x = torch.randn(8, dim, device=gpu_device)
    clean = layer_norm(x, w, b)
    x[2, 5], x[4, 95], x[6, 0] = float("inf"), float("nan"), -float("inf")
    y = layer_norm(x, w, b)
    bad = torch.tensor([2, 4, 6], device=gpu_device)
    good = torch.tensor([0, 1, 3, 5, 7], device=gpu_device)
    assert torch.isnan(y[bad]).all() and torch.equal(y[good], clean[good])


def test_gradients_against_differences(gpu_device):
    # f(p) = sum(y v) for fp32 leaves: the directional derivative against a central difference of
    # the forward summed in 64 bits.  With h = 2^-6 the difference's own error is of h^2 times third
    # derivatives (all of order 1 here: 3e-4) and of rounding N / h (3e-4) relative to the norms' product.
    T, dim, h = 23, 133, 2.0 ** -6
    x, w, b, v = inputs(T, dim, F32, F32, gpu_device, seed=9)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, v)
    f = lambda *p: float((layer_norm(*p).double() * v.double()).sum())
    with torch.no_grad():
        for i in range(3):
            d = torch.randn_like(leaves[i])
            lo, hi = list(leaves), list(leaves)
            lo[i], hi[i] = leaves[i] - h * d, leaves[i] + h * d
            diff = (f(*hi) - f(*lo)) / (2 * h)
            want = float((grads[i].double() * d.double()).sum())
            scale = float(grads[i].double().norm() * d.double().norm()) + float(v.double().norm())
            assert abs(diff - want) <= 2e-3 * scale, i


def test_module_and_autocast(gpu_device):
    ln = LayerNorm(130).to(gpu_device)
    ref = nn.LayerNorm(130).to(gpu_device)
    with torch.no_grad():
        ln.weight.normal_()
        ln.bias.normal_()
    ref.load_state_dict(ln.state_dict())
    x = torch.randn(4, 6, 130, device=gpu_device)
    torch.testing.assert_close(ln(x), ref(x), rtol=1e-5, atol=1e-5)
    # several normalised dimensions
    ln2 = LayerNorm((10, 13)).to(gpu_device)
    torch.testing.assert_close(ln2(x.view(4, 6, 10, 13)), nn.functional.layer_norm(x.view(4, 6, 10, 13), (10, 13)),
                               rtol=1e-5, atol=1e-5)
    with pytest.raises(RuntimeError, match="expected an input"):
        ln(torch.randn(4, 131, device=gpu_device))
    with torch.autocast("cuda", dtype=BF):
        y = ln(x.bfloat16().requires_grad_(True))
        assert y.dtype == F32 == ref(x.bfloat16()).dtype
        y.sum().backward()
    plain = LayerNorm(130, elementwise_affine=False).to(gpu_device)
    torch.testing.assert_close(plain(x), nn.functional.layer_norm(x, (130,)), rtol=1e-5, atol=1e-5)


def test_second_derivatives_are_refused(gpu_device):
    # refused where they are asked for, not before: a graph of the backward may be built around it
    w = torch.randn(64, device=gpu_device, requires_grad=True)
    for weight in (None, w):
        x = torch.randn(3, 64, device=gpu_device, requires_grad=True)
        (want,) = torch.autograd.grad(layer_norm(x, weight).square().sum(), x)
        (g,) = torch.autograd.grad(layer_norm(x, weight).square().sum(), x, create_graph=True)
        assert torch.equal(g, want)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_side_stream_and_two_streams(gpu_device):
    x, w, b, dy = inputs(700, 768, BF, BF, gpu_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    want = (layer_norm(*leaves), *torch.autograd.grad(layer_norm(*leaves), leaves, dy.to(BF)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = layer_norm(*leaves)
            outs.append((y, *torch.autograd.grad(y, leaves, dy.to(BF))))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want))


def test_graph_replays(gpu_device):
    # forward and backward of two graphs on new inputs, with eager work between the replays
    T, dim = 300, 515
    x, w, b, dy = inputs(T, dim, BF, F32, gpu_device)
    dy = dy.to(BF)

    def step(xs, dys):
        y, mean, rstd = K.layer_norm_fwd(xs, w, b, 1e-5, BF)
        return (y, *K.layer_norm_bwd(dys, xs, mean, rstd, w, None, True, F32, F32))

    graphs = []
    for _ in range(2):
        xs, dys = x.clone(), dy.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(xs, dys)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(xs, dys)
        graphs.append((g, xs, dys, out))
    for rep in range(4):
        news = []
        for j, (g, xs, dys, out) in enumerate(graphs):
            nx, _, _, nd = inputs(T, dim, BF, F32, gpu_device, seed=100 + 10 * rep + j)
            xs.copy_(nx)
            dys.copy_(nd.to(BF))
            g.replay()
            news.append((nx, nd.to(BF)))
        torch.cuda.synchronize()
        for (g, xs, dys, out), (nx, nd) in zip(graphs, news):
            assert all(torch.equal(p, q) for p, q in zip(out, step(nx, nd))), rep


def test_compile_fullgraph(gpu_device):
    x, w, b, dy = inputs(40, 192, F32, F32, gpu_device)

    def f(x, w, b):
        return layer_norm(x * 2, w, b).tanh()

    eager = [t.clone().requires_grad_(True) for t in (x, w, b)]
    traced = [t.clone().requires_grad_(True) for t in (x, w, b)]
    ye = f(*eager)
    yc = torch.compile(f, fullgraph=True, backend="aot_eager")(*traced)
    torch.testing.assert_close(yc, ye)
    ye.backward(dy)
    yc.backward(dy)
    for p, q in zip(traced, eager):
        torch.testing.assert_close(p.grad, q.grad)
    # a norm without bias, whose weight gets its gradient through the operator
    g = torch.compile(lambda x, w: layer_norm(x, w), fullgraph=True, backend="aot_eager")
    for p in traced[:2]:
        p.grad = None
    g(*traced[:2]).backward(dy)
    want = torch.autograd.grad(layer_norm(*eager[:2]), eager[:2], dy)
    assert all(torch.equal(p.grad, q) for p, q in zip(traced, want))


@pytest.mark.parametrize("T", [1, 7, 300])
@pytest.mark.parametrize("mode", ["bf16", "autocast"])
def test_moe_residual_with_layer_norm(gpu_device, T, mode):
    """x + moe(norm(x)) fused against the same pieces one after the other: the norm, the
    block (whose input gradient comes back rounded to its input's type) and the add."""
    cfg = configs.BlockConfig("t", T, dim=128, inter=192, n_experts=4, topk=2)
    data = configs.make_block(cfg, seed=3)
    dt = BF if mode == "bf16" else F32
    moe = build_module(cfg, data, gpu_device, dt)
    norm = LayerNorm(128).to(gpu_device, dt)
    with torch.no_grad():
        norm.weight.add_(0.2 * torch.randn_like(norm.weight))
        norm.bias.add_(0.2 * torch.randn_like(norm.bias))
    moe2, norm2 = copy.deepcopy(moe), copy.deepcopy(norm)
    x = data.x.to(gpu_device, dt).view(1, T, 128).requires_grad_(True)
    x2 = x.detach().clone().requires_grad_(True)
    dy = data.dy.to(gpu_device, dt).view(1, T, 128)
    ctx = lambda: torch.autocast("cuda", dtype=BF, enabled=mode == "autocast")
    with ctx():
        y = moe_residual(x, norm, moe)
        y2 = x2 + moe2(norm2(x2))
        with torch.no_grad():
            y3 = moe_residual(x, norm, moe)
    assert y.dtype == y2.dtype == dt and torch.equal(y, y3)
    assert torch.equal(moe._last_indices, moe2._last_indices)
    y.backward(dy)
    y2.backward(dy)
    # pieces round the block's output and its input's gradient to bf16 (2^-8 of values of about the
    # size of the terms) where the fused form keeps fp32; the sums of the norm's gradients add those
    tol = 2.0 ** -7
    close = lambda a, b: (a.double() - b.double()).norm() <= tol * b.double().norm()
    assert close(y, y2) and close(x.grad, x2.grad)
    assert close(norm.weight.grad, norm2.weight.grad) and close(norm.bias.grad, norm2.bias.grad)
    for (name, p), q in zip(moe.named_parameters(), moe2.parameters()):
        assert (p.grad is None) == (q.grad is None), name
        if p.grad is not None:
            assert torch.equal(p.grad, q.grad), name  # the same rows through the same kernels


def test_moe_residual_of_a_bf16_input_under_autocast_is_the_plain_expression(gpu_device):
    cfg = configs.BlockConfig("t", 9, dim=128, inter=192, n_experts=4, topk=2)
    data = configs.make_block(cfg, seed=3)
    moe = build_module(cfg, data, gpu_device, F32)
    norm = LayerNorm(128).to(gpu_device)
    x = data.x.to(gpu_device, BF)
    with torch.autocast("cuda", dtype=BF), torch.no_grad():
        y = moe_residual(x, norm, moe)
        want = x + moe(norm(x))
    assert y.dtype == want.dtype == F32 and torch.equal(y, want)


def test_timed_wrappers_give_the_same_bits(gpu_device):
    # with per-entry-point timing on, the Python form around the same entry points runs
    x, w, b, dy = inputs(130, 777, BF, F32, gpu_device)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def run():
        y = layer_norm(*leaves)
        with torch.no_grad():
            z = layer_norm(*leaves)
        return (y.detach(), z, *torch.autograd.grad(y, leaves, dy.to(BF)))

    want = run()
    store = {}
    K.set_timer(store)
    try:
        got = run()
    finally:
        K.set_timer(None)
    assert set(store) == {"layer_norm_fwd", "layer_norm_bwd"} and len(store["layer_norm_fwd"]) == 2
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_autograd_under_graph_capture(gpu_device):
    # forward and backward through autograd, captured with leaves of its own and replayed on new inputs
    T, dim = 70, 300
    x, w, b, dy = inputs(T, dim, BF, F32, gpu_device)
    dy = dy.to(BF)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]

    def step():
        y = layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for rep in range(3):
        nx, _, _, nd = inputs(T, dim, BF, F32, gpu_device, seed=50 + rep)
        with torch.no_grad():
            leaves[0].copy_(nx)
        dy.copy_(nd.to(BF))
        g.replay()
        torch.cuda.synchronize()
        y, mean, rstd = K.layer_norm_fwd(nx, w, b, 1e-5, BF)
        want = (y, *K.layer_norm_bwd(nd.to(BF), nx, mean, rstd, w, None, True, F32, F32))
        assert all(torch.equal(p, q) for p, q in zip(out, want)), rep


def test_input_changed_before_the_backward_is_an_error(gpu_device):
    x = torch.randn(4, 64, device=gpu_device, requires_grad=True)
    y = layer_norm(x * 1.0, torch.ones(64, device=gpu_device))
    h = x * 1.0
    z = layer_norm(h, torch.ones(64, device=gpu_device))
    h.add_(1.0)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()


def test_wrappers_refuse_what_the_kernels_do_not_take(gpu_device):
    x = torch.randn(8, 64, device=gpu_device)
    w = torch.ones(64, device=gpu_device)
    m = torch.zeros(8, device=gpu_device)
    with pytest.raises(RuntimeError, match="overlap"):
        K.layer_norm_fwd(x[:1].expand(8, 64), w, None, 1e-5, F32)
    with pytest.raises(RuntimeError, match="adjacent"):
        K.layer_norm_fwd(torch.randn(64, 8, device=gpu_device).t(), w, None, 1e-5, F32)
    with pytest.raises(RuntimeError, match="one dtype"):
        K.layer_norm_fwd(x, w, w.bfloat16(), 1e-5, F32)
    with pytest.raises(RuntimeError, match="hold 64"):
        K.layer_norm_fwd(x, w[:32], None, 1e-5, F32)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        K.layer_norm_fwd(x, w, None, 1e-5, torch.float16)
    with pytest.raises(RuntimeError, match="dy must be"):
        K.layer_norm_bwd(x[:4], x, m, m, w)
    with pytest.raises(RuntimeError, match="mean must hold"):
        K.layer_norm_bwd(x, x, m[:4], m, w)
    with pytest.raises(RuntimeError, match="d_residual"):
        K.layer_norm_bwd(x, x, m, m, w, x[:4])
    with pytest.raises(RuntimeError, match="one dtype"):
        K.layer_norm_bwd(x, x, m, m, w, None, True, BF, None)


def test_moe_residual_with_layer_norm_compiles(gpu_device):
    # traced: the plain expression around the block's and the norm's operators
    cfg = configs.BlockConfig("t", 40, dim=128, inter=192, n_experts=4, topk=2)
    data = configs.make_block(cfg, seed=3)
    moe = build_module(cfg, data, gpu_device, BF)
    norm = LayerNorm(128).to(gpu_device, BF)
    x = data.x.to(gpu_device, BF).requires_grad_(True)
    x2 = x.detach().clone().requires_grad_(True)
    y = torch.compile(lambda t: moe_residual(t, norm, moe), fullgraph=True, backend="aot_eager")(x)
    want = x2 + moe(norm(x2))
    assert torch.equal(y, want)
    y.backward(data.dy.to(gpu_device, BF))
    gw = norm.weight.grad.clone()
    norm.zero_grad()
    want.backward(data.dy.to(gpu_device, BF))
    assert torch.equal(x.grad, x2.grad) and torch.equal(gw, norm.weight.grad)


def test_more_rows_than_one_launch_and_32_bit_offsets_take(gpu_device):
    # 2^26 + 3 rows: more than 2^32 threads with a wave per row, and more than 2^31 elements.  y and dx in
    # rows around the places where a launch ends and an offset passes 31 bits; dw and db over all rows, with
    # a chain of T / 4096 rows per wave (1024 workgroups of four), 4 waves, 64 partial rows and 16 sums.
    T, dim = 2 ** 26 + 3, 40
    gen = torch.Generator(gpu_device).manual_seed(9)
    x = torch.randn(T, dim, dtype=BF, device=gpu_device, generator=gen)
    dy = torch.randn(T, dim, dtype=BF, device=gpu_device, generator=gen)
    w = (1 + 0.3 * torch.randn(dim, device=gpu_device, generator=gen))
    b = torch.randn(dim, device=gpu_device, generator=gen)
    for p in (x, w, b):
        p.requires_grad_(True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    x, y, w, b = x.detach(), y.detach(), w.detach(), b.detach()
    for mid in (0, 2 ** 25, 2 ** 31 // dim, T):
        rows = slice(max(mid - 600, 0), mid + 600)
        want, tol = truth(x[rows], w, b, dy[rows], 1e-5)
        check(y[rows], want, tol, "y")
        check(dx[rows], want, tol, "dx")
    total, bound = {"dw": 0.0, "db": 0.0}, {"dw": 0.0, "db": 0.0}
    chain = T // 4096 + 1 + 4 + 64 + 16
    for t in range(0, T, 2 ** 22):
        xs, d = x[t:t + 2 ** 22].double(), dy[t:t + 2 ** 22].double()
        xs -= xs.mean(-1, keepdim=True)
        r = 1 / (xs.square().mean(-1, keepdim=True) + 1e-5).sqrt()
        ax = x[t:t + 2 ** 22].double().abs().mean(-1, keepdim=True)
        xs *= r
        total["dw"] += (d * xs).sum(0)
        total["db"] += d.sum(0)
        bound["dw"] += (d.abs() * N * (r * ax + xs.abs())).sum(0) + (chain + 2) * U * (d * xs).abs().sum(0)
        bound["db"] += (chain + 2) * U * d.abs().sum(0)
    check(dw, total, bound, "dw")
    check(db, total, bound, "db")


def test_second_derivatives_of_the_fused_form_are_refused(gpu_device):
    # not left out in silence, also where another term of the sum has one
    cfg = configs.BlockConfig("t", 9, dim=128, inter=192, n_experts=4, topk=2)
    data = configs.make_block(cfg, seed=3)
    moe = build_module(cfg, data, gpu_device, BF)
    norm = LayerNorm(128).to(gpu_device, BF)
    x = data.x.to(gpu_device, BF).requires_grad_(True)
    (want,) = torch.autograd.grad(moe_residual(x, norm, moe).float().square().sum(), x)
    (g,) = torch.autograd.grad(moe_residual(x, norm, moe).float().square().sum(), x, create_graph=True)
    assert torch.equal(g, want)
    with pytest.raises(RuntimeError):
        (g.float().sum() + x.float().square().sum()).backward()


def test_moe_residual_of_fp32_outside_autocast(gpu_device):
    cfg = configs.BlockConfig("t", 33, dim=128, inter=192, n_experts=4, topk=2)
    data = configs.make_block(cfg, seed=3)
    moe = build_module(cfg, data, gpu_device, F32)
    norm = LayerNorm(128).to(gpu_device)
    moe2, norm2 = copy.deepcopy(moe), copy.deepcopy(norm)
    x = data.x.to(gpu_device, F32).requires_grad_(True)
    x2 = x.detach().clone().requires_grad_(True)
    dy = data.dy.to(gpu_device, F32)
    y, y2 = moe_residual(x, norm, moe), x2 + moe2(norm2(x2))
    y.backward(dy)
    y2.backward(dy)
    assert y.dtype == F32 and torch.equal(moe._last_indices, moe2._last_indices)
    # the block takes bf16 copies of the norm's output either way; its fp32 results are added in fp32
    tol = 2.0 ** -7
    for got, want in ((y, y2), (x.grad, x2.grad), (norm.weight.grad, norm2.weight.grad),
                      (norm.bias.grad, norm2.bias.grad)):
        assert float((got.double() - want.double()).norm()) <= tol * float(want.double().norm())


@pytest.mark.parametrize("kw", [dict(bias=False), dict(elementwise_affine=False)], ids=["no_bias", "no_vectors"])
@pytest.mark.parametrize("mode", ["bf16", "autocast"])
def test_moe_residual_with_fewer_vectors(gpu_device, kw, mode):
    # bounds as in test_moe_residual_with_layer_norm
    cfg = configs.BlockConfig("t", 61, dim=128, inter=192, n_experts=4, topk=2)
    data = configs.make_block(cfg, seed=5)
    dt = BF if mode == "bf16" else F32
    moe = build_module(cfg, data, gpu_device, dt)
    norm = LayerNorm(128, **kw).to(gpu_device, dt)
    with torch.no_grad():
        for p in norm.parameters():
            p.add_(0.2 * torch.randn_like(p))
    moe2, norm2 = copy.deepcopy(moe), copy.deepcopy(norm)
    x = data.x.to(gpu_device, dt).requires_grad_(True)
    x2 = x.detach().clone().requires_grad_(True)
    dy = data.dy.to(gpu_device, dt)
    with torch.autocast("cuda", dtype=BF, enabled=mode == "autocast"):
        y, y2 = moe_residual(x, norm, moe), x2 + moe2(norm2(x2))
        with torch.no_grad():
            assert torch.equal(moe_residual(x, norm, moe), y)
    y.backward(dy)
    y2.backward(dy)
    assert y.dtype == dt and torch.equal(moe._last_indices, moe2._last_indices)
    pairs = [(y, y2), (x.grad, x2.grad), *((p.grad, q.grad) for p, q in zip(norm.parameters(), norm2.parameters()))]
    assert len(pairs) == 2 + len(list(norm.parameters()))
    for got, want in pairs:
        assert float((got.detach().double() - want.detach().double()).norm()) <= 2.0 ** -7 * float(want.detach().double().norm())
    for p, q in zip(moe.parameters(), moe2.parameters()):
        assert (p.grad is None and q.grad is None) or torch.equal(p.grad, q.grad)


def test_moe_residual_partial_gradients(gpu_device):
    # only what is asked for is computed, with the same bits: input, weight, bias, each alone and none of them
    cfg = configs.BlockConfig("t", 37, dim=128, inter=192, n_experts=4, topk=2)
    data = configs.make_block(cfg, seed=6)
    moe = build_module(cfg, data, gpu_device, BF)
    norm = LayerNorm(128).to(gpu_device, BF)
    dy = data.dy.to(gpu_device, BF)
    x = data.x.to(gpu_device, BF)

    def run(pick, block):
        norm.weight.requires_grad_(1 in pick)
        norm.bias.requires_grad_(2 in pick)
        moe.requires_grad_(block)
        xs = x.clone().requires_grad_(0 in pick)
        leaves = [t for i, t in enumerate((xs, norm.weight, norm.bias)) if i in pick]
        leaves += [moe.experts[0].w1.weight] if block else []
        y = moe_residual(xs, norm, moe)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy)) if leaves else (y.detach(),)

    y, dx, dw, db, d1 = run((0, 1, 2), True)
    full = (dx, dw, db)
    for pick in ((), (0,), (1,), (2,), (0, 1), (1, 2), (0, 2)):
        for block in (True, False):
            got = run(pick, block)
            want = (y, *(full[i] for i in pick), *((d1,) if block else ()))
            assert len(got) == len(want) and all(torch.equal(p, q) for p, q in zip(got, want)), (pick, block)


def test_forward_mode_derivatives_are_refused(gpu_device):
    # eager, traced, through torch.func, and where a parameter requires a gradient; vmap has no rule either
    import torch.autograd.forward_ad as fw
    x, w, b, _ = inputs(6, 64, F32, F32, gpu_device)
    t = torch.ones_like(x)
    with fw.dual_level():
        d = fw.make_dual(x, t)
        for call in (lambda: layer_norm(d, w, b), lambda: layer_norm(d, w.clone().requires_grad_(True), b),
                     lambda: torch.ops.fusionllm.layer_norm_fwd(d, w, b, 1e-5, F32)):
            with pytest.raises(NotImplementedError):
                call()
        with torch.no_grad(), pytest.raises(NotImplementedError):
            layer_norm(d, w, b)
        layer_norm(x, w, b)  # no tangent: as ever
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda v: layer_norm(v, w, b), (x,), (t,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: layer_norm(v, w, b))(x)


def test_moe_residual_calls_hooks(gpu_device):
    cfg = configs.BlockConfig("t", 20, dim=128, inter=192, n_experts=4, topk=2)
    data = configs.make_block(cfg, seed=7)
    moe = build_module(cfg, data, gpu_device, BF)
    x = data.x.to(gpu_device, BF)
    for norm in (LayerNorm(128).to(gpu_device, BF), nn.RMSNorm(128).to(gpu_device, BF)):
        seen = []
        handle = norm.register_forward_hook(lambda m, a, out: seen.append(out) or 2 * out)
        with torch.no_grad():
            y = moe_residual(x, norm, moe)
            assert len(seen) == 1
            handle.remove()
            assert torch.equal(y, x + moe(2 * norm(x)))
            # bounds as above: the block's output is rounded before the add, or after it
            want = (x + moe(norm(x))).double()
            assert float((moe_residual(x, norm, moe).double() - want).norm()) <= 2.0 ** -7 * float(want.norm())
