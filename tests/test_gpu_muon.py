"""Orthogonalised updates and the Muon step against their formulas in 64 bits.

Tolerances.  The kernels round to fp16 at stated places (X with an fp8 remainder, A and
a I + B; hi + lo where an operand is held in 22 bits) and sum in fp32.  ``emulate`` does the same roundings
in 64 bits, so |emulate - exact| is the error that the scheme makes on this very
matrix.  The kernel's roundings fall elsewhere in their last place (its sums are
fp32, in another order), so its error is another draw of the same size: bound 3 x,
plus the fp32 sums themselves: a product over K is a chain of K / 32 accumulations
(K padded to 64) whose running sum loses at most 2^-23 of itself each, even where the
matrix unit cuts instead of rounding, so K / 32 2^-23 of the product in one direction
(three accumulations for every 32 in the 22-bit form).  How far such a loss in every product moves the result is
computed too: ``emulate`` with every product scaled by it, against the one without.
Plus half a step of the result's type.  An element is within 8 standard deviations (the bound's root mean square)
of its value, plus half a step of it."""
import copy
import math

import pytest
import torch

from fusionllm_amd import _kernels as K
from fusionllm_amd.optim import NS_COEFFICIENTS, Muon, orthogonalize

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
SMALL_SPLIT = 128  # matrices of a smaller side up to this are held in 22 bits whatever their type


def half(t):
    return torch.finfo(t).eps / 2


def exact(g, steps=5, co=NS_COEFFICIENTS, eps=1e-7):
    flip = g.shape[0] > g.shape[1]
    x = g.double()
    x = x.t().contiguous() if flip else x
    x = x / max(float(x.norm()), eps)
    for _ in range(steps):
        a = x @ x.t().contiguous()
        x = co[0] * x + (co[1] * a + co[2] * (a @ a)) @ x
    return x.t() if flip else x


def is_small(g):
    """Whether the fp32 kernels of small matrices run: a side up to 64, 32 panels of 128 columns."""
    return min(g.shape) <= 64 and max(g.shape) <= 4096


def emulate(g, steps=5, co=NS_COEFFICIENTS, eps=1e-7, split=False, cut=False):
    if is_small(g):
        return emulate_small(g, steps, co, eps, cut)

    def parts(v, scale):
        s = v * 2.0 ** scale
        h = s.half().double()
        lo = (s - h).half().double()
        return h * 2.0 ** -scale, lo * 2.0 ** -scale

    def mul(p, q):
        r = p[0] @ q[0]
        r = r + p[0] @ q[1] + p[1] @ q[0] if split else r
        k = -(-p[0].shape[1] // 64) * 2 * (3 if split else 1)
        return r * (1 - k * 2.0 ** -23) if cut else r

    tr = lambda p: tuple(t.t().contiguous() for t in p)
    flip = g.shape[0] > g.shape[1]
    x = g.double()
    x = x.t().contiguous() if flip else x
    x = x / max(float(x.norm()), eps)
    eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    for k in range(steps):
        xs = parts(x, 14)
        a = parts(mul(xs, tr(xs)), 13)
        b = parts(co[0] * eye + co[1] * (a[0] + a[1] if split else a[0]) + co[2] * mul(a, tr(a)), 13)
        # the remainder of X, where it is no operand: fp8, and not in the last step
        lo = ((x - xs[0]) * 2.0 ** 18).float().to(torch.float8_e4m3fn).double() * 2.0 ** -18
        x = mul(b, xs) + (0 if split or k == steps - 1 else co[0] * lo)
    return x.t() if flip else x


def emulate_small(g, steps, co, eps, cut):
    """fp32 operands: X, A and a I + b A + c A^2 rounded to fp32.  The sums: a product over K takes K / 4
    accumulations, the Gram matrix in panels of 128 columns whose sums are added in a chain."""
    r = lambda v: v.float().double()

    def mul(p, q, panels=0):
        k = p.shape[1] / 4 if not panels else 32 + panels
        return p @ q * (1 - k * 2.0 ** -23 if cut else 1)

    flip = g.shape[0] > g.shape[1]
    x = g.double()
    x = x.t().contiguous() if flip else x
    panels = -(-x.shape[1] // 128)
    x = x / max(float(x.norm()), eps)
    eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    for _ in range(steps):
        x = r(x)
        a = r(mul(x, x.t().contiguous(), panels))
        x = mul(r(co[0] * eye + co[1] * a + co[2] * mul(a, a)), x)
    return x.t() if flip else x


def ortho_bound(g, want, dtype, **kw):
    """Bounds of a result of dtype before its rounding: of the relative error (2-norm), and of every
    element's."""
    if not want.any():
        return 0.0, torch.zeros_like(want)
    split = dtype == F32 or min(g.shape) <= SMALL_SPLIT
    e = emulate(g, split=split, **kw)
    cut = emulate(g, split=split, cut=True, **kw) - e
    d = e - want
    rms = lambda t, dim=None: (t * t).mean(dim, keepdim=dim is not None).sqrt()
    size = rms(d, 1) * rms(d, 0) / rms(d).clamp_min(1e-300) + rms(d)
    rel = (3 * float(d.norm()) + float(cut.norm())) / float(want.norm()) + 2.0 ** -22
    return rel, 24 * size + cut.abs() + 2.0 ** -20 * want.abs()


def check_ortho(got, g, dtype, **kw):
    want = exact(g, **kw)
    assert got.dtype == dtype and got.shape == g.shape
    err = got.double() - want
    rel_tol, tol = ortho_bound(g, want, dtype, **kw)
    rel = float(err.norm()) / max(float(want.norm()), 1e-300)
    assert rel <= rel_tol + half(dtype), f"{tuple(g.shape)}: {rel:.2e} off, {rel_tol + half(dtype):.2e} allowed"
    bad = err.abs() > tol + half(dtype) * (want.abs() + tol)
    assert not bad.any(), (f"{tuple(g.shape)}: {int(bad.sum())} elements off, worst "
                           f"{float((err.abs() / (tol + half(dtype) * (want.abs() + tol))).max()):.2f} x the bound")


def gradient(rows, cols, dev, seed, rank=None, fall=0.5):
    gen = torch.Generator().manual_seed(seed)
    rank = min(rows, cols) + 8 if rank is None else rank
    left = torch.randn(rows, rank, generator=gen) * (torch.arange(rank) + 1.0) ** -fall
    return (left @ torch.randn(rank, cols, generator=gen) * 1e-3).to(dev)


SHAPES = [(1, 1), (1, 7), (9, 1), (2, 3), (8, 768), (64, 64), (63, 65), (65, 64), (5, 200), (128, 130), (129, 129),
          (130, 700), (64, 4096), (4097, 64), (48, 4097), (17, 129), (257, 191), (300, 301), (512, 512), (768, 2048), (2048, 768), (1001, 1503)]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_orthogonalize_against_64_bits(gpu_device, rows, cols, dtype):
    g = gradient(rows, cols, gpu_device, rows * 7 + cols).to(dtype)
    check_ortho(orthogonalize(g), g, dtype)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rank,fall", [(1, 0.0), (8, 0.5), (64, 0.5), (400, 1.0)])
def test_low_rank_and_steep_spectra(gpu_device, rank, fall, dtype):
    # an expert that saw few tokens: its gradient has their rank, and the directions that it does
    # not have must not grow out of roundings
    for rows, cols in ((256, 640), (640, 256)):
        g = gradient(rows, cols, gpu_device, rank, rank, fall).to(dtype)
        check_ortho(orthogonalize(g), g, dtype)


@pytest.mark.parametrize("co,steps", [((1.5, -0.5, 0.0), 12), ((2.0, -1.5, 0.5), 8), (NS_COEFFICIENTS, 1),
                                      (NS_COEFFICIENTS, 2), (NS_COEFFICIENTS, 10)])
def test_other_polynomials_and_steps(gpu_device, co, steps):
    for dtype in (BF, F32):
        g = gradient(150, 222, gpu_device, 5, fall=0.2).to(dtype)
        check_ortho(orthogonalize(g, steps=steps, coefficients=co), g, dtype, steps=steps, co=co)


def test_scale_of_the_input(gpu_device):
    # values near the ends of the type's range: the norm is summed in fp64; below eps it is eps
    g = gradient(70, 90, gpu_device, 1)
    for g in (g, gradient(40, 300, gpu_device, 2)):
        for scale in (1e30, 1e-3, 1e-20):
            x = g * scale
            check_ortho(orthogonalize(x, eps=1e-30), x, F32, eps=1e-30)
        x = g * 1e-9
        check_ortho(orthogonalize(x, eps=1e-3), x, F32, eps=1e-3)
        # columns of very different size (panels of a small matrix have factors of their own)
        x = g * torch.exp2(torch.linspace(-40, 40, g.shape[1], device=gpu_device)).round()
        check_ortho(orthogonalize(x), x, F32)


def test_norms_far_below_eps(gpu_device):
    # X is stored in steps of at least 2^-24 / 2^14 (fp16's smallest, times X's factor), and five steps multiply
    # what is that small by a each: the error of an element is below steps a^5 2^-38, some 2^-27
    for dtype in (BF, F32):
        g = (gradient(150, 260, gpu_device, 8) * 1e-14).to(dtype)
        err = orthogonalize(g).double() - exact(g)
        assert float(err.abs().max()) <= 5 * NS_COEFFICIENTS[0] ** 5 * 2.0 ** -38


def test_zero_nan_and_infinite_matrices(gpu_device):
    # in one launch with a clean one, which they leave alone
    for rows, cols in ((96, 160), (30, 260), (260, 30)):
        g = gradient(rows, cols, gpu_device, 3)
        stack = torch.stack([g, torch.zeros_like(g), g, g, g])
        stack[2, 5, 7] = float("nan")
        stack[3, rows - 1, cols - 1] = float("inf")
        out = orthogonalize(stack)
        assert torch.equal(out[0], out[4]) and torch.equal(out[0], orthogonalize(g))
        assert not out[1].any()
        assert torch.isnan(out[2]).all() and torch.isnan(out[3]).all()


def test_stacks_lists_and_mixed_sizes(gpu_device):
    # each matrix as it comes out alone, whatever it is launched with
    mats = [gradient(r, c, gpu_device, i).to(d) for i, (r, c, d) in enumerate(
        [(40, 200, BF), (200, 40, BF), (64, 64, F32), (200, 40, F32), (40, 200, BF), (33, 33, BF)])]
    stack = torch.stack([gradient(40, 200, gpu_device, 50 + i) for i in range(6)]).to(BF).view(2, 3, 40, 200)
    outs = orthogonalize([*mats, stack])
    for m, o in zip(mats, outs):
        assert o.shape == m.shape and torch.equal(o, orthogonalize(m))
    for i in range(2):
        for j in range(3):
            assert torch.equal(outs[-1][i, j], orthogonalize(stack[i, j]))
    # a transposed view, a slice of wider rows, more matrices than a launch takes, none at all
    t = mats[0].t()
    assert torch.equal(orthogonalize(t), orthogonalize(t.contiguous()))
    s = mats[0][:, 3:150]
    assert torch.equal(orthogonalize(s), orthogonalize(s.contiguous()))
    many = torch.stack([gradient(20, 30, gpu_device, i) for i in range(70)])
    out = orthogonalize(many)
    assert torch.equal(out[0], orthogonalize(many[0])) and torch.equal(out[69], orthogonalize(many[69]))
    assert orthogonalize([]) == [] and orthogonalize(torch.empty(3, 0, 5, device=gpu_device)).shape == (3, 0, 5)


def test_many_matrices_take_the_large_tiles(gpu_device):
    # enough of them for the 128 x 128 tiles; some against 64 bits, and twice the same bits
    for dtype, rows, cols in ((BF, 320, 450), (F32, 320, 450), (BF, 450, 321)):
        stack = torch.stack([gradient(rows, cols, gpu_device, i) for i in range(64)]).to(dtype)
        out = orthogonalize(stack)
        for i in (0, 17, 63):
            check_ortho(out[i], stack[i], dtype)
            if dtype == BF:
                # every tile size sums in the same order.  (With operands hi + lo, the two small products of an
                # element above the diagonal come in one order where a tile has it and in the other where
                # a tile below mirrors it.)
                assert torch.equal(out[i], orthogonalize(stack[i]))
        assert torch.equal(out, orthogonalize(stack))


def test_output_is_written_whole_and_nothing_else(gpu_device):
    for r, c in ((65, 129), (129, 65), (33, 130), (130, 33)):
        g = gradient(r, c, gpu_device, 2)
        buf = torch.full((r * c + 64,), 7.0, device=gpu_device)
        out = buf[32:32 + r * c].view(r, c)
        K.orthogonalize([g], [out], 5, NS_COEFFICIENTS, 1e-7)
        assert torch.equal(out, orthogonalize(g))
        assert (buf[:32] == 7).all() and (buf[32 + r * c:] == 7).all()
        inplace = g.clone()
        K.orthogonalize([inplace], [inplace], 5, NS_COEFFICIENTS, 1e-7)
        assert torch.equal(inplace, out)


# ---- Muon -----------------------------------------------------------------------------------


def model(dev, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    shapes = [(48, 200), (200, 48), (48, 200), (64, 64), (300, 140), (1, 40), (129, 131)]
    ps = [torch.nn.Parameter((0.05 * torch.randn(s, generator=gen)).to(dev, dtype)) for s in shapes]
    return ps


def set_grads(ps, seed):
    for i, p in enumerate(ps):
        p.grad = gradient(*p.shape, p.device, seed * 100 + i).to(p.dtype)


def expect_step(p, g, buf, lr, wd, mom, nesterov, adjust, **kw):
    """(param, momentum) after a step in 64 bits and the bounds of their errors before rounding."""
    p, g, buf = p.double(), g.double(), buf.double()
    buf = mom * buf + (1 - mom) * g
    u = (1 - mom) * g + mom * buf if nesterov else buf
    r, c = p.shape
    lr_ = lr * 0.2 * math.sqrt(max(r, c)) if adjust == "match_rms_adamw" else lr * math.sqrt(max(1, r / c))
    o = exact(u, **kw)
    return p * (1 - lr * wd) - lr_ * o, buf, lr_, o, u


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("nesterov,adjust,wd", [(True, None, 0.1), (False, "match_rms_adamw", 0.0),
                                                (True, "original", 0.3)])
def test_muon_steps_against_64_bits(gpu_device, dtype, nesterov, adjust, wd):
    """Each step from the state it finds.  Momentum: three fp32 operations and a rounding.
    Parameters: the bound of the orthogonalised update (whose input differs by fp32
    operations: 2^-22 more, of the size of the bound's floor) times the step size, three fp32
    operations and a rounding."""
    lr, mom = 0.03, 0.9
    ps = model(gpu_device, dtype)
    opt = Muon(ps, lr=lr, weight_decay=wd, momentum=mom, nesterov=nesterov, adjust_lr_fn=adjust)
    for step in range(3):
        set_grads(ps, step)
        before = [(p.detach().clone(), p.grad.clone(),
                   opt.state[p]["momentum_buffer"].clone() if step else torch.zeros_like(p)) for p in ps]
        opt.step()
        for p, (p0, g, b0) in zip(ps, before):
            want, buf, lr_, o, u = expect_step(p0, g, b0, lr, wd, mom, nesterov, adjust)
            got = opt.state[p]["momentum_buffer"]
            berr = (got.double() - buf).abs()
            size = mom * b0.double().abs() + (1 - mom) * g.double().abs()
            assert (berr <= 4 * 2.0 ** -24 * size + half(dtype) * buf.abs() * (1 + 2.0 ** -20)).all()
            rms = float(o.norm()) / math.sqrt(o.numel())
            tol = lr_ * (ortho_bound(u, o, dtype)[1] + 8 * 2.0 ** -20 * rms)
            err = (p.detach().double() - want).abs()
            tol = tol + 4 * 2.0 ** -24 * (p0.double().abs() + lr_ * o.abs())
            assert (err <= tol + half(dtype) * (want.abs() + tol)).all(), (step, tuple(p.shape))
            assert torch.equal(p.grad, g)  # read only


def test_muon_is_the_pieces_one_after_the_other(gpu_device):
    # momentum in fp32 by torch, the public orthogonalize, the update: the same launch sequence inside
    p = torch.nn.Parameter(gradient(140, 300, gpu_device, 1))
    p.grad = gradient(140, 300, gpu_device, 2)
    p0 = p.detach().clone()
    Muon([p], lr=0.5, weight_decay=0.0, momentum=0.0, nesterov=False).step()
    want = p0.double() - 0.5 * orthogonalize(p.grad).double()
    torch.testing.assert_close(p.detach().double(), want, rtol=1e-6, atol=1e-7)


def test_launches_are_split_by_their_workspace(gpu_device, monkeypatch):
    from fusionllm_amd import optim
    mats = torch.stack([gradient(70, 80, gpu_device, i) for i in range(6)])
    want = orthogonalize(mats)
    calls = []
    launch = K.orthogonalize
    monkeypatch.setattr(K, "orthogonalize", lambda m, *a: (calls.append(len(m)), launch(m, *a)))
    monkeypatch.setattr(optim, "LAUNCH_ELEMENTS", 4 * 70 * 80 + 1)
    assert torch.equal(orthogonalize(mats), want) and calls == [4, 2]
    monkeypatch.setattr(optim, "LAUNCH_ELEMENTS", 1)
    assert torch.equal(orthogonalize(mats), want) and calls[2:] == [1] * 6


@pytest.mark.parametrize("nesterov,adjust", [(True, None), (False, "match_rms_adamw")])
def test_muon_is_a_drop_in_for_torchs(gpu_device, nesterov, adjust):
    # the same two steps by torch.optim.Muon on the CPU, whose products are bf16: its updates are within
    # 1 - 2 % (bf16 products, simulated: 1.0e-2 .. 1.4e-2) of the exact ones; a wrong scale,
    # momentum or decay is not within 5 %
    if not hasattr(torch.optim, "Muon"):
        pytest.skip("this torch has no Muon")
    ps = [torch.nn.Parameter(0.05 * torch.randn(s)) for s in ((48, 200), (200, 48), (96, 96))]
    mine = [torch.nn.Parameter(p.detach().to(gpu_device)) for p in ps]
    kw = dict(lr=0.05, weight_decay=0.2, momentum=0.9, nesterov=nesterov, adjust_lr_fn=adjust)
    a, b = torch.optim.Muon(ps, **kw), Muon(mine, **kw)
    for step in range(2):
        for i, (p, q) in enumerate(zip(ps, mine)):
            g = gradient(*p.shape, "cpu", 10 * step + i, fall=0.2)
            p.grad, q.grad = g, g.to(gpu_device)
        before = [p.detach().clone() for p in ps]
        for p, q in zip(ps, mine):
            with torch.no_grad():
                q.copy_(p)
        a.step()
        b.step()
        for p, q, p0 in zip(ps, mine, before):
            moved = p.detach() - p0
            assert (q.detach().cpu() - p.detach()).norm() <= 0.05 * moved.norm()
            torch.testing.assert_close(b.state[q]["momentum_buffer"].cpu(), a.state[p]["momentum_buffer"],
                                       rtol=1e-6, atol=1e-9)


def test_muon_skips_groups_and_state(gpu_device):
    ps = model(gpu_device, F32)
    opt = Muon([{"params": ps[:3]}, {"params": ps[3:], "lr": 0.0, "weight_decay": 0.0}], lr=0.02)
    set_grads(ps, 1)
    ps[1].grad = None
    before = [p.detach().clone() for p in ps]
    opt.step()
    assert torch.equal(ps[1], before[1]) and ps[1] not in opt.state  # no gradient: untouched
    assert not torch.equal(ps[0], before[0])
    assert all(torch.equal(p, b) for p, b in zip(ps[3:], before[3:]))  # step size 0
    assert all(opt.state[p]["momentum_buffer"].any() for p in ps[3:])
    # a checkpoint goes on with the same bits
    twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt2 = Muon([{"params": twin[:3]}, {"params": twin[3:]}])
    opt2.load_state_dict(copy.deepcopy(opt.state_dict()))
    set_grads(ps, 2)
    set_grads(twin, 2)
    opt.step()
    opt2.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, twin))
    # a closure runs with gradients on and its loss comes back
    assert opt.step(lambda: (ps[0] ** 2).sum().requires_grad_() * 0 + 3.0) == 3.0


def test_muon_launch_groupings_give_the_same_bits(gpu_device):
    # 70 matrices of one size (two launches) against one optimizer each
    mats = [gradient(24, 40, gpu_device, i) for i in range(70)]
    a = [torch.nn.Parameter(m.clone()) for m in mats]
    b = [torch.nn.Parameter(m.clone()) for m in mats]
    for i, (p, q) in enumerate(zip(a, b)):
        p.grad = q.grad = gradient(24, 40, gpu_device, 1000 + i)
    Muon(a, lr=0.1).step()
    for q in b:
        Muon([q], lr=0.1).step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_muon_of_two_parameters_on_one_storage(gpu_device):
    # tied weights given as two parameters: the updates are applied one after the other
    w = gradient(32, 48, gpu_device, 1)
    store = w.clone()
    p, q = torch.nn.Parameter(store), torch.nn.Parameter(store)
    assert p.data_ptr() == q.data_ptr()
    p.grad, q.grad = gradient(32, 48, gpu_device, 2), gradient(32, 48, gpu_device, 3)
    Muon([p, q], lr=0.1).step()
    r = torch.nn.Parameter(w.clone())
    for g in (p.grad, q.grad):
        r.grad = g
        Muon([r], lr=0.1).step()
    assert torch.equal(p, r)


def test_muon_under_graph_capture(gpu_device):
    # one step captured; every replay on new gradients against the eager optimizer
    for dtype in (BF, F32):
        ps = model(gpu_device, dtype)
        twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        opt, ref = Muon(ps, lr=0.05), Muon(twin, lr=0.05)
        for step in range(2):  # state and kernels exist before the capture
            set_grads(ps, step)
            set_grads(twin, step)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                opt.step()
            torch.cuda.current_stream().wait_stream(side)
            ref.step()
        static = [p.grad for p in ps]
        graph = torch.cuda.CUDAGraph()
        saved = [(p.detach().clone(), opt.state[p]["momentum_buffer"].clone()) for p in ps]
        with torch.cuda.graph(graph):
            opt.step()
        for p, (w, m) in zip(ps, saved):  # a capture runs nothing
            assert torch.equal(p, w) and torch.equal(opt.state[p]["momentum_buffer"], m)
        for step in range(2, 6):
            set_grads(twin, step)
            for s, q in zip(static, twin):
                s.copy_(q.grad)
            graph.replay()
            ref.step()
            torch.cuda.synchronize()
            for p, q in zip(ps, twin):
                assert torch.equal(p, q), step
                assert torch.equal(opt.state[p]["momentum_buffer"], ref.state[q]["momentum_buffer"]), step


def test_orthogonalize_on_two_streams(gpu_device):
    g = [torch.stack([gradient(130, 260, gpu_device, 10 * k + i) for i in range(4)]) for k in range(2)]
    want = [orthogonalize(x) for x in g]
    torch.cuda.synchronize()
    outs = [None, None]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[k] = orthogonalize(g[k])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_a_block_trains_with_layer_norm_and_muon(gpu_device):
    """The operators as they are used together: x + moe(layer_norm(x)), backward, one Muon
    step over the block's matrices; every gradient and update as the pieces give it."""
    from fusionllm_amd import LayerNorm, configs, moe_residual
    from tests.gpu_util import build_module
    cfg = configs.BlockConfig("t", 64, dim=128, inter=192, n_experts=4, topk=2)
    data = configs.make_block(cfg, seed=1)
    moe = build_module(cfg, data, gpu_device, BF)
    norm = LayerNorm(128).to(gpu_device, BF)
    x = data.x.to(gpu_device, BF)
    mats = [p for p in moe.parameters() if p.dim() == 2]
    opt = Muon(mats, lr=0.02)
    for step in range(3):
        opt.zero_grad()
        norm.zero_grad()
        y = moe_residual(x, norm, moe)
        y.backward(data.dy.to(gpu_device, BF))
        assert torch.isfinite(norm.weight.grad).all() and norm.weight.grad.any() and norm.bias.grad.any()
        before = [p.detach().clone() for p in mats]
        grads = [None if p.grad is None else p.grad.clone() for p in mats]
        bufs = [opt.state[p]["momentum_buffer"].clone() if p in opt.state and opt.state[p] else None for p in mats]
        opt.step()
        for p, p0, g, b in zip(mats, before, grads, bufs):
            if g is None:
                assert torch.equal(p, p0)
                continue
            want, _, lr_, o, u = expect_step(p0, g, torch.zeros_like(g) if b is None else b, 0.02, 0.1, 0.95, True,
                                             None)
            rms = float(o.norm()) / math.sqrt(o.numel())
            tol = lr_ * (ortho_bound(u, o, BF)[1] + 8 * 2.0 ** -20 * rms) + 1e-9
            err = (p.detach().double() - want).abs()
            assert (err <= tol + half(BF) * (want.abs() + tol)).all()


def test_wrappers_refuse_what_the_kernels_do_not_take(gpu_device):
    a, b = torch.randn(2, 32, 48, device=gpu_device)
    out = torch.empty_like(a)
    go = lambda m, o: K.orthogonalize(m, o, 5, NS_COEFFICIENTS, 1e-7)
    with pytest.raises(RuntimeError, match="one output per matrix"):
        go([a, b], [out])
    with pytest.raises(RuntimeError, match="matrix of shape"):
        go([a], [out.t().contiguous()])
    with pytest.raises(RuntimeError, match="contiguous"):
        go([a.t()], [out.t()])
    with pytest.raises(RuntimeError, match="float32"):
        go([a], [out.bfloat16()])
    with pytest.raises(RuntimeError, match="unsupported shape"):
        go([a, torch.randn(32, 40, device=gpu_device)], [out, torch.empty(32, 40, device=gpu_device)])
    with pytest.raises(RuntimeError, match="at most 64"):
        go([a] * 65, [out] * 65)
    with pytest.raises(RuntimeError, match="coefficients"):
        K.orthogonalize([a], [out], 5, (4.0, -4.775, 2.0315), 1e-7)
    with pytest.raises(RuntimeError, match="coefficients"):
        orthogonalize(a, coefficients=(3.0, 0.0, 0.0))
    p = torch.nn.Parameter(a.clone())
    p.grad = b.clone()
    before = p.detach().clone()
    with pytest.raises(RuntimeError, match="coefficients"):
        Muon([p], ns_coefficients=(8.0, -9.0, 1.5)).step()
    q = torch.nn.Parameter(torch.randn(48, 32, device=gpu_device).t())
    q.grad = b.clone()
    with pytest.raises(NotImplementedError, match="contiguous"):
        Muon([q]).step()
    assert torch.equal(p, before)


def test_muon_takes_gradients_of_any_stride(gpu_device):
    p = torch.nn.Parameter(gradient(40, 70, gpu_device, 1))
    q = torch.nn.Parameter(p.detach().clone())
    g = gradient(70, 40, gpu_device, 2)
    p.grad, q.grad = g.t(), g.t().contiguous()
    Muon([p], lr=0.1).step()
    Muon([q], lr=0.1).step()
    assert torch.equal(p, q)


def test_muon_on_a_side_stream(gpu_device):
    ps, twin = model(gpu_device, BF), model(gpu_device, BF)
    set_grads(ps, 4)
    set_grads(twin, 4)
    a, b = Muon(ps, lr=0.1), Muon(twin, lr=0.1)
    b.step()
    b.step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a.step()
        a.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ps, twin))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("tall", [False, True], ids=["wide", "tall"])
def test_largest_matrix(gpu_device, tall, dtype):
    # 8192 x 65536, offsets up to 2^31 bytes; one step, every 13th column against 64 bits.  X = P X0: the
    # error of P is at most its operands' roundings and its sums' losses, each relative to the Frobenius norm of
    # what is rounded or summed, and a column of X is off by at most that times its X0's norm.
    m, n = 8192, 65536
    g = torch.Generator(gpu_device).manual_seed(5)
    x = (torch.randn(m, 8, device=gpu_device, generator=g) @ torch.randn(8, n, device=gpu_device, generator=g)
         + 0.01 * torch.randn(m, n, device=gpu_device, generator=g)).to(dtype)
    got = orthogonalize(x.t().contiguous() if tall else x, steps=1)
    got = (got.t() if tall else got)[:, ::13].double()
    x0 = x.double()
    del x
    x0 /= x0.norm()
    a = torch.zeros(m, m, dtype=torch.float64, device=gpu_device)
    for part in x0.split(8192, 1):
        a += part.contiguous() @ part.t().contiguous()
    ca, cb, cc = NS_COEFFICIENTS
    sq = a @ a
    xs = x0[:, ::13].contiguous()
    want = ca * xs + (cb * a + cc * sq) @ xs
    f = lambda t: float(t.norm())
    operand = 2.0 ** -11 if dtype == BF else 2.0 ** -21
    step = 2.0 ** -23 * (1 if dtype == BF else 3)  # lost per accumulation of 32 (three of them in the 22-bit form)
    top = float(torch.linalg.vector_norm(a @ xs[:, 0]) / torch.linalg.vector_norm(xs[:, 0])) * 1.5  # > largest value of A
    err_a = (3 * operand + n / 32 * step) * f(a)          # X twice and A itself
    err_p = (abs(cb) + 2 * abs(cc) * top) * err_a + m / 32 * step * abs(cc) * f(sq)
    err_p += operand * (ca + f(cb * a + cc * sq))         # P's rounding
    err = err_p + (operand + m / 32 * step) * (ca + f(cb * a + cc * sq))  # the last product
    off = (got - want).norm(dim=0)
    allowed = err * xs.norm(dim=0) + half(dtype) * want.norm(dim=0)
    assert bool((off <= allowed).all()), (float((off / allowed).max()), int((off / allowed).argmax()))


def test_many_large_matrices_in_one_launch(gpu_device):
    # 20 of 8192 x 8192 in fp32: 5 GiB of X.  The same kernels run for one of them: the same bits.
    g = torch.Generator(gpu_device).manual_seed(6)
    x = torch.randn(20, 8192, 8192, device=gpu_device, generator=g)
    out = torch.empty_like(x)
    K.orthogonalize(list(x), list(out), 1, NS_COEFFICIENTS, 1e-7)
    one = torch.empty_like(x[0])
    for i in (0, 1, 7, 8, 13, 19):
        K.orthogonalize([x[i]], [one], 1, NS_COEFFICIENTS, 1e-7)
        assert torch.equal(one, out[i]), i


def test_muon_of_overlapping_parameters(gpu_device):
    # rows 0 .. 39 and 20 .. 59 of one matrix, given together: one after the other, as the formulas say
    g = torch.Generator(gpu_device).manual_seed(3)
    base = torch.randn(60, 96, device=gpu_device, generator=g)
    grads = [torch.randn(40, 96, device=gpu_device, generator=g) for _ in range(2)]

    def run(groups, t):
        ps = [torch.nn.Parameter(t[:40]), torch.nn.Parameter(t[20:])]
        for p, q in zip(ps, grads):
            p.grad = q
        for group in groups:
            Muon([ps[i] for i in group], lr=0.1).step()
        return t

    assert torch.equal(run([(0, 1)], base.clone()), run([(0,), (1,)], base.clone()))


def test_muon_of_overlapping_parameters_of_other_sides(gpu_device):
    # rows 0 .. 19, 15 .. 44 and 40 .. 59 of one matrix: each update as if it were alone, in their order
    g = torch.Generator(gpu_device).manual_seed(4)
    base = torch.randn(60, 96, device=gpu_device, generator=g)
    cuts = ((0, 20), (15, 45), (40, 60))
    grads = [torch.randn(b - a, 96, device=gpu_device, generator=g) for a, b in cuts]

    def run(groups, t):
        ps = [torch.nn.Parameter(t[a:b]) for a, b in cuts]
        for p, q in zip(ps, grads):
            p.grad = q
        for group in groups:
            Muon([ps[i] for i in group], lr=0.1).step()
        return t

    assert torch.equal(run([(0, 1, 2)], base.clone()), run([(0,), (1,), (2,)], base.clone()))


@pytest.mark.parametrize("eps", [1e-7, 1e-30, 1e-40, 1e-310, 5e-324])
def test_zero_parts_under_any_eps(gpu_device, eps):
    # zeros stay zeros whatever they are divided by: a whole matrix, and 128 columns of one whose norm is as
    # small as eps (1 / eps is beyond fp32, or beyond fp64)
    for rows, cols in ((96, 160), (30, 300), (300, 30)):
        z = torch.zeros(rows, cols, device=gpu_device)
        assert not orthogonalize(z, eps=eps).any()
        assert not orthogonalize(z.bfloat16(), eps=eps).any()
        z[3, 5] = 2.0 ** -140
        z[5, 3] = -2.0 ** -140
        check_ortho(orthogonalize(z, eps=eps), z, F32, eps=eps)


# Launches that take every tile size, none with sides that are multiples of it: sides, matrices, tile rows of
# the symmetric products and of the updates (checked on the host: test_host_training_ops.py has the same table)
LAUNCHES = [(700, 1030, 27, 256, 256), (700, 1030, 10, 128, 128), (400, 600, 56, 256, 256), (1400, 1500, 24, 256, 256),
            (320, 450, 64, 128, 256), (321, 449, 20, 64, 128), (700, 1030, 3, 64, 64)]
LAUNCH_IDS = [f"{c}x{m}x{n}" for m, n, c, _, _ in LAUNCHES]


def mixed(m, n, count, dev, dtype, seed=0, rank=None):
    """count matrices, wide and tall ones in turn; every one another (rows and columns rolled)."""
    base = [gradient(m, n, dev, seed + i, rank) for i in range(3)]
    mats = [base[i % 3].roll((7 * i, 11 * i), (0, 1)) * (1 + i % 5) for i in range(count)]
    return [(x.t().contiguous() if i % 2 else x).to(dtype) for i, x in enumerate(mats)]


def emulate_chain(g, steps=5, co=NS_COEFFICIENTS, eps=1e-7):
    """The 22-bit form with its sums as they are formed: a chain of accumulations, hi lo, lo hi and hi hi of every
    32 products, each cut to 24 bits.

    ``emulate(cut=True)`` scales a product as a whole and so takes a sum's loss to be a share of what it ends
    as.  Off the diagonal of A it is more: K products of mixed sign that end near zero stand at up to sqrt(K) of
    their size on the way, and each of the 3 K / 32 accumulations loses up to 2^-23 of where the sum stands.
    Cutting loses 2^-23 / sqrt(3) of the running sum in the root mean square, rounding half as much; over
    3 K / 32 = 132 accumulations of 1408 products, sqrt(132) 2^-23 / sqrt(3) = 7.9e-7 of a running sum of
    about half of sqrt(1408) products.  Of 1400 x 1500 the operands' roundings move the result by 1.0e-8 (root mean
    square, of values of 2.2e-2), the chain with rounding by 3.9e-8, the chain with cuts by twice that: at sides
    beyond some hundred the sums are what the error is made of."""
    def parts(v, scale):
        s = v.float().double() * 2.0 ** scale
        h = s.half().double()
        return h * 2.0 ** -scale, (s - h).half().double() * 2.0 ** -scale

    def cut(v):
        f = v.float()
        return torch.where(f.double().abs() > v.abs(), torch.nextafter(f, torch.zeros_like(f)), f)

    def mul(p, q):
        acc = torch.zeros(p[0].shape[0], q[0].shape[1], dtype=torch.float32, device=p[0].device)
        for k in range(0, p[0].shape[1], 32):
            for x, y in ((0, 1), (1, 0), (0, 0)):
                acc = cut(acc.double() + p[x][:, k:k + 32].contiguous() @ q[y][k:k + 32])
        return acc.double()

    tr = lambda p: tuple(t.t().contiguous() for t in p)
    flip = g.shape[0] > g.shape[1]
    x = g.double()
    x = x.t().contiguous() if flip else x
    x = x / max(float(x.norm()), eps)
    eye = torch.eye(x.shape[0], dtype=torch.float64, device=x.device)
    for _ in range(steps):
        xs = parts(x, 14)
        a = parts(mul(xs, tr(xs)), 13)
        x = mul(parts(co[0] * eye + co[1] * (a[0] + a[1]) + co[2] * mul(a, tr(a)), 13), xs)
    return x.t() if flip else x


def launch_bound(g, want, dtype):
    """ortho_bound, with the sums' chain emulated where operands are held in 22 bits: the same multiples of
    its error (3 x, 8 standard deviations)."""
    if dtype == BF:
        return ortho_bound(g, want, dtype)
    d = emulate_chain(g) - want
    rms = lambda t, dim=None: (t * t).mean(dim, keepdim=dim is not None).sqrt()
    size = rms(d, 1) * rms(d, 0) / rms(d) + rms(d)
    return 3 * float(d.norm()) / float(want.norm()) + 2.0 ** -22, 24 * size + 2.0 ** -20 * want.abs()


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("m,n,count,sym,update", LAUNCHES, ids=LAUNCH_IDS)
def test_every_tile_size_at_its_edges(gpu_device, m, n, count, sym, update, dtype):
    lib = K._lib.load()
    assert [lib.fmoe_newton_schulz_tile(m, n, count, s) for s in (1, 0)] == [sym, update]
    mats = mixed(m, n, count, gpu_device, dtype)
    outs = orthogonalize(mats)
    for x, o in zip(mats, outs):
        want = exact(x)
        rel, tol = launch_bound(x, want, dtype)
        err = o.double() - want
        assert o.dtype == dtype and float(err.norm()) <= (rel + half(dtype)) * float(want.norm()), tuple(x.shape)
        assert (err.abs() <= tol + half(dtype) * (want.abs() + tol)).all(), tuple(x.shape)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("m,n,count,sym,update", LAUNCHES, ids=LAUNCH_IDS)
def test_muon_in_every_tile_size(gpu_device, m, n, count, sym, update, dtype):
    """The parameters' update in the last product's epilogue, tall and wide, bounds as above; memory
    between the parameters stays as it was."""
    lib = K._lib.load()
    assert [lib.fmoe_newton_schulz_tile(n, m, count, s) for s in (1, 0)] == [sym, update]
    lr, wd, mom = 0.03, 0.1, 0.9
    grads = mixed(m, n, count, gpu_device, dtype, 10)
    gap = 5
    store = torch.randn(count * (m * n + gap), generator=torch.Generator(gpu_device).manual_seed(1),
                        device=gpu_device).mul_(0.05).to(dtype)
    ps, gaps = [], []
    for i, g in enumerate(grads):
        o = i * (m * n + gap)
        ps.append(torch.nn.Parameter(store[o:o + m * n].view(g.shape)))
        gaps.append((store[o + m * n:o + m * n + gap], store[o + m * n:o + m * n + gap].clone()))
        ps[-1].grad = g
    opt = Muon(ps, lr=lr, weight_decay=wd, momentum=mom)
    bufs = [b.mul_(0.5) for b in mixed(m, n, count, gpu_device, dtype, 20)]
    before = [(p.detach().clone(), b.clone()) for p, b in zip(ps, bufs)]
    for p, b in zip(ps, bufs):
        opt.state[p]["momentum_buffer"] = b
    opt.step()
    for p, g, b, (p0, b0) in zip(ps, grads, bufs, before):
        want, buf, lr_, o, u = expect_step(p0, g, b0, lr, wd, mom, True, None)
        size = mom * b0.double().abs() + (1 - mom) * g.double().abs()
        assert ((b.double() - buf).abs() <= 4 * 2.0 ** -24 * size + half(dtype) * buf.abs() * (1 + 2.0 ** -20)).all()
        rms = float(o.norm()) / math.sqrt(o.numel())
        tol = lr_ * (launch_bound(u, o, dtype)[1] + 8 * 2.0 ** -20 * rms)
        tol = tol + 4 * 2.0 ** -24 * (p0.double().abs() + lr_ * o.abs())
        err = (p.detach().double() - want).abs()
        assert (err <= tol + half(dtype) * (want.abs() + tol)).all(), tuple(p.shape)
    assert all(torch.equal(x, y) for x, y in gaps)
