"""CPU tests of the training operators' host side: declared symbols, argument
checks before any GPU call, and the refusals of the Python entry points."""
import re
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import fusionllm_amd
from fusionllm_amd import LayerNorm, _lib, layer_norm

ROOT = Path(__file__).resolve().parents[1]
FAKE = 1 << 20  # a non-null address that is never dereferenced (rejected first)


def test_library_exports_the_training_symbols():
    lib = _lib.load()
    text = (ROOT / "include" / "fusiontrain.h").read_text()
    syms = set(re.findall(r"^\s*(?:int|size_t|const char\*)\s+(fmoe_\w+)\(", text, re.M))
    assert syms == set(_lib.TRAIN_SIGNATURES) and not syms & set(_lib.SIGNATURES)
    for s in syms:
        assert hasattr(lib, s), s


def test_layer_norm_argument_errors_without_gpu():
    lib = _lib.load()

    def fwd(x=FAKE, xd=1, ldx=64, w=FAKE, b=FAKE, wd=1, T=4, dim=64, y=FAKE, yd=1):
        return lib.fmoe_layer_norm_fwd(x, xd, ldx, w, b, wd, T, dim, 1e-5, y, yd, None, None, None)

    assert fwd(T=-1) == 1 and fwd(dim=0) == 1 and fwd(dim=-8) == 1
    assert fwd(dim=16385, ldx=1 << 20) == 2 and fwd(T=1 << 31) == 2
    assert fwd(ldx=63) == 2 and fwd(ldx=-64) == 2 and fwd(ldx=1 << 62) == 2  # overlapping rows, offsets beyond 63 bits
    assert fwd(xd=2) == 4 and fwd(yd=-1) == 4 and fwd(wd=7) == 4
    assert fwd(x=None) == 1 and fwd(y=None) == 1
    assert fwd(x=FAKE + 2) == 3 and fwd(y=FAKE + 1, yd=0) == 3 and fwd(w=FAKE + 2) == 3 and fwd(b=FAKE + 1) == 3
    assert fwd(T=0) == 0 and fwd(T=0, x=None, y=None) == 0

    def bwd(dy=FAKE, dyd=1, lddy=64, x=FAKE, xd=1, ldx=64, m=FAKE, w=FAKE, wd=1, T=4, dim=64, dx=FAKE, dw=FAKE,
            db=FAKE, ws=FAKE, n=1 << 20, res=None):
        return lib.fmoe_layer_norm_bwd(dy, dyd, lddy, x, xd, ldx, m, m, w, wd, res, T, dim, dx, dw, db, ws, n, None)

    assert bwd(T=-1) == 1 and bwd(dim=0) == 1 and bwd(dim=16385) == 2 and bwd(lddy=10) == 2 and bwd(ldx=10) == 2
    assert bwd(dyd=3) == 4 and bwd(xd=3) == 4 and bwd(wd=3) == 4
    assert bwd(n=lib.fmoe_layer_norm_bwd_workspace_bytes(4, 64) - 1) == 6 and bwd(ws=None) == 6
    assert bwd(dy=None) == 1 and bwd(x=None) == 1 and bwd(m=None) == 1
    assert bwd(dx=FAKE + 2) == 3 and bwd(dw=FAKE + 2) == 3 and bwd(db=FAKE + 1) == 3 and bwd(ws=FAKE + 2) == 3
    assert bwd(res=FAKE + 2) == 3 and bwd(m=FAKE + 1) == 3
    assert bwd(dx=None, dw=None, db=None) == 0  # nothing wanted
    # one partial row pair per workgroup: 4 rows each below dim 1025, at most 2048 waves in all (4096
    # where each has 16 rows)
    assert lib.fmoe_layer_norm_bwd_workspace_bytes(4, 64) == 2 * 64 * 4
    assert lib.fmoe_layer_norm_bwd_workspace_bytes(1 << 15, 768) == 512 * 2 * 768 * 4
    assert lib.fmoe_layer_norm_bwd_workspace_bytes(1 << 20, 768) == 1024 * 2 * 768 * 4
    assert lib.fmoe_layer_norm_bwd_workspace_bytes(1 << 20, 16384) == 256 * 2 * 16384 * 4
    assert lib.fmoe_layer_norm_bwd_workspace_bytes(0, 64) == lib.fmoe_layer_norm_bwd_workspace_bytes(4, 0) == 0


def test_layer_norm_refusals():
    with pytest.raises(RuntimeError, match="ROCm device"):
        layer_norm(torch.randn(4, 64))
    with pytest.raises(RuntimeError, match="ROCm device"):
        LayerNorm(64)(torch.randn(4, 64))
    with FakeTensorMode():
        x = torch.empty(4, 64, device="cuda")
        w = torch.empty(64, device="cuda")
        with pytest.raises(NotImplementedError, match="bf16 and fp32"):
            layer_norm(x.half())
        with pytest.raises(NotImplementedError, match="bf16 and fp32"):
            layer_norm(x, w.double(), w.double())
        with pytest.raises(NotImplementedError, match="one dtype"):
            layer_norm(x, w, w.bfloat16())
        with pytest.raises(ValueError, match="shape"):
            layer_norm(x, torch.empty(63, device="cuda"))
        with pytest.raises(ValueError, match="shape"):
            layer_norm(x, None, torch.empty(1, 64, device="cuda"))
        with pytest.raises(RuntimeError, match="input's device"):
            layer_norm(x, torch.empty(64))
        with pytest.raises(NotImplementedError, match="16384"):
            layer_norm(torch.empty(2, 16385, device="cuda"))
        with pytest.raises(NotImplementedError, match="16384"):
            layer_norm(torch.empty(2, 0, device="cuda"))
        with pytest.raises(ValueError, match="dimension"):
            layer_norm(torch.empty((), device="cuda"))


def test_layer_norm_module_interface():
    torch.manual_seed(0)
    a, b = LayerNorm(96, eps=1e-6), torch.nn.LayerNorm(96, eps=1e-6)
    assert isinstance(a, torch.nn.LayerNorm) and a.eps == b.eps
    assert {k: tuple(v.shape) for k, v in a.state_dict().items()} == {
        k: tuple(v.shape) for k, v in b.state_dict().items()}
    assert LayerNorm(96, bias=False).bias is None and LayerNorm(96, elementwise_affine=False).weight is None
    assert fusionllm_amd.LayerNorm is LayerNorm


def test_layer_norm_operator_fake_shapes():
    with FakeTensorMode():
        x = torch.empty(7, 96, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(96, device="cuda")
        y, mean, rstd = torch.ops.fusionllm.layer_norm_fwd(x, w, None, 1e-5, torch.float32)
        assert (y.shape, y.dtype) == ((7, 96), torch.float32)
        assert mean.shape == rstd.shape == (7,) and mean.dtype == rstd.dtype == torch.float32
        dx, dw = torch.ops.fusionllm.layer_norm_bwd(y, x, mean, rstd, w, None)
        assert (dx.shape, dx.dtype, dw.shape, dw.dtype) == ((7, 96), torch.bfloat16, (96,), torch.float32)


def _ns(lib, call="ortho", p=FAKE, rows=768, cols=2048, n=1, dtype=0, steps=5, co=(3.4445, -4.775, 2.0315), eps=1e-7,
        ws=FAKE, nbytes=None, second=None):
    import ctypes
    pp = _lib.ptr_array([p] * max(n, 1))
    good = _lib.ptr_array([FAKE] * max(n, 1))
    r = (ctypes.c_int64 * max(n, 1))(*[rows] * max(n, 1))
    c = (ctypes.c_int64 * max(n, 1))(*[cols] * max(n, 1))
    if second:
        r[1], c[1] = second
    if nbytes is None:
        nbytes = lib.fmoe_orthogonalize_workspace_bytes(rows, cols, n, dtype) - 1  # stops before the launches
    co = (ctypes.c_double * 3)(*co)
    if call == "ortho":
        return lib.fmoe_orthogonalize(pp, good, r, c, n, dtype, steps, co, eps, ws, nbytes, None)
    return lib.fmoe_muon_step(good, pp, good, r, c, n, dtype, 0.1, 0.1, 0.9, 0.95, 1, steps, co, eps, ws, nbytes,
                              None)


@pytest.mark.parametrize("call", ["ortho", "muon"])
def test_newton_schulz_argument_errors_without_gpu(call):
    lib = _lib.load()
    f = lambda **kw: _ns(lib, call, **kw)
    assert f() == 6 and f(ws=None) == 6 and f(nbytes=0) == 6  # admitted up to the workspace
    assert f(n=65) == 1 and f(n=-1) == 1 and f(n=0) == 0
    assert f(steps=0) == 1 and f(steps=65) == 1
    assert f(dtype=2) == 4 and f(p=None) == 1 and f(p=FAKE + 1) == 3 and f(p=FAKE + 2, dtype=1) == 3
    assert f(rows=0) == 1 and f(rows=-4) == 1 and f(cols=0) == 1 and f(cols=65537) == 2
    assert f(rows=16385, cols=32768, nbytes=0) == 2 and f(rows=16384, cols=32768, nbytes=0) == 6
    assert f(eps=0.0) == 1 and f(eps=-1.0) == 1 and f(eps=float("nan")) == 1
    # one pair of sides per call, in either order
    assert f(n=2, second=(2048, 768)) == 6 and f(n=2, second=(768, 2047)) == 2
    # coefficients: those of the literature's cubic and quintic stay in range, these do not
    assert f(co=(1.5, -0.5, 0.0), steps=20) == 6 and f(co=(2.0, -1.5, 0.5), steps=20) == 6
    assert f(steps=64) == 6
    assert f(co=(4.0, -4.775, 2.0315)) == 9 and f(co=(3.0, 0.0, 0.0)) == 9 and f(co=(8.0, -9.0, 1.5)) == 9
    assert f(co=(float("nan"), 0.0, 0.0)) == 9 and f(co=(float("inf"), 0.0, 0.0)) == 9
    assert b"coefficients" in lib.fmoe_status_string(9)


def test_newton_schulz_range_check_covers_the_iterates():
    # the host's bound of the singular values against the polynomial on a fine grid
    import numpy as np
    lib = _lib.load()
    rng = np.random.default_rng(0)
    admitted = 0
    for _ in range(400):
        a, b, c = rng.uniform(0.5, 4), rng.uniform(-6, 1), rng.uniform(-1, 4)
        s = np.linspace(0, 1, 20001)
        worst, poly = 1.0, 0.0
        for _ in range(5):
            t = s * s
            poly = max(poly, np.abs(a + b * t + c * t * t).max())
            s = np.abs(s * (a + t * (b + c * t)))
            s = np.linspace(0, s.max(), 20001)
            worst = max(worst, s.max())
            if worst > 1e3:
                break
        rc = _ns(lib, co=(a, b, c))
        if rc == 6:
            admitted += 1
            assert worst < 2.8 and poly < 7.9, (a, b, c)
        else:
            assert rc == 9 and (worst > 2.7 or poly > 7.7), (a, b, c)
    assert 20 < admitted < 380


def test_newton_schulz_workspace_size():
    lib = _lib.load()
    q = lib.fmoe_orthogonalize_workspace_bytes
    # partial sums; X twice, with an fp8 remainder once or (fp32 and small sides) lo twice; A and B with the
    # same lo; sides padded to 64
    assert q(768, 2048, 3, 0) == (3 * 64 * 8 + 255) // 256 * 256 + 3 * 2 * (5 * 768 * 2048 // 2 + 2 * 768 * 768)
    assert q(768, 2048, 3, 1) == (3 * 64 * 8 + 255) // 256 * 256 + 3 * 2 * (4 * 768 * 2048 + 4 * 768 * 768)
    assert q(2048, 768, 3, 0) == q(768, 2048, 3, 0)
    assert q(65, 70, 1, 0) == 256 + 2 * (4 * 128 * 128 + 4 * 128 * 128)
    # small sides: per panel of 128 columns the norm, the exponent, X and two partial Gram matrices
    assert q(5, 129, 3, 0) == 256 + 256 + 3 * 2 * 4 * (64 * 128 + 2 * 10 * 256)
    assert q(64, 4097, 1, 0) > 4 * 2 * 64 * 4096  # 33 panels: the general form
    assert q(0, 5, 1, 0) == q(5, 5, 0, 0) == q(5, 5, 65, 0) == q(65537, 5, 1, 0) == q(16385, 32768, 1, 0) == 0


def test_muon_and_orthogonalize_refusals():
    from fusionllm_amd.optim import Muon, orthogonalize
    P = torch.nn.Parameter
    with pytest.raises(ValueError, match="matrices"):
        Muon([P(torch.zeros(4))])
    with pytest.raises(ValueError, match="matrices"):
        Muon([P(torch.zeros(2, 2, 2))])
    p = P(torch.zeros(4, 4))
    with pytest.warns(UserWarning), pytest.raises(ValueError, match="twice"):
        Muon([p, p])
    for kw in (dict(lr=-1.0), dict(weight_decay=-0.1), dict(momentum=1.0), dict(momentum=-0.1), dict(eps=0.0),
               dict(ns_steps=0), dict(ns_steps=65), dict(ns_coefficients=(1.0, 2.0)), dict(adjust_lr_fn="other")):
        with pytest.raises(ValueError):
            Muon([p], **kw)
    opt = Muon([p])
    assert opt.defaults["ns_steps"] == 5 and opt.defaults["lr"] == 1e-3 and opt.defaults["momentum"] == 0.95
    opt.step()  # no gradient: nothing to do
    p.grad = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="ROCm device"):
        opt.step()
    with pytest.raises(RuntimeError, match="ROCm device"):
        orthogonalize(torch.zeros(4, 4))
    with pytest.raises(ValueError, match="matrices"):
        orthogonalize(torch.zeros(4))
    with pytest.raises(ValueError, match="steps"):
        orthogonalize(torch.zeros(4, 4), steps=0)
    with FakeTensorMode():
        x = torch.empty(4, 6, device="cuda")
        with pytest.raises(NotImplementedError, match="bf16 and fp32"):
            orthogonalize(x.half())
        with pytest.raises(RuntimeError, match="no backward"):
            orthogonalize(x.requires_grad_())
        with pytest.raises(NotImplementedError, match="65536"):
            orthogonalize(torch.empty(2, 65537, device="cuda"))
        with pytest.raises(NotImplementedError, match="elements"):
            orthogonalize(torch.empty(16385, 32768, device="cuda"))


def test_training_kernels_read_no_register_a_load_is_still_filling():
    # The Newton-Schulz products issue their global -> LDS copies (and, in 256 x 256 tiles, their
    # MFMAs) from inline assembly with explicit waits, which the compiler does not see.
    from tests import isa_check as ic
    build = ROOT / "fusionllm_amd" / "_build"
    objs = [build / "newton_schulz.o", build / "layer_norm.o"]
    if not (ic.ROCM_LLVM / "llvm-objdump").exists() or not all(o.exists() for o in objs):
        pytest.skip("no built objects or no llvm-objdump")
    checked = 0
    for o in objs:
        n, hazards = ic.check_object(o)
        assert not hazards, "\n".join(hazards[:10])
        checked += n
    assert checked >= 80


def test_training_kernels_keep_their_values_in_registers(tmp_path):
    # A product that needs scratch memory pays for it in every tile, a norm in every row.
    import shutil
    import subprocess

    from fusionllm_amd import build
    from tests import isa_check as ic
    if not ic.ROCM_LLVM.exists():
        pytest.skip("no LLVM tools here")
    seen = 0
    for name in ("newton_schulz", "layer_norm"):
        obj = build.BUILD_DIR / f"{name}.o"
        if not obj.exists():
            pytest.skip("no built objects")
        work = tmp_path / name
        work.mkdir()
        shutil.copy(obj, work / obj.name)
        subprocess.run([str(ic.ROCM_LLVM / "llvm-objdump"), "--offloading", obj.name], check=True,
                       capture_output=True, cwd=work)
        dev = next(p for p in work.iterdir() if "gfx950" in p.name)
        notes = subprocess.run([str(ic.ROCM_LLVM / "llvm-readelf"), "--notes", str(dev)], check=True,
                               capture_output=True, text=True).stdout
        for entry in notes.split("  - .agpr_count:")[1:]:
            kernel = re.search(r"\.name:\s+(\S+)", entry).group(1)
            seen += 1
            spilled = int(re.search(r"\.vgpr_spill_count:\s*(\d+)", entry).group(1))
            # the backward of bf16 rows of two chunks per lane is one register over
            assert spilled <= (1 if "layer_norm_bwd" in kernel else 0), kernel
    assert seen >= 80


def test_muon_has_torchs_constructor():
    import inspect

    from fusionllm_amd.optim import Muon
    if not hasattr(torch.optim, "Muon"):
        pytest.skip("this torch has no Muon")
    args = lambda cls: [(p.name, p.default) for p in inspect.signature(cls).parameters.values()]
    assert args(Muon) == args(torch.optim.Muon)
    p = torch.nn.Parameter(torch.zeros(2, 3))
    assert Muon([p]).defaults == torch.optim.Muon([p]).defaults


def _order(params, **kw):
    """Launches that ``_launches`` forms of Muon-like items, as lists of their indices."""
    from fusionllm_amd import optim
    items = [(p, torch.empty_like(p), torch.empty_like(p)) for p in params]
    at = {id(it): i for i, it in enumerate(items)}
    return [[at[id(it)] for it in chunk] for chunk in optim._launches(items, lambda it: (it[0], it[2]), **kw)]


def test_overlapping_matrices_keep_their_order_whatever_their_sides():
    t = torch.zeros(60, 96)
    # rows 15 .. 44 overlap the rows before and after, which have other sides than they
    assert _order([t[:20], t[15:45], t[40:60]]) == [[0], [1], [2]]
    flat = torch.zeros(200)
    assert _order([flat[:64].view(4, 16), flat[32:160].view(8, 16), flat[128:192].view(4, 16)]) == [[0], [1], [2]]
    # of another dtype too: the same memory
    as_bf16 = torch.zeros(64).view(torch.bfloat16).view(4, 32)
    assert _order([as_bf16.view(torch.float32), as_bf16, torch.zeros(4, 16)]) == [[0, 2], [1]]
    # what does not overlap goes together, whatever stands between
    assert _order([t[:20], torch.zeros(8, 8), t[20:40], torch.zeros(8, 8), t[40:60]]) == [[0, 2, 4], [1, 3]]
    assert _order([t[:20], t[:20], t[20:40]]) == [[0], [1, 2]]
    # and in order around an overlap of two others
    u = torch.zeros(40, 30)
    assert _order([t[:20], u[:30], u[10:], t[20:40], t[10:30]]) == [[0, 3], [1], [2], [4]]


def test_launches_keep_the_order_of_every_overlapping_pair():
    # random views of one storage, a few sides: each pair that overlaps is launched in order, never together
    import random
    rng = random.Random(0)
    for trial in range(200):
        base = torch.zeros(400)
        params = []
        for _ in range(rng.randint(2, 14)):
            r, c = rng.choice([(2, 8), (4, 16), (8, 2), (5, 10)])
            o = rng.randint(0, 400 - r * c)
            params.append(base[o:o + r * c].view(r, c))
        chunks = _order(params)
        assert sorted(i for c in chunks for i in c) == list(range(len(params)))
        where = {i: k for k, c in enumerate(chunks) for i in c}
        span = lambda p: (p.storage_offset(), p.storage_offset() + p.numel())
        for i, p in enumerate(params):
            for j in range(i):
                (a, b), (c, d) = span(p), span(params[j])
                if a < d and c < b:
                    assert where[j] < where[i], (trial, j, i)


def test_a_gradient_on_anothers_memory_is_read_in_order():
    # matrix 1's gradient is matrix 0's memory: it is read after matrix 0 was written, and before matrix 2,
    # whose memory matrix 1's gradient is no part of, nothing is between
    from fusionllm_amd import optim
    new = lambda: torch.zeros(4, 16)
    p, q, r = new(), new(), new()
    items = [(p, new(), new()), (q, p, new()), (r, new(), new())]
    chunks = optim._launches(items, lambda it: (it[0], it[2]), lambda it: (it[1],))
    assert [len(c) for c in chunks] == [1, 2] and chunks[1][0] is items[1]
    # read first, written by a later one
    items = [(q, p, new()), (p, new(), new())]
    assert [len(c) for c in optim._launches(items, lambda it: (it[0], it[2]), lambda it: (it[1],))] == [1, 1]
    # one gradient of two matrices is only read
    g = new()
    items = [(p, g, new()), (q, g, new())]
    assert [len(c) for c in optim._launches(items, lambda it: (it[0], it[2]), lambda it: (it[1],))] == [2]


def test_coefficients_are_checked_on_the_host_and_by_the_constructor():
    from fusionllm_amd.optim import Muon
    lib = _lib.load()
    import ctypes
    f = lambda *co, steps=5: lib.fmoe_newton_schulz_check(steps, (ctypes.c_double * 3)(*co))
    good = (3.4445, -4.775, 2.0315)
    assert f(*good) == 0 and f(*good, steps=64) == 0 and f(1.5, -0.5, 0.0, steps=20) == 0
    assert f(*good, steps=0) == 1 and f(*good, steps=65) == 1 and lib.fmoe_newton_schulz_check(5, None) == 1
    assert f(4.0, -4.775, 2.0315) == 9 and f(float("nan"), 0.0, 0.0) == 9
    P = lambda: torch.nn.Parameter(torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match="coefficients"):
        Muon([P()], ns_coefficients=(8.0, -9.0, 1.5))
    # a group's own values too, and the group is not taken
    opt = Muon([P()])
    for own, error in ((dict(ns_coefficients=(8.0, -9.0, 1.5)), RuntimeError), (dict(ns_steps=0), ValueError),
                       (dict(eps=0.0), ValueError), (dict(ns_coefficients=(1.0,)), ValueError)):
        with pytest.raises(error):
            opt.add_param_group({"params": [P()], **own})
        assert len(opt.param_groups) == 1


def test_muon_checks_every_group_before_it_updates_any(monkeypatch):
    # what a second group is refused for leaves the first one's parameters and state alone
    from fusionllm_amd import optim
    from fusionllm_amd.optim import Muon
    launched = []
    monkeypatch.setattr(optim.K, "muon_step", lambda *a: launched.append(a))

    def make(shape=(4, 6), dtype=torch.float32, device="cuda"):
        p = torch.nn.Parameter(torch.empty(shape, dtype=dtype, device=device))
        p.grad = torch.empty(shape, dtype=dtype, device=device)
        return p

    def bad_buffer(opt, p, buf):
        opt.state[p]["momentum_buffer"] = buf

    cases = [
        (lambda opt, p: bad_buffer(opt, p, torch.empty(6, 4, device="cuda").t()), RuntimeError, "contiguous"),
        (lambda opt, p: bad_buffer(opt, p, torch.empty(4, 6, device="cuda", dtype=torch.bfloat16)), RuntimeError,
         "momentum"),
        (lambda opt, p: bad_buffer(opt, p, torch.empty(4, 6, device="cpu")), RuntimeError, "momentum"),
        (lambda opt, p: bad_buffer(opt, p, torch.empty(4, 5, device="cuda")), RuntimeError, "momentum"),
        (lambda opt, p: opt.param_groups[1].update(ns_coefficients=(8.0, -9.0, 1.5)), RuntimeError, "coefficients"),
        (lambda opt, p: opt.param_groups[1].update(ns_steps=0), ValueError, "steps"),
        (lambda opt, p: opt.param_groups[1].update(eps=-1.0), ValueError, "eps"),
    ]
    with FakeTensorMode():
        for spoil, error, match in cases:
            first, second = make(), make()
            opt = Muon([{"params": [first]}, {"params": [second]}])
            spoil(opt, second)
            with pytest.raises(error, match=match):
                opt.step()
            assert not launched and first not in opt.state, match
        for shape, dtype, device, error in (((4, 6), torch.float16, "cuda", NotImplementedError),
                                            ((4, 6), torch.float32, "cpu", RuntimeError),
                                            ((2, 65537), torch.float32, "cuda", NotImplementedError)):
            first, second = make(), make(shape, dtype, device)
            opt = Muon([{"params": [first]}, {"params": [second]}])
            with pytest.raises(error):
                opt.step()
            assert not launched and first not in opt.state and second not in opt.state


def test_muon_refuses_to_create_momentum_in_a_capture(monkeypatch):
    # the captured zeros would clear the momentum in every replay
    from fusionllm_amd import optim
    from fusionllm_amd.optim import Muon
    launched = []
    monkeypatch.setattr(optim.K, "muon_step", lambda *a: launched.append(a))
    with FakeTensorMode():
        ps = [torch.nn.Parameter(torch.empty(4, 6, device="cuda")) for _ in range(2)]
        for p in ps:
            p.grad = torch.empty(4, 6, device="cuda")
        opt = Muon(ps)
        opt.state[ps[0]]["momentum_buffer"] = torch.empty(4, 6, device="cuda")
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="captur"):
            opt.step()
        assert not launched and ps[1] not in opt.state
        ps[1].grad = None  # every matrix of this step has its momentum
        monkeypatch.setattr(optim, "_launches", lambda items, *a: [items])
        monkeypatch.setattr(torch.cuda, "device", lambda d: __import__("contextlib").nullcontext())
        opt.step()
        assert len(launched) == 1


def _duals(n, *tensors):
    """The tensors, the n-th of them with a tangent (inside a dual level)."""
    import torch.autograd.forward_ad as fw
    return [fw.make_dual(t, torch.ones_like(t)) if i == n else t for i, t in enumerate(tensors)]


def test_forward_mode_derivatives_are_refused():
    # not lost without a word: a tensor with a tangent need not require a gradient
    import torch.autograd.forward_ad as fw

    from fusionllm_amd import DeepSeekMoE, moe_residual
    from fusionllm_amd.optim import orthogonalize
    with FakeTensorMode(), torch.device("cuda"):
        x, w, b = torch.empty(4, 64), torch.empty(64), torch.empty(64)
        moe = DeepSeekMoE(dict(dim=64, n_routed_experts=4, n_shared_experts=1, n_activated_experts=2,
                               moe_inter_dim=64)).requires_grad_(False)
        norm = LayerNorm(64).requires_grad_(False)
        with fw.dual_level():
            for i in range(3):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    layer_norm(*_duals(i, x, w, b))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.func.functional_call(norm, {"bias": _duals(0, b)[0]}, x)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                moe_residual(_duals(0, x)[0], norm, moe)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                moe(_duals(0, x)[0])
            with pytest.raises(NotImplementedError, match="forward-mode"):
                orthogonalize(_duals(0, x)[0])
            with pytest.raises(NotImplementedError, match="forward-mode"):
                orthogonalize([x, _duals(0, x)[0]])


def test_moe_residual_fuses_only_what_it_knows(monkeypatch):
    """A norm or a block with a forward of its own, or with hooks, is called; the fused form would pass it by."""
    from torch.nn.modules import module as nnm

    from fusionllm_amd import DeepSeekMoE, moe_residual

    fused = []
    monkeypatch.setattr(DeepSeekMoE, "forward_norm_residual", lambda self, x, norm: fused.append(norm) or x)
    monkeypatch.setattr(DeepSeekMoE, "forward", lambda self, x: x)
    for cls in (LayerNorm, torch.nn.RMSNorm):
        monkeypatch.setattr(cls, "forward", lambda self, x: x)
    cfg = dict(dim=64, n_routed_experts=4, n_shared_experts=1, n_activated_experts=2, moe_inter_dim=64)

    class Own(LayerNorm):
        def forward(self, x):
            return 2 * x

    class OwnRMS(torch.nn.RMSNorm):
        def forward(self, x):
            return 2 * x

    class OwnMoE(DeepSeekMoE):
        def forward(self, x):
            return 2 * x

    class Named(LayerNorm):
        pass

    with FakeTensorMode(), torch.device("cuda"):
        x = torch.empty(4, 64)

        def takes(norm, moe):
            del fused[:]
            moe_residual(x, norm, moe)
            return bool(fused)

        moe = DeepSeekMoE(cfg)
        assert takes(LayerNorm(64), moe) and takes(torch.nn.RMSNorm(64), moe) and takes(Named(64), moe)
        assert not takes(torch.nn.LayerNorm(64), moe)
        assert not takes(Own(64), moe) and not takes(OwnRMS(64), moe) and not takes(LayerNorm(64), OwnMoE(cfg))
        for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook",
                         "register_full_backward_pre_hook"):
            for cls in (LayerNorm, torch.nn.RMSNorm):
                norm = cls(64)
                handle = getattr(norm, register)(lambda *a: None)
                assert not takes(norm, moe), register
                handle.remove()
                assert takes(norm, moe), register
            handle = getattr(moe, register)(lambda *a: None)
            assert not takes(LayerNorm(64), moe), register
            handle.remove()
        for register in (nnm.register_module_forward_hook, nnm.register_module_forward_pre_hook):
            handle = register(lambda *a: None)
            assert not takes(LayerNorm(64), moe)
            handle.remove()
        # a forward put on the instance
        norm = LayerNorm(64)
        norm.forward = lambda t: 2 * t
        assert not takes(norm, moe)


def test_tiles_of_a_launch():
    # the shapes by which the GPU tests reach every tile size; both sides of the rule
    tile = _lib.load().fmoe_newton_schulz_tile
    for m, n, count, sym, update in [(700, 1030, 27, 256, 256), (700, 1030, 10, 128, 128), (400, 600, 56, 256, 256),
                                     (1400, 1500, 24, 256, 256), (320, 450, 64, 128, 256), (321, 449, 20, 64, 128),
                                     (700, 1030, 3, 64, 64)]:
        assert (tile(m, n, count, 1), tile(m, n, count, 0)) == (sym, update) == (tile(n, m, count, 1), tile(n, m, count, 0))
    assert tile(64, 4096, 64, 1) == 0 and tile(64, 4097, 1, 1) == 64  # the form of small sides
    assert tile(0, 5, 1, 0) == tile(5, 5, 65, 0) == tile(65537, 5, 1, 0) == tile(16385, 32768, 1, 0) == 0


def test_training_kernels_without_scratch_memory(tmp_path):
    # none but the backward of bf16 rows of two chunks per lane, which keeps one register of its 128 there
    import shutil
    import subprocess

    from fusionllm_amd import build
    from tests import isa_check as ic
    if not ic.ROCM_LLVM.exists():
        pytest.skip("no LLVM tools here")
    scratch = {}
    for name in ("newton_schulz", "layer_norm"):
        obj = build.BUILD_DIR / f"{name}.o"
        if not obj.exists():
            pytest.skip("no built objects")
        work = tmp_path / name
        work.mkdir()
        shutil.copy(obj, work / obj.name)
        subprocess.run([str(ic.ROCM_LLVM / "llvm-objdump"), "--offloading", obj.name], check=True,
                       capture_output=True, cwd=work)
        dev = next(p for p in work.iterdir() if "gfx950" in p.name)
        notes = subprocess.run([str(ic.ROCM_LLVM / "llvm-readelf"), "--notes", str(dev)], check=True,
                               capture_output=True, text=True).stdout
        for entry in notes.split("  - .agpr_count:")[1:]:
            kernel = re.search(r"\.name:\s+_ZN4fmoe\d+(\w+)", entry).group(1)
            value = lambda key: int(re.search(rf"\.{key}:\s*(\d+)", entry).group(1))
            if value("private_segment_fixed_size") or value("vgpr_spill_count"):
                scratch[kernel] = (value("private_segment_fixed_size"), value("vgpr_spill_count"))
    # x bf16, dy bf16 or fp32, chunks of 8, two per lane
    assert {k.split("EEEv")[0] for k in scratch} <= {"layer_norm_bwd_kernelILi0ELi0ELi8ELi2",
                                                     "layer_norm_bwd_kernelILi0ELi1ELi8ELi2"}
    assert all(size <= 8 and spilled <= 1 for size, spilled in scratch.values())
