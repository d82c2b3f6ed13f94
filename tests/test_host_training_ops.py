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
    # one partial row pair per workgroup: 4 rows each below dim 1025, at most 4096 waves in all
    assert lib.fmoe_layer_norm_bwd_workspace_bytes(4, 64) == 2 * 64 * 4
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
