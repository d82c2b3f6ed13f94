"""CPU tests of the vocabulary operators' host side: declared symbols, argument checks before any GPU call,
the refusals of the Python entry points, operator shapes, and the machine code."""
import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import fusionllm_amd
from fusionllm_amd import Embedding, _lib, embedding, linear_cross_entropy, linear_distillation
from fusionllm_amd import _kernels as K

ROOT = Path(__file__).resolve().parents[1]
FAKE = 1 << 20  # a non-null address that is never dereferenced (rejected first)


def test_library_exports_the_vocabulary_symbols():
    lib = _lib.load()
    text = (ROOT / "include" / "fusionvocab.h").read_text()
    syms = set(re.findall(r"^\s*(?:int|size_t)\s+(fmoe_\w+)\(", text, re.M))
    assert syms == set(_lib.VOCAB_SIGNATURES)
    assert not syms & (set(_lib.SIGNATURES) | set(_lib.TRAIN_SIGNATURES))
    for s in syms:
        assert hasattr(lib, s), s


def test_embedding_argument_errors_without_gpu():
    lib = _lib.load()

    def fwd(ids=FAKE, i64=1, w=FAKE, dt=1, ldw=64, T=4, V=10, d=64, y=FAKE):
        return lib.fmoe_embedding_fwd(ids, i64, w, dt, ldw, T, V, d, 1.0, y, None)

    assert fwd(T=-1) == 1 and fwd(V=0) == 1 and fwd(d=0) == 1 and fwd(i64=2) == 1
    assert fwd(d=16385, ldw=1 << 20) == 2 and fwd(T=(1 << 24) + 1) == 2 and fwd(V=(1 << 24) + 1) == 2
    assert fwd(ldw=63) == 2 and fwd(ldw=1 << 40) == 2
    assert fwd(T=1 << 24, d=1024, ldw=1024) == 2 and fwd(V=1 << 24, d=1024, ldw=1024) == 2  # too many elements
    assert fwd(dt=2) == 4 and fwd(ids=None) == 1 and fwd(w=None) == 1 and fwd(y=None) == 1
    assert fwd(ids=FAKE + 4) == 3 and fwd(ids=FAKE + 2, i64=0) == 3 and fwd(w=FAKE + 2) == 3 and fwd(y=FAKE + 1, dt=0) == 3
    assert fwd(T=0) == 0 and fwd(T=0, ids=None, w=None, y=None) == 0

    size = lib.fmoe_embedding_bwd_workspace_bytes(100, 10, 64)

    def bwd(ids=FAKE, i64=1, dy=FAKE, dyt=1, ld=64, T=100, V=10, d=64, pad=-1, dw=FAKE, dt=1, ws=FAKE, n=size):
        return lib.fmoe_embedding_bwd(ids, i64, dy, dyt, ld, T, V, d, 1.0, pad, dw, dt, ws, n, None)

    assert bwd(T=-1) == 1 and bwd(pad=10) == 1 and bwd(pad=-2) == 1 and bwd(dw=None) == 1 and bwd(dy=None) == 1
    assert bwd(ld=63) == 2 and bwd(dyt=5) == 4 and bwd(dt=5) == 4
    assert bwd(n=size - 1) == 6 and bwd(ws=None) == 6 and bwd(ws=FAKE + 16) == 3 and bwd(dw=FAKE + 2) == 3
    # slot starts (512 slots and the end), sorted tokens, two partial rows a tile of 16; none up to 64 tokens
    assert size == 513 * 4 // 256 * 256 + 256 + 1024 + 7 * 2 * 64 * 4
    assert lib.fmoe_embedding_bwd_workspace_bytes(64, 10, 64) == 0
    assert bwd(T=64, ws=FAKE + 16, n=0) == 3 and bwd(T=64, ws=None, n=0, dw=None) == 1
    assert lib.fmoe_embedding_bwd_workspace_bytes(-1, 10, 64) == lib.fmoe_embedding_bwd_workspace_bytes(4, 0, 64) == 0


def test_loss_argument_errors_without_gpu():
    lib = _lib.load()
    state = lib.fmoe_vocab_loss_state_bytes(4, 64, 1, 1)
    fws = lib.fmoe_vocab_loss_fwd_workspace_bytes(4, 64, 100, 1, 1, 0)
    bws = lib.fmoe_vocab_loss_bwd_workspace_bytes(4, 64, 100, 1, 0)
    assert state > 0 and fws > 0 and bws > 0

    def fwd(h=FAKE, ht=0, ldh=64, w=FAKE, wt=0, ldw=64, i=FAKE, i64=1, t=None, tt=1, T=4, d=64, V=100, top=1,
            scale=1.0, temp=1.0, planes=1, red=1, loss=FAKE, st=FAKE, sn=state, ws=FAKE, wn=fws):
        return lib.fmoe_vocab_loss_fwd(h, ht, ldh, w, wt, ldw, i, i64, t, tt, T, d, V, top, -100, scale, temp, planes,
                                       red, loss, st, sn, ws, wn, None)

    assert fwd(T=-1) == 1 and fwd(d=0) == 1 and fwd(V=0) == 1 and fwd(top=0) == 1 and fwd(red=3) == 1 and fwd(planes=2) == 1
    assert fwd(temp=0.0) == 1 and fwd(temp=float("nan")) == 1 and fwd(temp=2.0) == 1 and fwd(i64=-1) == 1
    assert fwd(top=5) == 1  # a list without a teacher
    assert fwd(d=16385, ldh=1 << 15, ldw=1 << 15) == 2 and fwd(top=1025, t=FAKE) == 2 and fwd(V=(1 << 24) + 1) == 2
    assert fwd(ldh=63) == 2 and fwd(ldw=63) == 2 and fwd(ldw=1 << 22) == 2
    assert fwd(ht=2) == 4 and fwd(wt=2) == 4 and fwd(t=FAKE, tt=7) == 4 and fwd(planes=3) == 4
    assert fwd(planes=3, ht=1) == 4 and fwd(planes=3, wt=1) == 4
    assert fwd(h=None) == 1 and fwd(w=None) == 1 and fwd(i=None) == 1 and fwd(loss=None) == 1
    assert fwd(h=FAKE + 1) == 3 and fwd(w=FAKE + 1) == 3 and fwd(i=FAKE + 4) == 3 and fwd(loss=FAKE + 2) == 3
    assert fwd(st=FAKE + 8) == 3 and fwd(ws=FAKE + 8) == 3
    assert fwd(sn=state - 1) == 6 and fwd(wn=fws - 1) == 6 and fwd(st=None) == 6 and fwd(ws=None) == 6

    def bwd(dl=FAKE, w=FAKE, wt=0, ldw=64, T=4, d=64, V=100, top=1, dis=0, temp=1.0, planes=1, red=1, st=FAKE, sn=state,
            dh=FAKE, dht=0, dw=FAKE, dwt=0, ws=FAKE, wn=bws):
        return lib.fmoe_vocab_loss_bwd(dl, w, wt, ldw, T, d, V, top, dis, 1.0, temp, planes, red, st, sn, dh, dht, dw, dwt,
                                       ws, wn, None)

    assert bwd(T=-1) == 1 and bwd(top=2) == 1 and bwd(dis=2) == 1 and bwd(temp=2.0) == 1 and bwd(red=-1) == 1
    assert bwd(dl=None) == 1 and bwd(w=None) == 1
    assert bwd(ldw=10) == 2 and bwd(wt=3) == 4 and bwd(dht=3) == 4 and bwd(dwt=3) == 4 and bwd(planes=3) == 4
    assert bwd(dl=FAKE + 2) == 3 and bwd(dh=FAKE + 1) == 3 and bwd(dw=FAKE + 1) == 3 and bwd(st=FAKE + 4) == 3
    assert bwd(sn=state - 1) == 6 and bwd(wn=bws - 1) == 6 and bwd(ws=None) == 6
    assert bwd(dh=None, dw=None) == 0  # nothing wanted
    for a in [(-1, 64, 1, 1), (4, 0, 1, 1), (4, 64, 0, 1), (4, 64, 1, 2), (4, 64, 1025, 1)]:
        assert lib.fmoe_vocab_loss_state_bytes(*a) == 0


def test_gradients_at_once_and_scale_argument_errors_without_gpu():
    lib = _lib.load()
    ws = lib.fmoe_vocab_loss_grad_workspace_bytes(100, 64, 100, 1, 1, 0)

    def call(h=FAKE, T=100, V=100, d=64, top=1, red=1, planes=1, loss=FAKE, dh=FAKE, dht=0, dw=FAKE, dwt=0, w=FAKE,
             n=ws, t=None):
        return lib.fmoe_vocab_loss_fwd_grad(h, 0, 64, FAKE, 0, 64, FAKE, 1, t, 1, T, d, V, top, -100, 1.0, 1.0, planes,
                                            red, loss, dh, dht, dw, dwt, w, n, None)

    assert call(red=0) == 1 and call(T=-1) == 1 and call(loss=None) == 1 and call(h=None) == 1 and call(planes=3) == 4
    assert call(dht=2) == 4 and call(dwt=-1) == 4 and call(dh=FAKE + 1) == 3 and call(dw=FAKE + 1) == 3 and call(w=FAKE + 1) == 3
    assert call(T=64) == 2 and call(n=ws - 1) == 6 and call(w=None) == 6 and call(top=3) == 1

    def scale(f=FAKE, a=FAKE, b=FAKE, dt=1, n=4, count=1):
        one = lambda kind, v: (kind * 1)(v)
        return lib.fmoe_scale(f, one(ctypes.c_void_p, a), one(ctypes.c_void_p, b), one(ctypes.c_int, dt),
                              one(ctypes.c_int64, n), count, None)

    assert scale(n=-1) == 1 and scale(dt=9) == 4 and scale(f=None) == 1 and scale(a=None) == 1 and scale(b=None) == 1
    assert scale(f=FAKE + 2) == 3 and scale(a=FAKE + 2) == 3 and scale(b=FAKE + 1, dt=0) == 3 and scale(n=0, a=None) == 0
    assert scale(count=9) == 1 and scale(count=-1) == 1 and scale(count=0, f=None) == 0


def test_calls_without_rows_are_not_refused_for_their_missing_teacher():
    # an empty tensor has no address, so nothing tells a distillation of no rows, lists of one, from cross entropy: its
    # temperature passes the check of arguments (the workspace that is too small is what comes next, before any launch)
    lib = _lib.load()
    state = lib.fmoe_vocab_loss_state_bytes(0, 64, 1, 1)

    def fwd(T, top, temp, teacher):
        return lib.fmoe_vocab_loss_fwd(None, 0, 64, FAKE, 0, 64, None, 1, teacher, 1, T, 64, 100, top, -100, 1.0, temp, 1, 1,
                                       FAKE, FAKE, state, FAKE, 0, None)

    for top in (1, 2, 7):
        for temp in (1.0, 2.0, 0.5):
            for teacher in (None, FAKE):
                assert fwd(0, top, temp, teacher) == 6, (top, temp, teacher)
            assert fwd(0, top, -temp, None) == 1
    assert fwd(1, 1, 2.0, None) == 1


def test_state_size_is_the_librarys():
    lib = _lib.load()
    for a in [(0, 1, 1, 1), (1, 1, 1, 1), (5, 7, 3, 3), (64, 64, 64, 1), (65, 65, 1, 3), (16384, 768, 1, 1),
              (4096, 2048, 1000, 3)]:
        assert lib.fmoe_vocab_loss_state_bytes(*a) == K.vocab_loss_state_bytes(*a), a


def test_rule_of_gradients_at_once_is_the_librarys():
    lib = _lib.load()
    taken = 0
    for T in (0, 1, 64, 65, 256, 257, 2000, 2049, 5000, 32768, 100000):
        for V in (1, 255, 257, 32768, 50021, 131072, 262145, 1 << 22, (1 << 22) + 1):
            for d in (1, 768, 2048, 4096):
                for planes in (1, 3):
                    for packs in (0, 1):
                        want = lib.fmoe_vocab_loss_grad_workspace_bytes(T, d, V, 1, planes, packs) > 0
                        assert K.vocab_loss_takes_gradients(T, d, V, planes, packs) == want, (T, V, d, planes, packs)
                        taken += want
    assert 0 < taken < 11 * 9 * 4 * 4


def test_workspaces_stay_bounded():
    # no logits: a piece of the vocabulary in bf16 (2 GiB), partial tiles (256 MiB), the sum of d_hidden between pieces
    lib = _lib.load()
    n = lib.fmoe_vocab_loss_bwd_workspace_bytes(32768, 2048, 131072, 1, 0)
    assert n <= (1 << 31) + (1 << 28) + 32768 * 2048 * 4 + 1024
    assert n < 32768 * 131072 * 2 // 3
    # the forward's: a maximum and a sum per row and 128 columns
    assert lib.fmoe_vocab_loss_fwd_workspace_bytes(32768, 2048, 131072, 1, 1, 0) <= 32768 * 1024 * 8 + (1 << 18)
    # gradients at once: a piece of 8192 rows, d_weight's sum, partial tiles, packed and scaled rows
    n = lib.fmoe_vocab_loss_grad_workspace_bytes(32768, 2048, 131072, 1, 1, 0)
    assert 0 < n <= (1 << 31) + 131072 * 2048 * 4 + (1 << 28) + 33792 * 2048 * 2 + 8192 * (2048 * 2 + 1024 * 8) + (1 << 20)
    # not for few rows, nor vocabularies whose pieces would have few rows
    assert lib.fmoe_vocab_loss_grad_workspace_bytes(64, 2048, 131072, 1, 1, 0) == 0
    assert lib.fmoe_vocab_loss_grad_workspace_bytes(32768, 2048, 600000, 1, 1, 0) == 0
    assert lib.fmoe_vocab_loss_grad_workspace_bytes(1000, 2048, 600000, 1, 1, 0) > 0
    # rows that the products read as they lie
    assert lib.fmoe_vocab_loss_packs(FAKE, 0, 128, 128, 1) == 0
    for w, dt, ld, d, planes in [(FAKE + 2, 0, 128, 128, 1), (FAKE, 1, 128, 128, 1), (FAKE, 0, 129, 128, 1),
                                 (FAKE, 0, 128, 100, 1), (FAKE, 1, 128, 128, 3)]:
        assert lib.fmoe_vocab_loss_packs(w, dt, ld, d, planes) == 1


def test_workspaces_hold_the_logits_of_few_rows():
    # the forward of up to 64 rows (up to 32, or 64 where the weight is copied or small) stores a long list's logits: whole
    # rows of 256-column tiles in fp32, for every row of the call
    lib = _lib.load()
    stored = 0
    for V in (5, 1000, 131071, 131072, 262143, 262144, 262145, 262208, 300001, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, 1 << 22):
        tiles = (V + 255) // 256
        for T in (1, 2, 7, 8, 31, 32, 33, 50, 63, 64):
            for planes, packs in ((1, 0), (1, 1), (3, 1)):
                size = lambda top: lib.fmoe_vocab_loss_fwd_workspace_bytes(T, 64, V, top, planes, packs)
                thin = T <= 32 or packs or tiles < 512
                for top in (5, 8, 1024):
                    more = size(top) - size(1)
                    if thin and V <= 1 << 20:
                        assert T * tiles * 1024 <= more < T * tiles * 1024 + 512, (T, V, planes, packs, top)
                        stored += 1
                    else:
                        assert more == 0, (T, V, planes, packs, top)
                assert size(4) == size(1)
    assert stored > 500
    # more rows: parts of at most 256 MiB, of whole row tiles, or all of the rows
    for T, V, top in ((65, 600, 900), (300, 32768, 256), (1500, 60000, 800), (1024, 65536, 1024), (100000, 1664, 156)):
        more = lib.fmoe_vocab_loss_fwd_workspace_bytes(T, 2944, V, top, 1, 0) - lib.fmoe_vocab_loss_fwd_workspace_bytes(T, 2944, V, 1, 1, 0)
        assert min(T, 256) * ((V + 255) // 256) * 1024 <= more <= 1 << 28, (T, V, top)


def test_embedding_refusals():
    with pytest.raises(RuntimeError, match="ROCm device"):
        embedding(torch.zeros(3, dtype=torch.long), torch.randn(4, 64))
    with pytest.raises(RuntimeError, match="ROCm device"):
        Embedding(10, 64)(torch.zeros(3, dtype=torch.long))
    for bad in (dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)):
        with pytest.raises(NotImplementedError, match="max_norm"):
            Embedding(10, 64, **bad)
    with FakeTensorMode():
        w = torch.empty(10, 64, device="cuda")
        ids = torch.empty(3, dtype=torch.long, device="cuda")
        with pytest.raises(ValueError, match=r"\[vocab, dim\]"):
            embedding(ids, w[0])
        with pytest.raises(ValueError, match=r"\[vocab, dim\]"):
            embedding(ids, w[:0])
        with pytest.raises(NotImplementedError, match="16384"):
            embedding(ids, torch.empty(2, 16385, device="cuda"))
        with pytest.raises(NotImplementedError, match="bf16 and fp32"):
            embedding(ids, w.half())
        with pytest.raises(ValueError, match="int32 or int64"):
            embedding(ids.float(), w)
        with pytest.raises(RuntimeError, match="weight's device"):
            embedding(torch.empty(3, dtype=torch.long), w)
        for pad in (10, -11):
            with pytest.raises(ValueError, match="padding_idx"):
                embedding(ids, w, padding_idx=pad)


def test_loss_refusals():
    with pytest.raises(RuntimeError, match="ROCm device"):
        linear_cross_entropy(torch.randn(3, 64), torch.randn(10, 64), torch.zeros(3, dtype=torch.long))
    with FakeTensorMode():
        h, w = torch.empty(2, 3, 64, device="cuda"), torch.empty(10, 64, device="cuda")
        t = torch.empty(2, 3, dtype=torch.long, device="cuda")
        index = torch.empty(2, 3, 5, dtype=torch.long, device="cuda")
        z = torch.empty(2, 3, 5, device="cuda")
        for call in (lambda h=h, w=w, **k: linear_cross_entropy(h, w, t, **k),
                     lambda h=h, w=w, **k: linear_distillation(h, w, index, z, **k)):
            with pytest.raises(ValueError, match="columns"):
                call(h[..., :63])
            with pytest.raises(RuntimeError, match="one dtype"):
                call(h.bfloat16())
            with pytest.raises(NotImplementedError, match="bf16 and fp32"):
                call(h.half())
            with pytest.raises(NotImplementedError, match="bf16 and fp32"):
                call(h, w.double())
            with pytest.raises(RuntimeError, match="device"):
                call(torch.empty(2, 3, 64))
            with pytest.raises(ValueError, match="reduction"):
                call(reduction="batchmean")
            for bad in (float("inf"), float("nan")):
                with pytest.raises(ValueError, match="logit_scale"):
                    call(logit_scale=bad)
        with pytest.raises(ValueError, match="shape"):
            linear_cross_entropy(h, w, t[0])
        with pytest.raises(ValueError, match="int32 or int64"):
            linear_cross_entropy(h, w, t.float())
        with pytest.raises(ValueError, match="shape"):
            linear_distillation(h, w, index[0], z[0])
        with pytest.raises(ValueError, match="teacher_logits"):
            linear_distillation(h, w, index, z[..., :4])
        with pytest.raises(NotImplementedError, match="bf16 and fp32"):
            linear_distillation(h, w, index, z.half())
        with pytest.raises(NotImplementedError, match="1024"):
            linear_distillation(h, w, index[..., :0], z[..., :0])
        with pytest.raises(NotImplementedError, match="1024"):
            linear_distillation(h, w, t[..., None].expand(2, 3, 1025), z[..., :1].expand(2, 3, 1025))
        with pytest.raises(NotImplementedError, match="teacher"):
            linear_distillation(h, w, index, z.requires_grad_(True))
        for bad in (0.0, -1.0, float("inf"), float("nan")):
            with pytest.raises(ValueError, match="temperature"):
                linear_distillation(h, w, index, z.detach(), temperature=bad)


def test_factors_outside_fp32_are_refused():
    # the logits' factor logit_scale / temperature, the gradients' logit_scale * temperature and the loss's temperature^2
    # are fp32 numbers in the kernels
    with FakeTensorMode():
        h, w = torch.empty(3, 64, device="cuda"), torch.empty(10, 64, device="cuda")
        index, z = torch.empty(3, 5, dtype=torch.long, device="cuda"), torch.empty(3, 5, device="cuda")
        for bad in (dict(temperature=1e-20), dict(temperature=1e-300), dict(temperature=1e20), dict(logit_scale=-1e38),
                    dict(logit_scale=1e300), dict(logit_scale=1e25, temperature=1e-15), dict(logit_scale=1e25, temperature=1e15)):
            with pytest.raises(ValueError, match="fp32"):
                linear_distillation(h, w, index, z, **bad)
        with pytest.raises(ValueError, match="fp32"):
            linear_cross_entropy(h, w, index[:, 0], logit_scale=1e38)
    lib = _lib.load()
    big = 1 << 40  # (more than any workspace below; nothing is launched: the loss's address is missing)

    def fwd(scale, temp, teacher=FAKE, grad=False):
        head = (FAKE, 0, 64, FAKE, 0, 64, FAKE, 1, teacher, 1, 100, 64, 100, 1, -100, scale, temp, 1, 1)
        if grad:
            return lib.fmoe_vocab_loss_fwd_grad(*head, FAKE + 2, FAKE, 0, FAKE, 0, FAKE, big, None)
        return lib.fmoe_vocab_loss_fwd(*head, FAKE + 2, FAKE, big, FAKE, big, None)

    def bwd(scale, temp):
        return lib.fmoe_vocab_loss_bwd(FAKE + 2, FAKE, 0, 64, 100, 64, 100, 1, 1, scale, temp, 1, 1, FAKE, big, FAKE, 0, FAKE,
                                       0, FAKE, big, None)

    for scale, temp, rc in ((1.0, 2.0, 3), (-1e3, 1e-3, 3), (1.0, 1e-20, 1), (1.0, 1e20, 1), (1e38, 1.0, 1), (1e25, 1e15, 1),
                            (1e25, 1e-15, 1), (float("nan"), 1.0, 1), (float("inf"), 1.0, 1)):
        assert fwd(scale, temp) == fwd(scale, temp, grad=True) == bwd(scale, temp) == rc, (scale, temp)


def test_embedding_module_has_torchs_interface():
    a, b = Embedding(12, 8, padding_idx=2, scale=3.0), torch.nn.Embedding(12, 8, padding_idx=2)
    assert isinstance(a, torch.nn.Embedding) and a.scale == 3.0 and a.padding_idx == 2
    assert not a.weight[2].any() and "scale=3.0" in repr(a)
    assert {k: tuple(v.shape) for k, v in a.state_dict().items()} == {
        k: tuple(v.shape) for k, v in b.state_dict().items()}
    c = Embedding.from_pretrained(b.weight.detach(), freeze=False)
    assert torch.equal(c.weight, b.weight) and c.scale == 1.0
    assert fusionllm_amd.Embedding is Embedding


def test_operator_fake_shapes():
    with FakeTensorMode():
        w = torch.empty(10, 64, device="cuda", dtype=torch.bfloat16)
        ids = torch.empty(7, dtype=torch.long, device="cuda")
        y = torch.ops.fusionllm.embedding_fwd(ids, w, 1.0, -1)
        assert (y.shape, y.dtype) == ((7, 64), torch.bfloat16)
        dw = torch.ops.fusionllm.embedding_bwd(ids, y, 10, 1.0, -1)
        assert (dw.shape, dw.dtype) == ((10, 64), torch.bfloat16)
        for reduction, shape in (("mean", ()), ("none", (7,))):
            loss, state = torch.ops.fusionllm.vocab_loss_fwd(y, w, ids[:, None], None, -100, 1.0, 1.0, 1, reduction)
            assert (loss.shape, loss.dtype) == (shape, torch.float32)
            assert state.shape == (K.vocab_loss_state_bytes(7, 64, 1, 1),)
            dh, dw = torch.ops.fusionllm.vocab_loss_bwd(loss, y, w, state, 1, False, 1.0, 1.0, 1, reduction)
            assert (dh.shape, dw.shape, dh.dtype) == ((7, 64), (10, 64), torch.bfloat16)


@pytest.mark.parametrize("need_h,need_w", [(True, True), (True, False), (False, True)])
def test_traced_backward_forms_the_wanted_gradients(need_h, need_w):
    # of the operators that torch.compile runs: a frozen head or frozen hidden states cost no product, and the hidden states,
    # which the state holds packed, are not kept a second time
    from torch.utils._python_dispatch import TorchDispatchMode
    calls = []

    class Calls(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if func is torch.ops.fusionllm.vocab_loss_bwd.default:
                calls.append((args, out))
            return out

    with FakeTensorMode():  # (on the CPU, where autograd runs without a device)
        h = torch.empty(7, 64, dtype=torch.bfloat16, requires_grad=need_h)
        w = torch.empty(10, 64, requires_grad=need_w)
        index = torch.empty(7, 1, dtype=torch.long)
        loss = torch.ops.fusionllm.vocab_loss_fwd(h, w, index, None, -100, 1.0, 1.0, 1, "none")[0]
        kept = [t for t in loss.grad_fn.saved_tensors]
        assert all(t.shape != h.shape for t in kept)
        with Calls():
            grads = torch.autograd.grad(loss, [t for t in (h, w) if t.requires_grad], torch.ones_like(loss))
    (args, out), = calls
    asked = (*args[10:], True, True)[:2]  # (arguments that have their defaults are left out)
    assert args[1].shape == (7, 0) and asked == (need_h, need_w)
    want = [((7, 64), torch.bfloat16)] * need_h + [((10, 64), torch.float32)] * need_w
    assert [(tuple(t.shape), t.dtype) for t in out] == want
    assert [(tuple(t.shape), t.dtype) for t in grads] == want


def _objects():
    from fusionllm_amd import build
    return [build.BUILD_DIR / "vocab_loss.o", build.BUILD_DIR / "embedding.o"]


def test_vocabulary_kernels_read_no_register_a_load_is_still_filling():
    # The products issue their global -> LDS copies and their MFMAs from inline assembly with explicit waits.
    from tests import isa_check as ic
    objs = _objects()
    if not (ic.ROCM_LLVM / "llvm-objdump").exists() or not all(o.exists() for o in objs):
        pytest.skip("no built objects or no llvm-objdump")
    checked = 0
    for o in objs:
        n, hazards = ic.check_object(o)
        assert not hazards, "\n".join(hazards[:10])
        checked += n
    assert checked >= 30


def test_vocabulary_kernels_keep_their_values_in_registers(tmp_path):
    from tests import isa_check as ic
    if not ic.ROCM_LLVM.exists() or not all(o.exists() for o in _objects()):
        pytest.skip("no built objects or no LLVM tools here")
    seen = 0
    for obj in _objects():
        work = tmp_path / obj.stem
        work.mkdir()
        shutil.copy(obj, work / obj.name)
        subprocess.run([str(ic.ROCM_LLVM / "llvm-objdump"), "--offloading", obj.name], check=True, capture_output=True,
                       cwd=work)
        dev = next(p for p in work.iterdir() if "gfx950" in p.name)
        notes = subprocess.run([str(ic.ROCM_LLVM / "llvm-readelf"), "--notes", str(dev)], check=True,
                               capture_output=True, text=True).stdout
        for entry in notes.split("  - .agpr_count:")[1:]:
            name = re.search(r"\.name:\s+(\S+)", entry).group(1)
            seen += 1
            assert re.search(r"\.private_segment_fixed_size:\s*0\s", entry), name
            assert re.search(r"\.vgpr_spill_count:\s*0\s", entry), name
    assert seen >= 30
