"""What a training step's operators (atlas_amd.train_ops, libatlas_train.so) promise without a GPU: the library's symbols and argument structs are
those of include/atlas_train.h, bad arguments are refused before anything is launched, and the 64-bit references of the GPU tests agree with autograd."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import train_ref
from atlas_amd import _lib, build, train_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "atlas_train.h")


@pytest.fixture(scope="module")
def so():
    return build.build_train()


def test_exports_are_exactly_the_headers(so):
    hdr = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"\b(atlas_[a-z0-9_]+)\s*\(", hdr))
    assert declared == set(_lib.TRAIN_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", so], capture_output=True, text=True, check=True).stdout
    assert {ln.split()[-1] for ln in out.splitlines() if ln.split()[-1].startswith("atlas_")} == declared
    data = open(so, "rb").read()
    assert b"gfx950" in data and b"gfx942" not in data and b"sm_90" not in data


@pytest.mark.parametrize("name,cls", [("atlas_attention_args", _lib.AttentionArgs), ("atlas_gemm_args", _lib.GemmArgs)])
def test_struct_layout_is_the_headers(name, cls, tmp_path):
    fields = [f for f, _ in cls._fields_]
    c = tmp_path / "s.c"
    c.write_text(f'#include "{HEADER}"\n#include <stdio.h>\nint main(void) {{ printf("%zu\\n", sizeof({name}));\n'
                 + "".join(f'printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields) + "return 0; }\n")
    subprocess.check_call(["gcc", str(c), "-o", str(tmp_path / "s")])
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def test_c_entries_refuse_bad_arguments(so):
    L = _lib.train_lib()
    a = _lib.AttentionArgs()
    assert L.atlas_attention_forward(None, None) == -1 and L.atlas_attention_forward(ctypes.byref(a), None) == -1
    a.dtype, a.heads, a.kv_heads, a.dim, a.scale, a.q_offsets, a.k_offsets = 2, 4, 4, 64, 1.0, 16, 16
    assert L.atlas_attention_forward(ctypes.byref(a), None) == 0                     # no rows: nothing to do
    a.total_q = 1
    assert L.atlas_attention_forward(ctypes.byref(a), None) == -1                    # rows, but no pointers
    a.q, a.k, a.v, a.out, a.lse = 16, 16, 16, 16, 16
    for field, value, rc in (("dim", 60, -3), ("dim", 136, -3), ("dim", 0, -3), ("kv_heads", 3, -1), ("kv_heads", 0, -1), ("dtype", 3, -1), ("scale", 0.0, -1),
                             ("scale", float("nan"), -1), ("q", 24, -1), ("q_row", 4, -1), ("q_offsets", None, -1), ("batch", -1, -1), ("max_q", -1, -1)):
        old = getattr(a, field)
        setattr(a, field, value)
        assert L.atlas_attention_forward(ctypes.byref(a), None) == rc, field
        setattr(a, field, old)
    assert L.atlas_attention_backward(ctypes.byref(a), None) == -1                   # no dout, dq, delta
    a.keep, a.keep_row = 16, 1 << 26
    assert L.atlas_attention_forward(ctypes.byref(a), None) == -3                    # decisions out of a wave's reach
    a.keep, a.keep_row = None, 0
    a.max_q, a.max_k, a.total_q, a.total_k, a.batch = 64, 4096, 64, 4096, 1          # one short walk owner, one long walk: split
    need = L.atlas_attention_workspace_bytes(ctypes.byref(a), 0)
    assert need >= 2 * 64 * 4 * (64 + 2) * 4 and L.atlas_attention_forward(ctypes.byref(a), None) == -2
    a.ws, a.ws_bytes = 16, need - 1
    assert L.atlas_attention_forward(ctypes.byref(a), None) == -2
    a.ws, a.ws_bytes = 24, need
    assert L.atlas_attention_forward(ctypes.byref(a), None) == -2                    # not aligned
    a.ws, a.max_q, a.max_k, a.total_q, a.total_k, a.batch = None, 0, 0, 1, 0, 0
    for field in ("total_q", "total_k"):                                             # a sequence's length is an int
        old = getattr(a, field)
        setattr(a, field, 1 << 31)
        assert L.atlas_attention_forward(ctypes.byref(a), None) == -3, field
        setattr(a, field, old)
    g = _lib.GemmArgs()
    g.m, g.n, g.k, g.dtype = 4, 4, 4, 2
    assert L.atlas_gemm(None, None) == -1 and L.atlas_gemm(ctypes.byref(g), None) == -1
    g.a, g.b, g.c = 16, 16, 16
    for field, value, rc in (("dtype", 7, -1), ("m", -1, -1), ("a_layout", 2, -1), ("act", 2, -1), ("a_layout", 1, -3), ("b_codes", 16, -1), ("save_z_codes", 16, -1)):
        old = getattr(g, field)
        setattr(g, field, value)
        assert L.atlas_gemm(ctypes.byref(g), None) == rc, field
        setattr(g, field, old)
    g.m, g.n, g.k, g.a_layout, g.b_layout, g.lda, g.ldb, g.ldc = 64, 64, 1 << 20, 1, 1, 64, 64, 64
    need = L.atlas_gemm_workspace_bytes(ctypes.byref(g))
    assert need >= 2 * 64 * 64 * 4 and need % (64 * 64 * 4) == 0                     # a long contraction with few tiles is split
    assert L.atlas_gemm(ctypes.byref(g), None) == -2
    assert L.atlas_compress(16, 8, 4, 8, 9, 16, 16, None) == -1 and L.atlas_compress(None, 8, 4, 8, 2, 16, 16, None) == -1
    assert L.atlas_compress(16, 8, 4, 8, 2, 24, 16, None) == -1 and L.atlas_compress(None, 8, 0, 8, 2, None, None, None) == 0
    assert L.atlas_decompress(None, None, 1, 8, 2, None, None) == -1
    assert L.atlas_linear_dz(16, 8, 16, 16, 16, None, 1.0, 4, 8, 2, 16, None, None, 0, None) == -1      # z twice
    assert L.atlas_linear_dz(16, 8, None, None, None, None, 1.0, 4, 8, 2, None, 16, None, 0, None) == -2
    assert L.atlas_layer_norm_forward(16, 8, 16, 16, -1.0, 4, 8, 2, 16, 16, None) == -1
    assert L.atlas_layer_norm_backward(16, 8, 16, 16, 16, 8, 4, 8, 2, 16, 16, None, None, 0, None) == -1  # dw without db
    assert L.atlas_layer_norm_backward(16, 8, 16, 16, 16, 8, 4, 8, 2, 16, 16, 16, None, 0, None) == -2


def test_cpu_tensors_are_refused():
    x, off = torch.zeros(4, 2, 64), torch.tensor([0, 4], dtype=torch.int32)
    for call in (lambda: train_ops.attention(x, x, x, off), lambda: train_ops.linear(torch.zeros(2, 8), torch.zeros(4, 8)),
                 lambda: train_ops.layer_norm(torch.zeros(2, 8), torch.zeros(8), torch.zeros(8)), lambda: train_ops.compress(torch.zeros(2, 8)),
                 lambda: train_ops.linear([1.0], torch.zeros(4, 8))):
        with pytest.raises(_lib.AtlasHipError):
            call()


def test_missing_library_fails_loudly(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_train", None)
    monkeypatch.setattr(_lib, "TRAIN_SO", str(tmp_path / "nope.so"))
    with pytest.raises(_lib.AtlasHipError, match="no CPU fallback"):
        _lib.train_lib()


# ---- the references themselves -------------------------------------------------------------------------------------------
def _autograd(fn, inputs, dy):
    inputs = [t.double().requires_grad_() for t in inputs]
    y = fn(*inputs)
    return [y.detach(), *torch.autograd.grad(y, inputs, dy.double())]


def test_attention_reference_is_autograds():
    g = torch.Generator().manual_seed(1)
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q, k, v, do = rnd(7, 4, 16), rnd(9, 2, 16), rnd(9, 2, 16), rnd(7, 4, 16)
    seen = torch.tensor([1, 0, 1, 1, 1, 1, 0, 1, 1], dtype=torch.bool)
    keep = torch.rand((7, 4, 6), generator=g) > 0.3
    qo, ko = [0, 3, 7], [0, 5, 9]

    def fn(q, k, v):
        outs = []
        for b in range(2):
            Q, K, V = q[qo[b]:qo[b + 1]], k[ko[b]:ko[b + 1]].repeat_interleave(2, 1), v[ko[b]:ko[b + 1]].repeat_interleave(2, 1)
            s = torch.einsum("ihd,jhd->hij", Q, K) * 0.25
            p = torch.softmax(s.masked_fill(~seen[ko[b]:ko[b + 1]], -float("inf")), -1)
            m = keep[qo[b]:qo[b + 1]].permute(1, 0, 2)[:, :, : K.shape[0]].double() / 0.7
            outs.append(torch.einsum("hij,jhd->ihd", p * m, V))
        return torch.cat(outs)

    want = _autograd(fn, (q, k, v), do)
    got = train_ref.attention(q, k, v, do, qo, ko, 0.25, seen, keep, 1 / 0.7)
    for w, name in zip(want, ("out", "dq", "dk", "dv")):
        assert torch.allclose(got[name][0], w, rtol=1e-11, atol=1e-12), name


@pytest.mark.parametrize("gelu,drop", [(False, False), (True, True)])
def test_linear_reference_is_autograds(gelu, drop):
    g = torch.Generator().manual_seed(2)
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x, w, b, dy, r = rnd(5, 12), rnd(7, 12), rnd(7), rnd(5, 7), rnd(5, 7)
    keep = torch.rand((5, 7), generator=g) > 0.4 if drop else None

    def fn(x, w, b):
        z = x @ w.T + b
        y = torch.nn.functional.gelu(z) if gelu else z
        return (y * keep / 0.6 if drop else y) + r

    want = _autograd(fn, (x, w, b), dy)
    got = train_ref.linear(x, w, b, dy, gelu, keep, 1 / 0.6, r)
    for t, name in zip(want, ("y", "dx", "dw", "db")):
        assert torch.allclose(got[name][0], t, rtol=1e-11, atol=1e-12), name


def test_layer_norm_reference_is_autograds():
    g = torch.Generator().manual_seed(3)
    x, w, b, dy = (torch.randn(s, generator=g) for s in ((6, 20), (20,), (20,), (6, 20)))
    want = _autograd(lambda x, w, b: w * (x - x.mean(1, keepdim=True)) / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-3) + b, (x, w, b), dy)
    got = train_ref.layer_norm(x, w, b, dy, 1e-3)
    for t, name in zip(want, ("y", "dx", "dw", "db")):
        assert torch.allclose(got[name][0], t, rtol=1e-11, atol=1e-12), name


def test_eight_bit_reference_is_torchs_rounding():
    x = torch.randn(40, 96, generator=torch.Generator().manual_seed(4)).double() * torch.logspace(-6, 6, 40).double()[:, None]
    x[0, :32] = 0.0
    x[1, 0], x[2, 5] = 448.0, 449.0
    y = train_ref.eight_bits(x)
    g = x.unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    s = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=-126))
    assert torch.equal(y, ((g / s).float().to(torch.float8_e4m3fn).double() * s).flatten(-2))


# ---- what would be lost without a word ---------------------------------------------------------------------------------------
def _operator_calls():
    """{name: (call of (tensors), the tensors that take a gradient)}"""
    off = torch.tensor([0, 4], dtype=torch.int32)
    z = torch.zeros
    return {
        "attention": (lambda q, k, v: train_ops.attention(q, k, v, off), [z(4, 2, 8), z(4, 2, 8), z(4, 2, 8)]),
        "linear": (lambda x, w, b, r: train_ops.linear(x, w, b, residual=r), [z(2, 8), z(4, 8), z(4), z(2, 4)]),
        "layer_norm": (lambda x, w, b: train_ops.layer_norm(x, w, b), [z(2, 8), z(8), z(8)]),
    }


@pytest.mark.parametrize("name", ["attention", "linear", "layer_norm"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(name, grad):
    """a tangent would be dropped, which says that the derivative is zero: whichever tensor carries it, with grad mode or without"""
    import torch.autograd.forward_ad as fw

    call, tensors = _operator_calls()[name]
    for i in range(len(tensors)):
        with fw.dual_level(), torch.set_grad_enabled(grad):
            dual = [fw.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(tensors)]
            with pytest.raises(_lib.AtlasHipError, match="forward-mode"):
                call(*dual)


@pytest.mark.parametrize("name", ["attention", "linear", "layer_norm", "compress"])
def test_traces_and_function_transforms_are_refused(name):
    """a trace would hold the empty result and none of the computation; a wrapped tensor has no memory that a kernel could read"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    call, tensors = {**_operator_calls(), "compress": (lambda x: train_ops.compress(x).codes, [torch.zeros(2, 8)])}[name]
    with pytest.raises(_lib.AtlasHipError, match="trace"):
        torch.jit.trace(call, tuple(tensors))
    with pytest.raises(_lib.AtlasHipError, match="trace|plain tensor"):
        make_fx(call)(*tensors)
    with pytest.raises(_lib.AtlasHipError, match="trace|plain tensor"), FakeTensorMode() as mode:
        call(*[mode.from_tensor(t) for t in tensors])
    for i in range(len(tensors)):
        batched = [t[None] if j == i else t for j, t in enumerate(tensors)]
        with pytest.raises(_lib.AtlasHipError, match="plain tensor"):
            torch.func.vmap(call, in_dims=tuple(0 if j == i else None for j in range(len(tensors))))(*batched)
        with pytest.raises(_lib.AtlasHipError, match="plain tensor|forward-mode"):
            torch.func.grad(lambda t: call(*tensors[:i], t, *tensors[i + 1:]).sum())(tensors[i])


def test_workspaces_off_their_border_are_refused(so):
    """parts are read 16 bytes at a time (the dense layer's) or as floats (sums of columns). The pointers are never followed: every call here ends in the host's checks"""
    L = _lib.train_lib()
    g = _lib.GemmArgs()
    g.a, g.b, g.c, g.dtype = 16, 16, 16, 2
    g.m, g.n, g.k, g.a_layout, g.b_layout, g.lda, g.ldb, g.ldc = 64, 64, 1 << 20, 1, 1, 64, 64, 64
    need = L.atlas_gemm_workspace_bytes(ctypes.byref(g))
    assert need > 0
    for ws in (24, 20, 17):
        g.ws, g.ws_bytes = ws, need
        assert L.atlas_gemm(ctypes.byref(g), None) == -2
    ws_bytes = 1 << 20
    for ws in (17, 18):
        assert L.atlas_linear_dz(16, 8, None, None, None, None, 1.0, 400, 8, 2, None, 16, ws, ws_bytes, None) == -2
        assert L.atlas_layer_norm_backward(16, 8, 16, 16, 16, 8, 400, 8, 2, 16, 16, 16, ws, ws_bytes, None) == -2


def test_attentions_rest_off_its_border_is_refused(so):
    L = _lib.train_lib()
    a = _lib.AttentionArgs()
    a.dtype, a.heads, a.kv_heads, a.dim, a.scale, a.q_offsets, a.k_offsets, a.total_q = 2, 4, 4, 64, 1.0, 16, 16, 1
    a.q, a.k, a.v, a.out, a.lse, a.out_rest = 16, 16, 16, 16, 16, 24
    assert L.atlas_attention_forward(ctypes.byref(a), None) == -1 and L.atlas_attention_backward(ctypes.byref(a), None) == -1
