"""Differentiable operators of a retriever training step on hand-written HIP kernels (include/atlas_train.h, csrc/train).

    attention(q, k, v, q_offsets, ...)      softmax attention over packed sequences; the backward pass recomputes the probabilities
    linear(x, weight, bias, ...)            dense layer with bias, GELU, dropout and residual in its epilogue
    layer_norm(x, weight, bias, eps)        BERT's layer norm with the uncentred second moment (src/modeling_bert.py:104-114)
    compress(x)                             an activation in 8 bits; linear(..., checkpoint="e4m3") keeps what its backward pass needs that way

They are what `Contriever` calls in training when `training_kernels` is on (atlas_amd.retriever_train), and can be called on their own.

All take and return tensors of one dtype (fp16, bf16 or fp32) on one MI355X; sums, softmax and norm statistics are fp32 and a result is
rounded once. Work is enqueued on the current stream of the tensors' device. Results and gradients are the same bits from call to call.
There is no CPU or eager fallback: anything the kernels do not take raises AtlasHipError before a launch. Once differentiable.
Calls can be captured into a CUDA graph, forward and backward; as with any autograd work, let no other graph of the same leaves live
through the capture.
"""
import ctypes

import torch

from . import _lib

_DTYPES = {torch.float16: 0, torch.float32: 1, torch.bfloat16: 2}       # ATLAS_TRAIN_*
_NAMES = {-1: "ATLAS_TRAIN_E_BADARG", -2: "ATLAS_TRAIN_E_WORKSPACE", -3: "ATLAS_TRAIN_E_UNSUPPORTED"}


def _refuse(what):
    raise _lib.AtlasHipError(what)


def _check(rc, what):
    if rc:
        raise _lib.AtlasHipError(f"{what} failed: {_NAMES.get(rc, 'hipError_t ' + str(rc))}")


def _operand(name, t, dtype=None, device=None):
    """a tensor the kernels can take: on a GPU, of a known dtype, like the others of the call"""
    if not isinstance(t, torch.Tensor):
        _refuse(f"{name} has to be a tensor, not {type(t).__name__}")
    if not t.is_cuda:
        _refuse(f"{name} is on {t.device}: train_ops run on an MI355X only; there is no CPU / eager fallback")
    if t.dtype not in _DTYPES:
        _refuse(f"{name}: unsupported dtype {t.dtype}")
    if dtype is not None and t.dtype != dtype:
        _refuse(f"{name} is {t.dtype}, the call's other tensors are {dtype}")
    if device is not None and t.device != device:
        _refuse(f"{name} is on {t.device}, the call's other tensors on {device}")


def _decisions(name, t, shape, device):
    """a 0 / 1 tensor as bytes"""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.bool, torch.uint8) or t.device != device:
        _refuse(f"{name} has to be a bool or uint8 tensor on {device}")
    if tuple(t.shape) != tuple(shape):
        _refuse(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


class _on:
    """the tensors' device as the current one, and its current stream"""

    def __init__(self, t):
        self.index = t.device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *a):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


# ---- attention --------------------------------------------------------------------------------------------------------
def _heads_ready(t):
    """[T, H, D] with a contiguous, 16-byte aligned last dimension, as a view where it is one already"""
    s = 16 // t.element_size()
    ok = (t.stride(2) == 1 or t.shape[2] == 1) and t.stride(0) % s == 0 and t.stride(1) % s == 0 and t.data_ptr() % 16 == 0 and t.stride(0) < s << 20
    return t if ok else t.contiguous()


def _attention_args(q, k, v, q_offsets, k_offsets, max_q, max_k, key_mask, scale, keep_scale, out, lse, cols, bits):
    a = _lib.AttentionArgs()
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_row, a.q_head = q.stride(0), q.stride(1)
    a.k_row, a.k_head = k.stride(0), k.stride(1)
    a.v_row, a.v_head = v.stride(0), v.stride(1)
    a.q_offsets, a.k_offsets = q_offsets.data_ptr(), k_offsets.data_ptr()
    a.total_q, a.total_k, a.batch = q.shape[0], k.shape[0], q_offsets.numel() - 1
    a.heads, a.kv_heads, a.dim = q.shape[1], k.shape[1], q.shape[2]
    a.max_q, a.max_k, a.dtype = max_q, max_k, _DTYPES[q.dtype]
    if key_mask is not None:
        a.key_mask = key_mask.data_ptr()
    a.keep_cols = cols
    if bits is not None:
        a.keep_bits = bits.data_ptr()
    a.scale, a.keep_scale = scale, keep_scale
    a.out, a.lse = out.data_ptr(), lse.data_ptr()
    return a


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_offsets, k_offsets, max_q, max_k, key_mask, scale, keep, keep_scale, grad_mode):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device)
        cols, bits = 0, None
        if keep is not None:
            cols = keep.shape[2]
            if grad_mode:                           # the decisions as bits are what the backward pass reads (never an empty tensor: its pointer says "dropout")
                bits = torch.empty(max(1, lse.numel() * ((cols + 31) // 32)), dtype=torch.int32, device=q.device)
        a = _attention_args(q, k, v, q_offsets, k_offsets, max_q, max_k, key_mask, scale, keep_scale, out, lse, cols, bits)
        if keep is not None:
            a.keep, a.keep_row, a.keep_head = keep.data_ptr(), keep.stride(0), keep.stride(1)
            if keep.numel() == 0:                   # no column to read, but dropout all the same: nothing is kept
                a.keep = q_offsets.data_ptr()
        with _on(q) as stream:
            _check(_lib.train_lib().atlas_attention_forward(ctypes.byref(a), stream), "atlas_attention_forward")
        ctx.save_for_backward(q, k, v, q_offsets, k_offsets, key_mask, bits, out, lse)
        ctx.rest = (max_q, max_k, scale, keep_scale, cols)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, q_offsets, k_offsets, key_mask, bits, out, lse = ctx.saved_tensors
        max_q, max_k, scale, keep_scale, cols = ctx.rest
        dout = _heads_ready(dout)
        a = _attention_args(q, k, v, q_offsets, k_offsets, max_q, max_k, key_mask, scale, keep_scale, out, lse, cols, bits)
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        delta = torch.empty_like(lse)
        a.dout, a.dout_row, a.dout_head = dout.data_ptr(), dout.stride(0), dout.stride(1)
        a.dq, a.dk, a.dv, a.delta = dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), delta.data_ptr()
        with _on(q) as stream:
            _check(_lib.train_lib().atlas_attention_backward(ctypes.byref(a), stream), "atlas_attention_backward")
        return (dq, dk, dv) + (None,) * 9


def _offsets(name, t, device):
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or t.numel() < 1 or t.dtype not in (torch.int32, torch.int64) or t.device != device:
        _refuse(f"{name} has to be a 1-d int32 (or int64) tensor of batch + 1 offsets on {device}")
    return t.to(torch.int32).contiguous()


def attention(q, k, v, q_offsets, k_offsets=None, *, max_q=None, max_k=None, key_mask=None, scale=None, keep=None, keep_scale=1.0):
    """Attention of packed sequences: out[t, h] = sum_j P[t, h, j] keep[t, h, j] keep_scale v[j, h'] with P = softmax_j(scale q[t, h] . k[j, h'])

    q [Tq, H, D]; k, v [Tk, H', D], H a multiple of H' (query head h reads key head h' = h // (H / H')); views of a fused projection are
    read in place. Sequence b is rows q_offsets[b] : q_offsets[b + 1] of q and k_offsets[b] : k_offsets[b + 1] of k and v (int32
    [batch + 1] on the device, non-decreasing; k_offsets defaults to q_offsets). D: a multiple of 8, at most 128.

    max_q, max_k    the longest sequence, as far as the host knows it (launch sizes; default: all rows)
    key_mask        bool [Tk]: False hides a key (its k and v are not used, whatever they hold)
    keep            bool [Tq, H, C]: dropout decisions, column j for key j of the row's sequence (columns from C on count as dropped)
    scale           default 1 / sqrt(D); positive

    A row that sees no key gives zeros and takes and gives no gradient; rows of q that belong to no sequence likewise."""
    _operand("q", q)
    for name, t in (("k", k), ("v", v)):
        _operand(name, t, q.dtype, q.device)
    if q.dim() != 3 or k.dim() != 3 or tuple(k.shape) != tuple(v.shape) or k.shape[2] != q.shape[2]:
        _refuse(f"attention takes q [Tq, H, D] and k, v [Tk, H', D]: got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    dim = q.shape[2]
    if dim == 0 or dim % 8 or dim > 128:
        _refuse(f"attention: head dimension {dim}; multiples of 8 up to 128 are implemented")
    if k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % k.shape[1]:
        _refuse(f"attention: {q.shape[1]} query heads cannot share {k.shape[1]} key heads evenly")
    q_offsets = _offsets("q_offsets", q_offsets, q.device)
    if k_offsets is None:
        if k.shape[0] != q.shape[0]:
            _refuse("attention: k_offsets is needed where q and k have different rows")
        k_offsets = q_offsets
    else:
        k_offsets = _offsets("k_offsets", k_offsets, q.device)
    if k_offsets.numel() != q_offsets.numel():
        _refuse(f"attention: {q_offsets.numel() - 1} query sequences, {k_offsets.numel() - 1} key sequences")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        _refuse(f"attention: scale {scale} is not positive")
    if key_mask is not None:
        key_mask = _decisions("key_mask", key_mask, (k.shape[0],), q.device).contiguous()
    if keep is not None:
        cols = keep.shape[2] if isinstance(keep, torch.Tensor) and keep.dim() == 3 else -1
        keep = _decisions("keep", keep, (q.shape[0], q.shape[1], cols), q.device)
        if keep.dtype == torch.uint8:
            keep = keep != 0
        if keep.stride(2) != 1 and cols > 1:
            keep = keep.contiguous()
    longest = lambda given, rows: min(rows, 2 ** 31 - 1) if given is None else max(0, min(int(given), rows))  # noqa: E731
    return _Attention.apply(_heads_ready(q), _heads_ready(k), _heads_ready(v), q_offsets, k_offsets, longest(max_q, q.shape[0]), longest(max_k, k.shape[0]),
                            key_mask, scale, keep, float(keep_scale), torch.is_grad_enabled())


# ---- 8-bit activations -------------------------------------------------------------------------------------------------
class Compressed:
    """An activation in 8 bits: e4m3 codes with a power of two for every 32 values of a row (1.03 bytes a value). `decode()` gives the values back."""

    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes, scales, shape, dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, shape, dtype

    def decode(self, dtype=None):
        """the values that the codes stand for, rounded to `dtype` (default: the compressed tensor's)"""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _DTYPES:
            _refuse(f"decode: unsupported dtype {dtype}")
        out = torch.empty(self.shape, dtype=dtype, device=self.codes.device)
        n = self.shape[-1]
        with _on(out) as stream:
            _check(_lib.train_lib().atlas_decompress(self.codes.data_ptr(), self.scales.data_ptr(), out.numel() // n if n else 0, n, _DTYPES[dtype],
                                                     out.data_ptr(), stream), "atlas_decompress")
        return out


def _code_buffers(m, n, device):
    groups = (n + 31) // 32
    return torch.empty((m, groups * 32), dtype=torch.uint8, device=device), torch.empty((m, groups), dtype=torch.uint8, device=device)


def _rows(t):
    """any tensor as [rows, last dimension] with a contiguous last dimension, as a view where it is one already, and its row stride"""
    n = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(t.numel() // n if n else 0, n)
    if t.shape[0] <= 1 or n == 0:
        return t.contiguous(), n
    if t.stride(1) != 1 and n > 1:
        t = t.contiguous()
    return t, t.stride(0)


def _compress_rows(x, ldx):
    codes, scales = _code_buffers(x.shape[0], x.shape[1], x.device)
    with _on(x) as stream:
        _check(_lib.train_lib().atlas_compress(x.data_ptr(), ldx, x.shape[0], x.shape[1], _DTYPES[x.dtype], codes.data_ptr(), scales.data_ptr(), stream),
               "atlas_compress")
    return codes, scales


def compress(x):
    """`x` (at least one dimension) in 8 bits. Every 32 consecutive values of the last dimension share a power of two, the smallest that keeps
    them within 448; a value is rounded to nearest even in e4m3: off by at most 1/16 of itself or 2^-17 of the group's largest. Values that are
    not finite come back as NaN and disturb no other. Not differentiable: what comes back is cut off from x's graph."""
    _operand("x", x)
    if x.dim() < 1:
        _refuse("compress takes a tensor of at least one dimension")
    x = x.detach()
    rows, ld = _rows(x)
    return Compressed(*_compress_rows(rows, ld), x.shape, x.dtype)


# ---- dense layer ------------------------------------------------------------------------------------------------------
def _gemm(a, lda, b, ldb, c, m, n, k, a_layout, b_layout, codes=None, **epilogue):
    L = _lib.train_lib()
    g = _lib.GemmArgs()
    g.a, g.lda, g.ldb, g.ldc = a.data_ptr(), lda, ldb, n
    if codes is None:
        g.b = b.data_ptr()
    else:
        g.b_codes, g.b_scales = codes[0].data_ptr(), codes[1].data_ptr()
    g.m, g.n, g.k, g.dtype, g.a_layout, g.b_layout = m, n, k, _DTYPES[a.dtype], a_layout, b_layout
    g.c = c.data_ptr()
    for name, value in epilogue.items():
        if value is not None:
            setattr(g, name, value.data_ptr() if isinstance(value, torch.Tensor) else value)
    need = L.atlas_gemm_workspace_bytes(ctypes.byref(g))
    ws = None
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=c.device)
        g.ws, g.ws_bytes = ws.data_ptr(), need
    with _on(c) as stream:
        _check(L.atlas_gemm(ctypes.byref(g), stream), "atlas_gemm")


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, keep, keep_scale, gelu, eight_bits, grad_mode):
        n, k = weight.shape
        x2, ldx = _rows(x)
        w2, ldw = _rows(weight)
        m = x2.shape[0]
        y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=x.device)
        r2, ldr = _rows(residual) if residual is not None else (None, 0)
        need_x, need_w, need_b = (grad_mode and need for need in ctx.needs_input_grad[:3])
        z = z_codes = z_scales = None
        if gelu and (need_x or need_w or need_b):                          # what the activation's slope is taken from
            if eight_bits:
                z_codes, z_scales = _code_buffers(m, n, x.device)
            else:
                z = torch.empty((m, n), dtype=x.dtype, device=x.device)
        _gemm(x2, ldx, w2, ldw, y, m, n, k, 0, 0, bias=bias, act=int(gelu), save_z=z, save_z_codes=z_codes, save_z_scales=z_scales, keep=keep,
              keep_scale=keep_scale, residual=r2, ld_residual=ldr)
        x_codes = x_scales = None
        if eight_bits and need_w:
            x_codes, x_scales = _compress_rows(x2, ldx)
        ctx.save_for_backward(x if need_w and not eight_bits else None, x_codes, x_scales, weight, z, z_codes, z_scales, keep)
        ctx.rest = (x.shape, bias is not None, keep_scale)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, x_codes, x_scales, weight, z, z_codes, z_scales, keep = ctx.saved_tensors
        x_shape, has_bias, keep_scale = ctx.rest
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        n, k = weight.shape
        L = _lib.train_lib()
        d2, ldd = _rows(dy)
        m, dtype = d2.shape[0], _DTYPES[dy.dtype]
        dx = dw = db = None
        changed = z is not None or z_codes is not None or keep is not None  # dz is dy otherwise
        need_b = need_b and has_bias
        dz, ldz = d2, ldd
        if (changed and (need_x or need_w)) or need_b:
            dz_out = torch.empty((m, n), dtype=dy.dtype, device=dy.device) if changed and (need_x or need_w) else None
            ws = None
            if need_b:
                db = torch.empty((n,), dtype=dy.dtype, device=dy.device)
                ws = torch.empty(L.atlas_linear_dz_workspace_bytes(m, n), dtype=torch.uint8, device=dy.device)
            p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
            with _on(dy) as stream:
                _check(L.atlas_linear_dz(d2.data_ptr(), ldd, p(z), p(z_codes), p(z_scales), p(keep), keep_scale, m, n, dtype, p(dz_out), p(db), p(ws),
                                         0 if ws is None else ws.numel(), stream), "atlas_linear_dz")
            if dz_out is not None:
                dz, ldz = dz_out, n
        if need_x:
            w2, ldw = _rows(weight)
            dx = torch.empty(x_shape, dtype=dy.dtype, device=dy.device)
            _gemm(dz, ldz, w2, ldw, dx, m, k, n, 0, 1)
        if need_w:
            dw = torch.empty((n, k), dtype=dy.dtype, device=dy.device)
            if x_codes is not None:
                _gemm(dz, ldz, None, x_codes.shape[1], dw, n, k, m, 1, 1, codes=(x_codes, x_scales))
            else:
                x2, ldx = _rows(x)
                _gemm(dz, ldz, x2, ldx, dw, n, k, m, 1, 1)
        return (dx, dw, db, dy if need_r else None) + (None,) * 5


def linear(x, weight, bias=None, *, activation=None, keep=None, keep_scale=1.0, residual=None, checkpoint=None):
    """y = act(x weight^T + bias) * (keep ? keep_scale : 0) + residual, one product with everything else in its epilogue, rounded once

    x [..., K], weight [N, K], bias [N], residual and keep [..., N]; activation None or "gelu" (exact erf form); keep: bool, the dropout's
    decisions. checkpoint="e4m3" keeps x and the pre-activation for the backward pass in 8 bits (see `compress`; the pre-activation is
    rounded from fp32): weight.grad and the activation's slope are then those of the 8-bit values, x.grad and bias.grad otherwise exact."""
    _operand("x", x)
    _operand("weight", weight, x.dtype, x.device)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        _refuse(f"linear takes x [..., K] and weight [N, K]: got {tuple(x.shape)} and {tuple(weight.shape)}")
    if 0 in weight.shape:
        _refuse(f"linear: a layer of {weight.shape[1]} inputs and {weight.shape[0]} outputs")
    out_shape = x.shape[:-1] + (weight.shape[0],)
    if x.numel() // max(1, x.shape[-1]) >= 2 ** 31 or max(weight.shape) >= 2 ** 31:
        _refuse("linear: a dimension of 2^31 or more")
    if bias is not None:
        _operand("bias", bias, x.dtype, x.device)
        if tuple(bias.shape) != (weight.shape[0],):
            _refuse(f"bias has shape {tuple(bias.shape)}, expected {(weight.shape[0],)}")
        bias = bias.contiguous()
    if residual is not None:
        _operand("residual", residual, x.dtype, x.device)
        if tuple(residual.shape) != tuple(out_shape):
            _refuse(f"residual has shape {tuple(residual.shape)}, expected {tuple(out_shape)}")
    if keep is not None:
        keep = _decisions("keep", keep, out_shape, x.device).contiguous()
    if activation not in (None, "gelu"):
        _refuse(f"activation={activation!r}: None and the exact-erf 'gelu' are implemented")
    if checkpoint not in (None, "e4m3"):
        _refuse(f"checkpoint={checkpoint!r}: None and 'e4m3' are implemented")
    return _Linear.apply(x, weight, bias, residual, keep, float(keep_scale), activation == "gelu", checkpoint == "e4m3", torch.is_grad_enabled())


# ---- layer norm -------------------------------------------------------------------------------------------------------
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2, ldx = _rows(x)
        m, n = x2.shape
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = torch.empty((m, 2), dtype=torch.float32, device=x.device)
        with _on(x) as stream:
            _check(_lib.train_lib().atlas_layer_norm_forward(x2.data_ptr(), ldx, weight.data_ptr(), bias.data_ptr(), eps, m, n, _DTYPES[x.dtype], y.data_ptr(),
                                                             stats.data_ptr(), stream), "atlas_layer_norm_forward")
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        x2, ldx = _rows(x)
        d2, ldd = _rows(dy)
        m, n = x2.shape
        L = _lib.train_lib()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        dw = db = ws = None
        if need_w or need_b:
            dw, db = torch.empty_like(weight), torch.empty_like(weight)
            ws = torch.empty(L.atlas_layer_norm_workspace_bytes(m, n), dtype=torch.uint8, device=x.device)
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        with _on(x) as stream:
            _check(L.atlas_layer_norm_backward(x2.data_ptr(), ldx, weight.data_ptr(), stats.data_ptr(), d2.data_ptr(), ldd, m, n, _DTYPES[x.dtype], p(dx), p(dw), p(db),
                                               p(ws), 0 if ws is None else ws.numel(), stream), "atlas_layer_norm_backward")
        return dx, dw if need_w else None, db if need_b else None, None


def layer_norm(x, weight, bias, eps=1e-12):
    """y = weight (x - mean(x)) / sqrt(mean(x^2) + eps) + bias over the last dimension: the reference's BertLayerNorm, whose scale is the root of the
    UNCENTRED second moment (src/modeling_bert.py:104-114)"""
    _operand("x", x)
    if x.dim() < 1:
        _refuse("layer_norm takes a tensor of at least one dimension")
    if x.shape[-1] == 0:
        _refuse("layer_norm: rows of length 0")
    for name, t in (("weight", weight), ("bias", bias)):
        _operand(name, t, x.dtype, x.device)
        if tuple(t.shape) != (x.shape[-1],):
            _refuse(f"{name} has shape {tuple(t.shape)}, expected {(x.shape[-1],)}")
    if not 0.0 <= eps < float("inf"):
        _refuse(f"layer_norm: eps {eps}")
    return _LayerNorm.apply(x, weight.contiguous(), bias.contiguous(), float(eps))
