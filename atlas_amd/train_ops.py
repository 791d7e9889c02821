"""Differentiable operators of a retriever training step on hand-written HIP kernels (include/atlas_train.h, csrc/train).

    attention(q, k, v, q_offsets, ...)      softmax attention over packed sequences; the backward pass recomputes the probabilities
    linear(x, weight, bias, ...)            dense layer with bias, GELU, dropout and residual in its epilogue
    layer_norm(x, weight, bias, eps)        BERT's layer norm with the uncentred second moment (src/modeling_bert.py:104-114)
    compress(x)                             an activation in 8 bits; linear(..., checkpoint="e4m3") keeps what its backward pass needs that way

They are what `Contriever` calls in training after `training_kernels_enable()` (atlas_amd.retriever_train), and can be called on their own.

All take and return tensors of one dtype (fp16, bf16 or fp32) on one MI355X, whatever autocast says; sums, softmax and norm statistics are fp32 and a result
is rounded once. In 16 bits so is what becomes an operand of a further product or is kept for the backward pass -- attention's probabilities and their
gradients, a dense layer's pre-activation and its gradient: where there are any, a gradient is off by some 1.45 of what rounding it once would cost
(bf16: 0.0024 of its norm for 0.0017). Work is enqueued on the current stream of the tensors' device. Results and gradients are the same bits from call to call.
There is no CPU or eager fallback: anything the kernels do not take raises AtlasHipError before a launch. Once differentiable, in reverse mode: a
tensor with a forward-mode tangent raises, and so does a call under torch.jit.trace, torch.export or the transforms of torch.func.
Calls can be captured into a CUDA graph, forward and backward. A backward pass cannot be captured while a graph of the same leaves from the
default stream is alive: a captured call that meets one raises.
"""

from . import _lib


def _call(name, *args):
    ext = _lib._ext or _lib.train_ext()
    try:
        return getattr(ext, name)(*args)
    except TypeError as e:                       # an argument that is no tensor, number or flag where one belongs
        raise _lib.AtlasHipError(f"{name}: {str(e).split(chr(10) + 'Invoked')[0]}") from None


def attention(q, k, v, q_offsets, k_offsets=None, *, max_q=None, max_k=None, key_mask=None, scale=None, keep=None, keep_scale=1.0):
    """Attention of packed sequences: out[t, h] = sum_j P[t, h, j] keep[t, h, j] keep_scale v[j, h'] with P = softmax_j(scale q[t, h] . k[j, h'])

    q [Tq, H, D]; k, v [Tk, H', D], H a multiple of H' (query head h reads key head h' = h // (H / H')); views of a fused projection are
    read in place. Sequence b is rows q_offsets[b] : q_offsets[b + 1] of q and k_offsets[b] : k_offsets[b + 1] of k and v (int32
    [batch + 1] on the device, non-decreasing; k_offsets defaults to q_offsets). D: a multiple of 8, at most 128.

    max_q, max_k    the longest sequence, as far as the host knows it (launch sizes; default: all rows)
    key_mask        bool [Tk]: False hides a key (its k and v are not used, whatever they hold)
    keep            bool [Tq, H, C]: dropout decisions, column j for key j of the row's sequence (columns from C on count as dropped)
    scale           default 1 / sqrt(D); positive

    A row that sees no key gives zeros and takes and gives no gradient; rows of q that belong to no sequence likewise. In 16 bits the
    probabilities and their gradients are rounded to the tensors' type before the matrix products (fp16: scaled into its range); what rounding leaves of
    the output is kept for the backward pass in another byte a value."""
    return _call("attention", q, k, v, q_offsets, k_offsets, max_q, max_k, key_mask, scale, keep, keep_scale)


class Compressed:
    """An activation in 8 bits: e4m3 codes with a power of two for every 32 values of a row (1.03 bytes a value). `decode()` gives the values back."""

    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes, scales, shape, dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, shape, dtype

    def decode(self, dtype=None):
        """the values that the codes stand for, rounded to `dtype` (default: the compressed tensor's)"""
        return _call("decompress", self.codes, self.scales, self.shape, self.dtype if dtype is None else dtype)


def compress(x):
    """`x` (at least one dimension) in 8 bits. Every 32 consecutive values of the last dimension share a power of two, the smallest that keeps
    them within 448; a value is rounded to nearest even in e4m3: off by at most 1/16 of itself or 2^-17 of the group's largest. Values that are
    not finite come back as NaN and disturb no other. Not differentiable: what comes back is cut off from x's graph (and from a
    forward-mode tangent)."""
    return Compressed(*_call("compress", x), x.shape, x.dtype)


def linear(x, weight, bias=None, *, activation=None, keep=None, keep_scale=1.0, residual=None, checkpoint=None):
    """y = act(x weight^T + bias) * (keep ? keep_scale : 0) + residual, one product with everything else in its epilogue, rounded once

    x [..., K], weight [N, K], bias [N], residual and keep [..., N]; activation None or "gelu" (exact erf form); keep: bool, the dropout's
    decisions. The pre-activation is kept for the backward pass in the tensors' dtype, and its gradient is rounded to that before the products of x.grad and
    weight.grad (not for bias.grad). checkpoint="e4m3" keeps x and the pre-activation for the backward pass in 8 bits (see `compress`; the pre-activation is
    rounded from fp32): weight.grad and the activation's slope are then those of the 8-bit values, x.grad and bias.grad otherwise exact."""
    return _call("linear", x, weight, bias, activation, keep, keep_scale, residual, checkpoint)


def layer_norm(x, weight, bias, eps=1e-12):
    """y = weight (x - mean(x)) / sqrt(mean(x^2) + eps) + bias over the last dimension: the reference's BertLayerNorm, whose scale is the root of the
    UNCENTRED second moment (src/modeling_bert.py:104-114)"""
    return _call("layer_norm", x, weight, bias, eps)
