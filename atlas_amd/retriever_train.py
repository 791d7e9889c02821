"""The TRAINING forward of the Contriever module: the one call of the reference that needs autograd.

`Atlas.forward` embeds the query (and, unless `query_side_retriever_training`, the retrieved passages) with the retriever in
train mode, under autograd, and back-propagates the retriever loss through it (src/atlas.py:452-465); `set_dropout` has set every
`nn.Dropout` of the model to `opt.dropout` by then (src/model_io.py:103, src/util.py:161-164). That step is OUTSIDE the path this
package accelerates (index refresh, query embedding and search run under `torch.no_grad()` on the HIP encoder and never come
here) -- but a drop-in retriever has to survive it, so `Contriever.forward` hands exactly two cases to this file:

    * autograd is on and a parameter requires grad                       (retriever training)
    * the module is in train mode with a non-zero dropout probability    (the reference would drop activations; the HIP
                                                                          encoder is an eval-mode encoder)

Everything here is written with torch operators on the module's own parameters, so torch's autograd provides the backward and the
optimizer / DDP / ShardedDDP wrappers of the reference see ordinary leaves. The operations, their order and the dtype at every step
are those of the reference's BERT (src/modeling_bert.py: embeddings 213-247, LayerNorm 104-114, self-attention 290-366 with the
softmax in fp32 :352, self-output 382-387, intermediate 448-451, output 461-466, encoder loop incl. gradient checkpointing
575-625) and of `Contriever.forward` (src/retrievers.py:49-60), including the four dropout sites (:246, :356, :384, :463) in that
order -- on the CPU, with the same generator state, the result and the gradients are bit-identical to the reference module
(tests/test_retriever_training.py). It is plumbing around the product, not the product: no HIP kernel is involved and nothing in
`bench.py` or the inference path may end up here (`Contriever.last_path` says which way a call went; the tests assert it).

`Contriever.training_kernels_enable()` serves the same two cases on the HIP kernels of `train_ops` instead (`kernel_training_forward`): the
same layers on packed tokens, a result rounded once where the operators above round after every step, and dropout decisions drawn in
another order (the same distribution, not the same masks).
"""
import math

import torch
import torch.nn.functional as F
import torch.utils.checkpoint


def _layer_norm(ln, x):
    """BertLayerNorm as the reference computes it (modeling_bert.py:104-114) -- NOT torch's LayerNorm: the scale is the root of the
    UNCENTRED second moment, statistics in fp32, the normalised value cast to a 16-bit weight's dtype before the affine step"""
    x32 = x.float()
    centred = x - torch.mean(x32, dim=-1, keepdim=True)
    y = centred * torch.rsqrt(torch.mean(x32.pow(2), dim=-1, keepdim=True) + ln.variance_epsilon)
    w = ln.weight
    if w.dtype.itemsize == 2:                      # fp16 / bf16 weights
        y = y.to(w.dtype)
    return w * y + ln.bias


def _embed(emb, input_ids, token_type_ids):
    seq = input_ids.shape[1]
    position_ids = emb.position_ids[:, :seq]
    if token_type_ids is None:
        token_type_ids = torch.zeros(input_ids.shape, dtype=torch.long, device=emb.position_ids.device)
    x = emb.word_embeddings(input_ids) + emb.token_type_embeddings(token_type_ids)
    x += emb.position_embeddings(position_ids)
    x = _layer_norm(emb.LayerNorm, x.float()).type_as(x)
    return emb.dropout(x)


def _heads(x, n_heads):
    b, s, h = x.shape
    return x.view(b, s, n_heads, h // n_heads).permute(0, 2, 1, 3)


def _layer(layer, n_heads, x, ext_mask):
    att = layer.attention.self
    q, k, v = _heads(att.query(x), n_heads), _heads(att.key(x), n_heads), _heads(att.value(x), n_heads)
    scores = torch.matmul(q, k.transpose(-1, -2))
    scores = scores / math.sqrt(q.shape[-1])
    scores = scores + ext_mask
    probs = F.softmax(scores.float(), dim=-1).type_as(scores)
    probs = att.dropout(probs)
    ctx = torch.matmul(probs, v).permute(0, 2, 1, 3).contiguous()
    ctx = ctx.view(ctx.shape[0], ctx.shape[1], -1)

    so = layer.attention.output                                   # BertSelfOutput
    a = so.dropout(so.dense(ctx)) + x
    a = _layer_norm(so.LayerNorm, a.float()).type_as(a)

    inter = F.gelu(layer.intermediate.dense(a))                   # ACT2FN["gelu"]: exact erf
    out = layer.output                                            # BertOutput
    y = out.dropout(out.dense(inter)) + a
    return _layer_norm(out.LayerNorm, y.float()).type_as(y)


def training_forward(model, input_ids, attention_mask, token_type_ids=None, normalize=False):
    """`Contriever.forward` (retrievers.py:22-60) of `model` (atlas_amd.retrievers.Contriever) with torch operators"""
    c = model.config
    dtype = model.embeddings.word_embeddings.weight.dtype
    if attention_mask is None:
        attention_mask = torch.ones(input_ids.shape, device=input_ids.device)
    # transformers 4.18 get_extended_attention_mask (the version the reference pins, requirements.txt:2)
    ext_mask = (1.0 - attention_mask[:, None, None, :].to(dtype)) * -10000.0
    x = _embed(model.embeddings, input_ids, token_type_ids)
    checkpointing = model.encoder.gradient_checkpointing and model.training
    for layer in model.encoder.layer:
        if checkpointing:
            x = torch.utils.checkpoint.checkpoint(_layer, layer, c.num_attention_heads, x, ext_mask, use_reentrant=False)
        else:
            x = _layer(layer, c.num_attention_heads, x, ext_mask)
    # retrievers.py:49-59: padded positions zeroed, then one of three poolings over the sequence axis
    if c.pooling not in _POOLINGS:
        raise ValueError(f"pooling={c.pooling!r}: the reference knows 'average', 'sqrt', 'cls' (retrievers.py:51-56)")
    hidden = x.masked_fill(attention_mask.unsqueeze(-1) == 0, 0.0)
    emb = _POOLINGS[c.pooling](hidden, attention_mask.sum(dim=1, keepdim=True))
    return F.normalize(emb, dim=-1) if normalize else emb


_POOLINGS = {
    "average": lambda hidden, count: hidden.sum(dim=1) / count,                       # integer count: true division in the sum's dtype
    "sqrt": lambda hidden, count: hidden.sum(dim=1) / count.float().sqrt(),           # fp32 divisor: promotes
    "cls": lambda hidden, count: hidden[:, 0],
}


def _keep(dropout, shape, device):
    """the decisions of an nn.Dropout as a bool tensor and what the kept values are multiplied by; (None, 1) where it does nothing"""
    if not dropout.training or dropout.p == 0.0:
        return None, 1.0
    if dropout.p >= 1.0:
        return torch.zeros(shape, dtype=torch.bool, device=device), 0.0
    return torch.empty(shape, dtype=torch.bool, device=device).bernoulli_(1.0 - dropout.p), 1.0 / (1.0 - dropout.p)


_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks")


def _read_modules(layer):
    att, so, out = layer.attention.self, layer.attention.output, layer.output
    return (att.query, att.key, att.value, so.dense, layer.intermediate.dense, out.dense), (att.dropout, so.dropout, out.dropout)


def _only_read(model, token_types):
    """The kernels read the weights (or the probability) of these modules and do not call them: one that does more when it is called -- hooks, an adapter, a forward of
    its own -- has to be refused, or what it does would be lost. (Weights that are computed when they are read, as parametrizations do, are fine.)"""
    from ._lib import AtlasHipError

    everywhere = torch.nn.modules.module
    if any(getattr(everywhere, "_global" + hooks, None) for hooks in _HOOKS):
        raise AtlasHipError("training kernels: a hook on every module is registered, and most modules are not called; training_kernels_disable() takes it")
    groups = [((model.embeddings.token_type_embeddings,), torch.nn.Embedding)] if not token_types else []
    for layer in model.encoder.layer:
        groups += zip(_read_modules(layer), (torch.nn.Linear, torch.nn.Dropout))
    for modules, kind in groups:
        for m in modules:
            own = m.__dict__
            if type(m).forward is not kind.forward or "forward" in own or own["_forward_hooks"] or own["_forward_pre_hooks"] or own["_backward_hooks"] or own["_backward_pre_hooks"]:
                name = next(n for n, other in model.named_modules() if other is m)
                raise AtlasHipError(f"training kernels: {name} is read and not called, and it has hooks or a forward of its own that would be lost; "
                                    "training_kernels_disable() takes it")


def _kernel_layer(layer, n_heads, x, offsets, longest, checkpoint):
    from . import train_ops as ops

    rows, hidden = x.shape
    att = layer.attention.self
    qkv = ops.linear(x, torch.cat([att.query.weight, att.key.weight, att.value.weight]), torch.cat([att.query.bias, att.key.bias, att.value.bias]),
                     checkpoint=checkpoint)
    q, k, v = (t.unflatten(1, (n_heads, hidden // n_heads)) for t in qkv.split(hidden, dim=1))
    keep, scale = _keep(att.dropout, (rows, n_heads, longest), x.device)
    ctx = ops.attention(q, k, v, offsets, max_q=longest, max_k=longest, keep=keep, keep_scale=scale).flatten(1)

    def dense_ln(out, h, residual):
        keep, scale = _keep(out.dropout, (rows, hidden), x.device)
        y = ops.linear(h, out.dense.weight, out.dense.bias, keep=keep, keep_scale=scale, residual=residual, checkpoint=checkpoint)
        return ops.layer_norm(y, out.LayerNorm.weight, out.LayerNorm.bias, out.LayerNorm.variance_epsilon)

    a = dense_ln(layer.attention.output, ctx, x)
    inter = layer.intermediate.dense
    return dense_ln(layer.output, ops.linear(a, inter.weight, inter.bias, activation="gelu", checkpoint=checkpoint), a)


def kernel_training_forward(model, input_ids, attention_mask, token_type_ids=None, normalize=False, checkpoint=None):
    """`training_forward` on the kernels of `train_ops`. Only tokens with attention_mask != 0 are rows (one host read of their number): hidden keys have
    probability exactly 0 in the reference and hidden tokens are dropped by the pooling, so leaving them out changes no result."""
    from . import train_ops as ops

    _only_read(model, token_type_ids is not None)
    c = model.config
    if c.pooling not in _POOLINGS:
        raise ValueError(f"pooling={c.pooling!r}: the reference knows 'average', 'sqrt', 'cls' (retrievers.py:51-56)")
    if attention_mask is None:
        attention_mask = torch.ones(input_ids.shape, device=input_ids.device)
    n, seq = input_ids.shape
    if seq > model.embeddings.position_ids.shape[1]:
        raise ValueError(f"sequences of {seq} tokens: the encoder has {model.embeddings.position_ids.shape[1]} positions")
    real = attention_mask != 0
    at = real.flatten().nonzero().squeeze(1)
    offsets = torch.zeros(n + 1, dtype=torch.int32, device=input_ids.device)
    offsets[1:] = real.sum(dim=1).cumsum(0)
    emb = model.embeddings
    x = emb.word_embeddings(input_ids.flatten()[at])
    x = x + (emb.token_type_embeddings(token_type_ids.flatten()[at]) if token_type_ids is not None else emb.token_type_embeddings.weight[0])
    x = x + emb.position_embeddings(emb.position_ids[0, at % max(1, seq)])
    x = emb.dropout(ops.layer_norm(x, emb.LayerNorm.weight, emb.LayerNorm.bias, emb.LayerNorm.variance_epsilon))
    recompute = model.encoder.gradient_checkpointing and model.training
    for layer in model.encoder.layer:
        args = (layer, c.num_attention_heads, x, offsets, seq, checkpoint)
        x = torch.utils.checkpoint.checkpoint(_kernel_layer, *args, use_reentrant=False) if recompute else _kernel_layer(*args)
    hidden = x.new_zeros((n * seq, x.shape[1])).index_copy(0, at, x).view(n, seq, x.shape[1])
    out = _POOLINGS[c.pooling](hidden, attention_mask.sum(dim=1, keepdim=True))
    return F.normalize(out, dim=-1) if normalize else out
