"""`Contriever.training_kernels_enable()`: the retriever's training forward on the kernels of atlas_amd.train_ops. On the CPU: the switch, what it refuses
and what it leaves as it was. On the GPU: embeddings and every parameter's gradient against the module's own torch operators."""
import types

import pytest
import torch

from atlas_amd import _lib, retrievers as R
from test_retriever_training import VOCAB, _batch, _cfg, _randomize


def _loss(emb):
    w = torch.randn(emb.shape, generator=torch.Generator().manual_seed(3))
    return (emb.double() * w.to(emb.device)).sum()


def test_the_switch_and_its_refusals():
    m = _randomize(R.Contriever(_cfg(1)), 1)
    keys = set(m.state_dict())
    ids, mask, tt = _batch(3, 12, 5)
    m.eval()
    want = m(ids, mask, tt)
    assert m.last_path == "autograd"
    m.training_kernels_enable()
    with pytest.raises(_lib.AtlasHipError, match="MI355X"):                # CPU tensors: no fallback
        m(ids, mask, tt)
    assert m.last_path == "kernels" and set(m.state_dict()) == keys
    with pytest.raises(ValueError):
        m.training_kernels_enable(checkpoint="int4")
    m.training_kernels_disable()
    assert torch.equal(m(ids, mask, tt), want) and m.last_path == "autograd"
    r = R.UntiedDualEncoderRetriever(types.SimpleNamespace(query_side_retriever_training=False), m, R.Contriever(_cfg(1)))
    r.training_kernels_enable("e4m3")
    assert all(c.training_kernels and c.activation_checkpoints == "e4m3" for c in r.children())
    r.training_kernels_disable()
    assert not any(c.training_kernels for c in r.children())


def _pair(layers, dtype, pooling="average", seed=7):
    mine = _randomize(R.Contriever(_cfg(layers), pooling=pooling), seed).to(dtype).cuda().train()
    ref = R.Contriever(_cfg(layers), pooling=pooling)
    ref.load_state_dict(mine.state_dict())
    ref = ref.double().train()                                              # torch operators in 64 bits (norm statistics in 32), on the CPU
    for mod in [*mine.modules(), *ref.modules()]:
        if isinstance(mod, torch.nn.Dropout):
            mod.p = 0.0
    return mine, ref


def _errors(mine, ref, got, want):
    err = {"emb": float((got.detach().double().cpu() - want.detach()).norm() / want.detach().norm())}
    theirs = dict(ref.named_parameters())
    for n, p in mine.named_parameters():
        g = theirs[n].grad
        if "key.bias" in n:                     # mathematically zero: what is there is rounding, judged against the key weight's gradient below
            continue
        err[n] = float((p.grad.double().cpu() - g).norm() / (g.norm() + 1e-30))
    return err


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pooling,checkpoint,again,bound", [
    (torch.float32, "average", None, False, 1e-4), (torch.float32, "sqrt", None, True, 1e-4), (torch.float32, "cls", None, False, 1e-4),
    (torch.bfloat16, "average", None, False, 0.1), (torch.float16, "average", None, True, 0.02), (torch.bfloat16, "average", "e4m3", False, 0.2),
    (torch.float32, "average", "e4m3", True, 0.15),
])
def test_embeddings_and_gradients_are_the_modules_own(dtype, pooling, checkpoint, again, bound):
    """Relative 2-norms over two layers. Between the loss and the deepest parameter lie about 25 roundings, each at most u = eps / 2 of its value, adding at
    worst linearly: 25 u = 0.098 (bf16), 0.012 (fp16); fp32: 25 sums of up to 768 terms (or the batch's 200 tokens), 25 * 768 * 2^-24 / sqrt(768) = 4e-5,
    and the reference's norm statistics in 32 bits. 8-bit checkpoints: every dense layer's weight gradient is off by at most 2^-4 of each term, and the
    slope's error (0.8 * 2^-4 |z|, two layers) passes on to what lies below: 0.0625 + 2 * 0.05 at worst"""
    mine, ref = _pair(2, dtype, pooling)
    ids, mask, tt = _batch(9, 41, 11, holes=True)
    mine.training_kernels_enable(checkpoint)
    if again:
        mine.gradient_checkpointing_enable()
    got = mine(ids.cuda(), mask.cuda(), tt.cuda())
    assert mine.last_path == "kernels" and got.dtype == mine._out_dtype()
    _loss(got).backward()
    want = ref(ids, mask, tt)
    _loss(want).backward()
    err = _errors(mine, ref, got, want)
    assert len(err) > 30 and max(err.values()) <= bound, sorted(err.items(), key=lambda e: -e[1])[:5]
    for a, b in zip(mine.encoder.layer, ref.encoder.layer):
        assert float(a.attention.self.key.bias.grad.double().norm()) <= bound * float(b.attention.self.key.weight.grad.norm())
    # the same bits again
    first = {n: p.grad.clone() for n, p in mine.named_parameters() if "word_embeddings" not in n}       # (torch's own embedding backward sums with atomics)
    mine.zero_grad()
    _loss(mine(ids.cuda(), mask.cuda(), tt.cuda())).backward()
    same = [n for n, g in first.items() if "embeddings" not in n and not torch.equal(g, dict(mine.named_parameters())[n].grad)]
    assert not same, same


@pytest.mark.gpu
def test_dropout_and_a_step_through_the_wrapper():
    """train mode with dropout: the same generator state gives the same embeddings, another one others; the two-encoder step of src/atlas.py:457-465
    reaches every parameter of both encoders; an all-padding passage is NaN under 'average' (0 / 0) as in the reference and spoils no other row"""
    opt = types.SimpleNamespace(query_side_retriever_training=False)
    r = R.UntiedDualEncoderRetriever(opt, _randomize(R.Contriever(_cfg(1)), 1), _randomize(R.Contriever(_cfg(1)), 2)).bfloat16().cuda().train()
    r.training_kernels_enable("e4m3")
    qi, qm, _ = (t.cuda() for t in _batch(2, 9, 31))
    pi, pm, _ = (t.cuda() for t in _batch(6, 14, 32))
    embs = []
    for seed in (5, 5, 6):
        torch.manual_seed(seed)
        embs.append(r(input_ids=pi, attention_mask=pm, is_passages=True))
    assert torch.equal(embs[0], embs[1]) and not torch.equal(embs[0], embs[2])
    q, p = r(input_ids=qi, attention_mask=qm, is_passages=False), embs[0].view(2, 3, -1)
    score = (q.float()[:, None] * p.float()).sum(-1)
    torch.log_softmax(score, -1)[:, 0].sum().backward()
    for n, t in r.named_parameters():
        assert t.grad is not None and bool(torch.isfinite(t.grad).all()), n
        assert bool(t.grad.any()) or "type" in n or "position" in n or "key.bias" in n, n
    pm = pm.clone()
    pm[1] = 0
    emb = r(input_ids=pi, attention_mask=pm, is_passages=True)
    assert bool(emb[1].isnan().all()) and bool(torch.isfinite(emb[[0, 2, 3, 4, 5]]).all())
    with torch.no_grad():                                                    # inference is the eval-mode encoder, as before
        r.eval()(input_ids=pi, attention_mask=pm, is_passages=True)
    assert r.passage_contriever.last_path == "hip"


class _Adapter(torch.nn.Module):
    """a wrapper with a forward of its own that keeps the weights of what it wraps in sight"""

    def __init__(self, base):
        super().__init__()
        self.base, self.more = base, torch.nn.Linear(base.in_features, base.out_features)

    weight = property(lambda self: self.base.weight)
    bias = property(lambda self: self.base.bias)

    def forward(self, x):
        return self.base(x) + self.more(x)


class _Doubled(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


class _NoDropout(torch.nn.Dropout):
    def forward(self, x):
        return x


def test_modules_that_do_more_than_their_weights_are_refused():
    """the kernels read a dense layer's weights and a dropout's probability and never call the modules: hooks, adapters and forwards of their own would be lost"""
    ids, mask, tt = _batch(3, 12, 5)
    path = ["attention.self.query", "attention.self.key", "attention.self.value", "attention.self.dropout", "attention.output.dense", "attention.output.dropout",
            "intermediate.dense", "output.dense", "output.dropout"]

    def outcome(m):
        m.training_kernels_enable()
        with pytest.raises(_lib.AtlasHipError) as e:
            m(ids, mask, tt)
        return "MI355X" if "run on an MI355X only" in str(e.value) else str(e.value)          # (plain modules come as far as the CPU tensors' refusal)

    m = _randomize(R.Contriever(_cfg(2)), 1).train()
    assert outcome(m) == "MI355X"
    last = m.encoder.layer[1]
    nothing = lambda *a: None  # noqa: E731
    for name in path:
        sub = last.get_submodule(name)
        for handle in (sub.register_forward_hook(nothing), sub.register_forward_pre_hook(nothing), sub.register_full_backward_hook(nothing),
                       sub.register_full_backward_pre_hook(nothing)):
            pass
        assert "encoder.layer.1." + name in outcome(m) and "hook" in outcome(m)
        for hooks in (sub._forward_hooks, sub._forward_pre_hooks, sub._backward_hooks, sub._backward_pre_hooks):
            hooks.clear()
        sub.forward = nothing                                                # replaced on the instance
        assert "encoder.layer.1." + name in outcome(m)
        del sub.forward
        other = _NoDropout() if "dropout" in name else _Adapter(sub)
        parent = last.get_submodule(name.rpartition(".")[0])
        setattr(parent, name.rpartition(".")[2], other)
        assert "encoder.layer.1." + name in outcome(m)
        setattr(parent, name.rpartition(".")[2], sub)
        assert outcome(m) == "MI355X"
    handle = torch.nn.modules.module.register_module_forward_hook(nothing)
    try:
        assert "hook" in outcome(m)
    finally:
        handle.remove()
    # the embedding of token types is read, not called, where the call has none
    sub = m.embeddings.token_type_embeddings
    handle = sub.register_forward_hook(nothing)
    assert outcome(m) == "MI355X"
    m.training_kernels_enable()
    with pytest.raises(_lib.AtlasHipError, match="token_type_embeddings"):
        m(ids, mask)
    handle.remove()
    # weights that are computed when they are read are right; computed by a hook, they would be stale
    dense = last.output.dense
    torch.nn.utils.parametrizations.weight_norm(dense)
    assert outcome(m) == "MI355X"
    torch.nn.utils.parametrize.remove_parametrizations(dense, "weight")
    last.output.dense = _Doubled(dense.in_features, dense.out_features)
    assert "encoder.layer.1.output.dense" in outcome(m)
    # and the module's own operators take all of them
    m.training_kernels_disable()
    assert m(ids, mask, tt).shape == (3, 768)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_gradient_but_the_tables_is_the_same_bits_again(dtype):
    """(torch's backward pass of an embedding table sums with atomics)"""
    m, _ = _pair(1, dtype)
    ids, mask, tt = (t.cuda() for t in _batch(9, 41, 11, holes=True))
    m.training_kernels_enable()
    grads = []
    for _ in range(2):
        m.zero_grad()
        _loss(m(ids, mask, tt)).backward()
        grads.append({n: p.grad.clone() for n, p in m.named_parameters() if not n.endswith("_embeddings.weight")})
    assert "embeddings.LayerNorm.weight" in grads[0] and "embeddings.LayerNorm.bias" in grads[0] and len(grads[0]) >= 18
    assert all(torch.equal(grads[0][n], grads[1][n]) for n in grads[0])
