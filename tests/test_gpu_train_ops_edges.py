"""The operators of a retriever training step (atlas_amd.train_ops) on the GPU at the ends of what they promise: pre-activations beyond a type's range, no
sequences at all, so many keys that a probability is below fp16's steps, norms of very small and very large rows. Against the formulas in 64 bits."""
import pytest
import torch

import train_ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from atlas_amd import train_ops

    return train_ops


def _ends(*lens):
    return torch.tensor([0, *lens], dtype=torch.int32, device="cuda").cumsum(0).int()


# ---- dense layer -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("drop", [False, True])
@pytest.mark.parametrize("dtype,big", [("fp16", 2.0 ** 8), ("bf16", 2.0 ** 70), ("fp32", 2.0 ** 70)])
def test_gelu_slope_of_infinite_pre_activations(dtype, big, drop, ops):
    """z = +-4 big^2: 2^18 is beyond fp16 and saved as infinity, 2^142 is infinite in fp32 already. The slope is 1 or 0 there (0.5 at z = 0), so with small whole
    numbers as dy every term is a whole number times 1 or big and every sum stays below 2^8 of them: exact in all three types"""
    g = torch.Generator().manual_seed(8)
    kind, feature = torch.arange(41) % 3, torch.arange(11) % 3
    x = torch.where(kind > 0, big, 0.0).double()[:, None].expand(41, 4)
    w = torch.tensor([-big, big, 0.0]).double()[feature][:, None].expand(11, 4)
    dy = 2.0 * torch.randint(-1, 2, (41, 11), generator=g).double()
    keep = torch.rand((41, 11), generator=g) < 0.5 if drop else None
    times = keep.double() * 2 if drop else torch.ones(41, 11).double()
    z = x @ w.T
    dz = dy * times * torch.where(z > 0, 1.0, torch.where(z < 0, 0.0, 0.5))
    want = {"dx": dz @ w, "dw": dz.T @ x, "db": dz.sum(0)}
    leaves = [t.to(DT[dtype]).cuda().requires_grad_() for t in (x, w, torch.zeros(11))]
    y = ops.linear(*leaves, activation="gelu", keep=None if keep is None else keep.cuda(), keep_scale=2.0 if drop else 1.0)
    assert torch.equal(y.detach().double().cpu(), torch.where((z > 0) & (times > 0), torch.inf, 0.0).double())
    for name, got in zip(want, torch.autograd.grad(y, leaves, dy.to(DT[dtype]).cuda())):
        assert torch.equal(got.double().cpu(), want[name]), name


def test_linear_of_2_to_the_30_rows(ops):
    """as many tiles as there can be: a launch takes less than 2^32 threads"""
    x = torch.randint(-100, 100, (1 << 30, 1), dtype=torch.int8, device="cuda").half()
    y = ops.linear(x, torch.full((1, 1), 2.0, dtype=torch.float16, device="cuda"))
    assert torch.equal(y, x.mul_(2))


# ---- attention -------------------------------------------------------------------------------------------------------------
def _norm_check(name, got, want, units):
    """in the 2-norm: `units` roundings of 2^-11 of a value, and half an fp16 step where a result is below 2^-14"""
    off_by, bound = float((got.double() - want).norm()), units * 2.0 ** -11 * float(want.norm()) + 2.0 ** -25 * want.numel() ** 0.5
    assert off_by <= bound, (name, off_by / float(want.norm()), bound / float(want.norm()))


@pytest.mark.parametrize("n", [4000, 65536, 262144])
def test_fp16_value_gradients_of_many_keys(n, ops):
    """near-uniform attention: every probability is about 1 / n, below 2^-14 where fp16 loses bits. Two roundings, of P as a product's operand and of the result; the
    fp32 sums (n terms in the softmax, 64 in dv) add less than half of one"""
    g = torch.Generator(device="cuda").manual_seed(n)
    rnd = lambda rows, std: (torch.randn(rows, 1, 64, generator=g, device="cuda") * std).half()  # noqa: E731
    q, k, v, dy = rnd(64, 0.25), rnd(n, 0.25), rnd(n, 1.0), rnd(64, 256.0)
    leaf = v.clone().requires_grad_()
    (got,) = torch.autograd.grad(ops.attention(q, k, leaf, _ends(64), _ends(n)), leaf, dy)
    p = torch.softmax(q.double()[:, 0] @ k.double()[:, 0].t() / 8, 1)
    _norm_check("dv", got[:, 0], p.t().contiguous() @ dy.double()[:, 0], 2.5)


def test_fp16_value_gradient_of_a_key_that_every_row_sees_a_little(ops):
    """4000 rows give the last of 4001 keys e^-11 / 4000 each: far below half of fp16's smallest step, and 1.3e-4 together. All rows round alike: two roundings and the fp32
    sums of 4000 terms, element by element"""
    q, k, v, dy = (torch.zeros(n, 1, 64, device="cuda", dtype=torch.float16) for n in (4000, 4001, 4001, 4000))
    q[:, 0, 0], k[-1, 0, 0], dy[:] = 8.0, -11.0, 8.0
    leaf = v.requires_grad_()
    (got,) = torch.autograd.grad(ops.attention(q, k, leaf, _ends(4000), _ends(4001)), leaf, dy)
    p = torch.softmax(torch.tensor([0.0] * 4000 + [-11.0], dtype=torch.float64), 0)
    want = (p * 4000 * 8.0)[:, None].expand(4001, 64)
    assert float(want[-1, 0]) > 1e-4
    off_by = (got.double().cpu()[:, 0] - want).abs()
    assert bool((off_by <= (2 * 2.0 ** -11 + 4000 * 2.0 ** -24) * want).all()), (float(off_by[-1].max()), float(want[-1, 0]))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens,std,drop", [([1] * 30, 1.2, 0), ([2] * 100, 1.2, 0), ([2] * 100, 3.0, 0), ([9] * 30, 6.0, 0), ([9] * 30, 3.0, 0.2), ([200, 70, 130], 6.0, 0),
                                           ([1500], 6.0, 0.1), ([700] * 6, 3.0, 0)])
def test_gradients_of_rows_that_one_key_dominates(lens, std, drop, dtype, ops):
    """There dS is small beside its two terms, P dP and P delta, and an error of delta is one of every dS of the row. Of delta = sum_j P_j M_j dP_j the forward pass
    rounds every P_j but the largest, which is a power of 2 to it, and the output's own rounding comes along in steps of 1/127 of it. In the 2-norm, roundings as independent
    errors of at most u = eps / 2 of the value (their mean square is a third of that or less, so a sum of hundreds stays below): of the result, of dS_j, of the P_j in delta; fp32
    sums at their worst"""
    g = torch.Generator(device="cuda").manual_seed(len(lens))
    heads, dim, total = 3, 64, sum(lens)
    rnd = lambda s: (torch.randn(total, heads, dim, generator=g, device="cuda") * s).to(DT[dtype])  # noqa: E731
    q, k, v, do = rnd(std), rnd(std), rnd(1.2), rnd(0.1)
    keep = (torch.rand((total, heads, max(lens)), generator=g, device="cuda") >= drop) if drop else None
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    y = ops.attention(*leaves, _ends(*lens), max_q=max(lens), max_k=max(lens), keep=keep, keep_scale=1 / (1 - drop))
    got = dict(zip(("dq", "dk"), torch.autograd.grad(y, leaves, do)))
    u, t, f = train_ref.unit(DT[dtype]), train_ref.tiny(DT[dtype]), 2.0 ** -24
    off_by, squares = ({n: 0.0 for n in got} for _ in range(2))
    at = 0
    for n in lens:
        rows = slice(at, at + n)
        at += n
        for h in range(heads):
            Q, K, V, D = (x[rows, h].double() for x in (q, k, v, do))
            S = Q @ K.t().contiguous() / 8
            P = torch.softmax(S, 1)
            M = torch.ones_like(P) if keep is None else keep[rows, h, :n].double() / (1 - drop)
            uf = u + 4 * f * (1.5 * float(S.abs().amax()) + 8)                               # and the error of an exponent
            dP = D @ V.t().contiguous()
            terms = P * M * dP
            delta = terms.sum(1, keepdim=True)
            others = (terms * terms).sum(1, keepdim=True) - terms.gather(1, S.argmax(1, keepdim=True)) ** 2
            O = (P * M) @ V
            sums = 2 * (dim + 8) * f * (D.abs() * ((P * M) @ V.abs())).sum(1, keepdim=True)
            edelta = uf ** 2 * others + (u / 127) ** 2 * (D * O).square().sum(1, keepdim=True) + sums ** 2
            dS = P * (M * dP - delta)
            edS = (uf * dS) ** 2 + (P * 2 * (dim + 8) * f * M * (D.abs() @ V.abs().t().contiguous())) ** 2
            want = {"dq": dS @ K / 8, "dk": dS.t().contiguous() @ Q / 8}
            err = {"dq": (edS @ K ** 2 + edelta * (P @ K) ** 2) / 64, "dk": ((edS + P ** 2 * edelta).t().contiguous() @ Q ** 2) / 64}
            for name in got:
                off_by[name] += float((got[name][rows, h].double() - want[name]).square().sum())
                squares[name] += float((err[name] + (u * want[name]) ** 2 + t ** 2).sum())
    for name in got:
        assert off_by[name] <= squares[name], (name, (off_by[name] / squares[name]) ** 0.5)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,heads,first", [(4096, 8, 0.34375), (4096, 8, 0.1), (65536, 4, 0.7)])
def test_fp32_sums_of_many_equal_terms(n, heads, first, dim, ops):
    """equal terms that are no power of 2 round one way: a chain of m sums of them is off by at most m 2^-25 of the result. Sixteen keys are summed by themselves, four an
    instruction, and then joined: n / 16 + 4 sums, and some 30 roundings besides; twice that for out, which is a sum over a sum, and four times for dv, whose terms have one in them"""
    rows = 4096
    q, k, v = (torch.zeros(m, heads, dim, device="cuda") for m in (rows, n, n))
    q[:, :, 0], k[0, :, 0], v[:] = dim ** 0.5, first, 1.0
    v[:, :, 1] = torch.arange(n, device="cuda")[:, None] % 2
    leaf = v.clone().requires_grad_()
    y = ops.attention(q, k, leaf, _ends(rows), _ends(n))
    (dv,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    p = torch.softmax(torch.cat([torch.full((1,), first), torch.zeros(n - 1)]).double(), 0).cuda()
    chain = (n / 16 + 4 + 30) * 2.0 ** -25
    for name, got, want, bound in (("out", y, (p[:, None] * v[:, 0].double()).sum(0)[None, None], 2 * chain), ("dv", dv, (p * rows)[:, None, None], 4 * (rows / 16 + 34) * 2.0 ** -25)):
        off_by = float(((got.double() - want) / want).abs().max())
        assert off_by <= bound, (name, off_by, bound)


def test_fp16_many_small_probabilities_beside_a_large_one(ops):
    """one key holds nearly all of a row, 65 535 others about 2^-25.6 of it each and 2^-9.6 together, which is the whole result where the first key's value is 0. Two
    roundings (of P and of the result), and fp32 sums of terms of one sign that add less than half of one"""
    g = torch.Generator(device="cuda").manual_seed(6)
    n, rows, heads = 65536, 4096, 8
    q, k = torch.zeros(rows, heads, 64, device="cuda"), torch.zeros(n, heads, 64, device="cuda")
    q[:, :, 0] = 8.0
    k[:, :, 0] = -0.5 * torch.rand(n, heads, generator=g, device="cuda")
    k[0, :, 0] = 17.5
    v = torch.rand(n, heads, 64, generator=g, device="cuda") + 0.5
    v[0] = 0
    q, k, v = q.half(), k.half(), v.half()
    got = ops.attention(q, k, v, _ends(rows), _ends(n))
    assert torch.equal(got, got[:1].expand_as(got))                        # (every row is the same one)
    p = torch.softmax(k[:, :, 0].double(), 0)
    want = (p[:, :, None] * v.double()).sum(0)
    off_by = (got[0].double() - want).abs()
    assert bool((off_by <= 2.5 * 2.0 ** -11 * want).all()), (float((off_by / want).max()), float(want.min()))


@pytest.mark.parametrize("rows,heads", [(10, 2), (1000, 1), (4000, 12)])
def test_attention_without_sequences(rows, heads, ops):
    """rows that belong to no sequence give zeros and take no gradient, however many there are"""
    q, k, v = (torch.randn(rows, heads, 64, device="cuda").bfloat16().requires_grad_() for _ in range(3))
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    for kw in ({}, {"max_q": 0, "max_k": 0}, {"keep": torch.ones(rows, heads, 40, dtype=torch.bool, device="cuda"), "keep_scale": 1.25}):
        y = ops.attention(q, k, v, none, **kw)
        assert not y.any() and not any(t.any() for t in torch.autograd.grad(y, (q, k, v), torch.ones_like(y)))


@pytest.mark.parametrize("dtype", list(DT))
def test_attention_of_nothing(dtype, ops):
    """no keys at all, no queries at all, neither: zeros, and nothing to read"""
    for rows, keys in ((70, 0), (0, 70), (0, 0)):
        q, k, v = (torch.randn(n, 2, 64, device="cuda").to(DT[dtype]).requires_grad_() for n in (rows, keys, keys))
        for kw in ({}, {"key_mask": torch.ones(keys, dtype=torch.bool, device="cuda")}, {"keep": torch.ones(rows, 2, keys, dtype=torch.bool, device="cuda")}):
            y = ops.attention(q, k, v, _ends(0, rows), _ends(keys, 0), **kw)
            grads = torch.autograd.grad(y, (q, k, v), torch.ones_like(y))
            assert y.shape == q.shape and not y.any() and all(g.shape == t.shape and not g.any() for g, t in zip(grads, (q, k, v)))


# ---- layer norm ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("n", [768, 100, 4100, 7])
@pytest.mark.parametrize("size,eps", [(1e-14, 0.0), (1e16, 1e-12), (0.0, 1e-30)], ids=["small rows", "large rows", "zero rows"])
def test_layer_norm_gradients_of_very_small_and_very_large_rows(size, eps, n, dtype, ops):
    """the scale r of a row is 1e14, 1e-16 and 1e15 here: r^3 is no fp32 number, dx is"""
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, w, b, dy = ((rnd(37, n) * size).to(DT[dtype]), (1 + 0.1 * rnd(n)).to(DT[dtype]), rnd(n).to(DT[dtype]), rnd(37, n).to(DT[dtype]))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ops.layer_norm(*leaves, eps=eps)
    got = dict(zip(("y", "dx", "dw", "db"), (y, *torch.autograd.grad(y, leaves, dy))))
    for name, (value, bound) in train_ref.layer_norm(x, w, b, dy, eps).items():
        train_ref.check(name, got[name], value, bound)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n", [7, 64, 100, 264, 768, 1032, 2056, 4100])
def test_layer_norm_of_views(n, dtype, ops):
    """rows of wider tensors, on and off a 16-byte border, every second row, columns as rows; gradients that are views like these, and one value for all"""
    g = torch.Generator(device="cuda").manual_seed(n)
    rnd = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda") * std).to(DT[dtype])  # noqa: E731
    m = 83
    wide, dwide = rnd(2 * m, 2 * n + 16), rnd(2 * m, 2 * n + 16)
    w, b = rnd(n, std=0.1) + 1, rnd(2 * n, std=0.1)[::2]
    views = [lambda t: t[:m, 8 : 8 + n], lambda t: t[:m, 3 : 3 + n], lambda t: t[::2, :n], lambda t: t[:m, : 2 * n : 2], lambda t: t.reshape(-1)[: n * m].view(n, m).t()]
    for i, view in enumerate(views):
        for dy in (views[i - 1](dwide), dwide[:1, :1].expand(m, n)):
            x = view(wide)
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            y = ops.layer_norm(*leaves, eps=1e-12)
            got = dict(zip(("y", "dx", "dw", "db"), (y, *torch.autograd.grad(y, leaves, dy))))
            for name, (value, bound) in train_ref.layer_norm(x, w, b, dy, 1e-12).items():
                train_ref.check(f"{name} of view {i}", got[name], value, bound)


# ---- gradients that are more than values -----------------------------------------------------------------------------------
def test_a_gradient_with_a_tangent_is_refused(ops):
    """forward over reverse: the backward pass would drop the tangent of the gradient that it is given"""
    import torch.autograd.forward_ad as fw

    x, w, q = (torch.randn(s, device="cuda").requires_grad_() for s in ((30, 16), (16, 16), (30, 2, 8)))
    for y, leaf in ((ops.linear(x, w), x), (ops.layer_norm(x, w[0], w[1]), x), (ops.attention(q, q, q, _ends(30)), q)):
        with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, leaf, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))


def _flagged(t):
    """-t as torch holds the imaginary part of a conjugate: t's own memory, and a flag that says that the values are negative"""
    f = torch.complex(torch.zeros_like(t), t).conj().imag
    assert f.is_neg() and torch.equal(f, -t)
    return f


def test_values_and_gradients_whose_sign_is_a_flag(ops):
    """read as the values they are, whatever their strides (a last dimension of 1 has none that would need a copy)"""
    g = torch.Generator(device="cuda").manual_seed(9)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    x, w, b, r, one, q = rnd(30, 16), rnd(16, 16), rnd(16), rnd(30, 16), rnd(1), rnd(30, 2, 8)
    x1, w1 = rnd(30, 1), rnd(1, 1)
    off = _ends(30)
    calls = [(lambda x, w, b, r: ops.linear(x, w, b, residual=r), (x, w, b, r)), (lambda x, w, b, r: ops.linear(x, w, b, residual=r, checkpoint="e4m3"), (x1, w1, one, x1 + 1)),
             (ops.layer_norm, (x, b, b + 1)), (ops.layer_norm, (x1, one, one + 1)), (lambda q, k, v: ops.attention(q, k, v, off), (q, q + 1, q - 1)),
             (lambda x: ops.compress(x).decode(), (x1,))]
    for n, (call, tensors) in enumerate(calls):
        for i in range(len(tensors)):
            pairs = []
            for make in (_flagged, torch.neg):
                leaves = [t.clone().requires_grad_() for t in tensors]
                args = list(leaves)
                args[i] = make(leaves[i])
                y = call(*args)
                dy = make(rnd(*y.shape) * 0 + torch.arange(y.numel(), device="cuda").view(y.shape).float().sin())
                pairs.append([y] + (list(torch.autograd.grad(y, leaves, dy)) if y.requires_grad else []))
            assert all(torch.equal(a, b) for a, b in zip(*pairs)), (n, i)


# ---- what is kept for the backward pass, through hooks ----------------------------------------------------------------------
def _three(ops, dtype):
    """a step of each operator with everything that it can save: () -> [outputs and gradients]"""
    g = torch.Generator(device="cuda").manual_seed(12)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, w, b, q = (t.requires_grad_() for t in (rnd(70, 48), rnd(48, 48), rnd(48), rnd(70, 6, 24)))
    off, keep, seen = _ends(30, 40), torch.rand((70, 6, 40), generator=g, device="cuda") >= 0.2, torch.rand(70, generator=g, device="cuda") >= 0.2
    half = torch.rand((70, 48), generator=g, device="cuda") >= 0.5

    def step():
        ys = [ops.linear(x, w, b, activation="gelu", keep=half, keep_scale=2.0), ops.linear(x.t().contiguous().t(), w, b, activation="gelu", checkpoint="e4m3"),
              ops.layer_norm(x, b, b), ops.attention(*(t.unflatten(1, (2, 24)) for t in q.flatten(1).split(48, 1)), off, key_mask=seen, keep=keep[:, :2], keep_scale=1.25)]
        return ys, lambda: [t for y in ys for t in torch.autograd.grad(y, [l for l in ((q,) if y.dim() == 3 else (x, w, b) if y is not ys[2] else (x, b))], torch.ones_like(y))]

    return step


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_saved_tensors_that_hooks_give_back_in_another_layout(dtype, ops):
    """kept on the host and brought back; brought back with other strides; not brought back, which is refused"""
    from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

    step = _three(ops, DT[dtype])
    want = step()[1]()
    turned = saved_tensors_hooks(lambda t: t, lambda t: t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() else t)
    apart = saved_tensors_hooks(lambda t: t, lambda t: torch.stack([t, t], -1)[..., 0])
    for hooks in (save_on_cpu(), save_on_cpu(pin_memory=True), turned, apart):
        with hooks:
            backward = step()[1]
        for a, b in zip(backward(), want):
            assert torch.equal(a, b)
    with saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
        ys = step()[0]
    for y in ys:
        with pytest.raises(RuntimeError, match="came back on cpu"):
            y.backward(torch.ones_like(y))
