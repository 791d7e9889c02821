"""The operators of a retriever training step (atlas_amd.train_ops) on the GPU, against their formulas in 64 bits (train_ref.py, whose bounds are
derived there), at the sizes, strides and masks where kernels like these go wrong; and what a caller may do with them: other streams, captured
graphs, repeated calls, views."""
import itertools

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


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rnd(g, *shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _offsets(lens, first=0):
    ends = list(itertools.accumulate([first] + list(lens)))
    return ends, torch.tensor(ends, dtype=torch.int32, device="cuda")


def _grads(y, inputs, dy):
    return torch.autograd.grad(y, inputs, dy)


# ---- attention -----------------------------------------------------------------------------------------------------------
ATT = [
    # name, query lengths, key lengths (None: the same), heads, key heads, dim, hidden share, dropout, options
    ("one token", [1], None, 1, 1, 64, 0, 0, ""),
    ("two queries", [9, 31], None, 12, 12, 64, 0, 0, ""),
    ("tile edges", [63, 64, 65, 1, 128, 129], None, 2, 2, 64, 0, 0, ""),
    ("dropout", [40, 100, 7], None, 3, 3, 64, 0, 0.2, ""),
    ("hidden keys", [70, 130, 5], None, 2, 2, 64, 0.4, 0, "nan"),
    ("hidden all", [20, 33], None, 2, 1, 64, 1.0, 0, "nan"),
    ("hidden and dropout", [65, 90], None, 4, 2, 64, 0.3, 0.1, "nan"),
    ("shared heads", [17, 80], None, 8, 2, 64, 0, 0, ""),
    ("one key head", [33, 64], None, 6, 1, 64, 0, 0.1, ""),
    ("cross, empty ones", [5, 0, 70, 12, 1], [100, 30, 0, 1, 65], 4, 4, 64, 0, 0, ""),
    ("dim 8", [33, 70], None, 2, 2, 8, 0, 0, ""),
    ("dim 32", [33, 70], None, 2, 2, 32, 0, 0.1, ""),
    ("dim 80", [33, 70], None, 2, 1, 80, 0.2, 0, ""),
    ("dim 128", [50, 129], [200, 64], 4, 2, 128, 0.2, 0.1, "nan"),
    ("gaps", [30, 41], None, 2, 2, 64, 0, 0, "gaps"),
    ("short launch", [200, 150], None, 2, 2, 64, 0, 0, "short"),
    ("few columns", [40, 70], None, 2, 2, 64, 0, 0.1, "columns"),
    ("fused rows", [60, 77], None, 4, 2, 64, 0, 0, "fused"),
    ("odd strides", [60, 77], None, 2, 2, 64, 0, 0.1, "odd"),
    ("longer", [700], [1500], 2, 2, 64, 0.1, 0, ""),
    # walks split over workgroups in many parts, or not at all because there are workgroups enough
    ("one query, many keys", [1, 3, 0], [2000, 700, 50], 4, 1, 64, 0.1, 0.1, "nan"),
    ("one sequence, one key head", [900], None, 8, 1, 128, 0, 0, "gaps"),
    ("few rows, dropout, gaps", [40, 500], None, 2, 2, 32, 0, 0.2, "gaps"),
    ("some keys, none, hidden ones", [3, 5, 40], [2000, 0, 1500], 2, 2, 64, 1.0, 0, "nan"),
    ("many keys or none", [3, 5, 40], [2000, 0, 1500], 2, 1, 32, 0, 0.1, ""),
    ("full chip", [200, 190, 130, 65] * 6, None, 16, 16, 32, 0, 0.1, ""),
    ("full chip, hidden keys", [200, 190, 130, 65] * 6, [150, 200, 64, 190] * 6, 16, 16, 64, 0.2, 0, "nan"),
    ("full chip, shared heads", [200, 190, 130, 65] * 6, None, 16, 8, 64, 0, 0, ""),
]


def _attention_inputs(case, dtype, seed):
    name, ql, kl, heads, kv, dim, hidden, drop, opt = case
    g = _gen(seed)
    first, behind = (3, 5) if opt == "gaps" else (0, 0)
    qo, q_off = _offsets(ql, first)
    ko, k_off = _offsets(kl or ql, first)
    tq, tk = qo[-1] + behind, ko[-1] + behind
    rnd = lambda *s, **kw: _rnd(g, *s, dtype=dtype, **kw)  # noqa: E731
    if opt == "fused":
        q, k, v = (t.unflatten(1, (-1, dim)) for t in rnd(tq, (heads + 2 * kv) * dim, std=1.2).split([heads * dim, kv * dim, kv * dim], dim=1))
    elif opt == "odd":                                                   # a row stride that is no multiple of 16 bytes, heads outermost
        q, k, v = (rnd(n, h, dim + 3, std=1.2).transpose(0, 1)[:, :, 1:dim + 1] for n, h in ((heads, tq), (kv, tk), (kv, tk)))
    else:
        q, k, v = rnd(tq, heads, dim, std=1.2), rnd(tk, kv, dim, std=1.2), rnd(tk, kv, dim)
    do = rnd(tq, heads, dim, std=0.5)
    seen = (torch.rand(tk, generator=g, device="cuda") >= hidden) if hidden else None
    if opt == "nan":                                                     # what hidden rows hold must not matter
        k, v = k.clone(), v.clone()
        k[~seen], v[~seen] = float("nan"), float("inf")
    cols = max(kl or ql) - (9 if opt == "columns" else 0)
    keep = (torch.rand((tq, heads, cols), generator=g, device="cuda") >= drop) if drop else None
    kw = dict(key_mask=seen, keep=keep, keep_scale=1 / (1 - drop), max_q=64 if opt == "short" else max(ql), max_k=64 if opt == "short" else max(kl or ql))
    return q, k, v, do, qo, q_off, ko, k_off, kw


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("case", ATT, ids=[c[0] for c in ATT])
def test_attention_and_gradients(case, dtype, ops):
    q, k, v, do, qo, q_off, ko, k_off, kw = _attention_inputs(case, DT[dtype], 11)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*leaves, q_off, k_off, **kw)
    got = dict(zip(("out", "dq", "dk", "dv"), (out, *_grads(out, leaves, do))))
    seen = kw["key_mask"]
    kc, vc = (k, v) if seen is None else (torch.where(seen[:, None, None], t, 0) for t in (k, v))
    want = train_ref.attention(q, kc, vc, do, qo, ko, q.shape[2] ** -0.5, seen, kw["keep"], kw["keep_scale"])
    for n, (value, bound) in want.items():
        train_ref.check(n, got[n], value, bound)
    # rows of no sequence, and gradients of hidden keys: zeros, not merely small
    for n, off in (("out", qo), ("dq", qo), ("dk", ko), ("dv", ko)):
        assert not got[n][: off[0]].any() and not got[n][off[-1]:].any(), n
    if seen is not None:
        assert not got["dk"][~seen].any() and not got["dv"][~seen].any()
    # the same bits again, and with no graph
    again = ops.attention(*leaves, q_off, k_off, **kw)
    assert torch.equal(again, out) and all(torch.equal(a, got[n]) for a, n in zip(_grads(again, leaves, do), ("dq", "dk", "dv")))
    with torch.no_grad():
        assert torch.equal(ops.attention(*leaves, q_off, k_off, **kw), out)


def test_attention_gradient_against_differences(ops):
    """fp32: (f(x + h d) - f(x - h d)) / 2h along random directions. Truncation: f''' h^2 / 6 with f''' of order |f| here, h = 2^-6: 4e-5; rounding: fp32 sums
    of ~1e4 terms, 1e-6 relative to |loss terms| over 2h: 3e-5 of the loss's scale"""
    g = _gen(5)
    rnd = lambda *s: _rnd(g, *s, dtype=torch.float32)  # noqa: E731
    qo, off = _offsets([19, 70])
    leaves = [rnd(89, 4, 32), rnd(89, 2, 32), rnd(89, 2, 32)]
    do = rnd(89, 4, 32)
    f = lambda *x: (ops.attention(*x, off).double() * do).sum()  # noqa: E731
    req = [t.clone().requires_grad_() for t in leaves]
    grads = _grads(ops.attention(*req, off), req, do)
    scale = float((ops.attention(*leaves, off).double() * do).abs().sum())
    for i in range(3):
        d = rnd(*leaves[i].shape)
        d /= d.norm()
        h = 2.0 ** -6
        up, down = list(leaves), list(leaves)
        up[i], down[i] = leaves[i] + h * d, leaves[i] - h * d
        slope = float((f(*up) - f(*down)) / (2 * h))
        assert abs(slope - float((grads[i].double() * d).sum())) <= 1e-4 * (1 + scale / 100), i


def test_attention_views_int64_offsets_and_expanded_gradient(ops):
    q, k, v, do, qo, q_off, ko, k_off, kw = _attention_inputs(ATT[2], torch.bfloat16, 3)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    ref = ops.attention(*leaves, q_off)
    assert torch.equal(ref, ops.attention(*leaves, q_off.long(), q_off.long()))
    one = torch.ones((), dtype=q.dtype, device="cuda").expand(q.shape)
    for a, b in zip(_grads(ref, leaves, one), _grads(ops.attention(*leaves, q_off), leaves, one.contiguous())):
        assert torch.equal(a, b)


def test_attention_rows_beyond_32_bit_offsets(ops):
    """key rows 2^21 elements apart: the last ones lie beyond 2^31 elements"""
    n, stride = 1100, 1 << 21
    big = torch.empty(n * stride + 128, dtype=torch.bfloat16, device="cuda")
    kv = torch.as_strided(big, (n, 2, 64), (stride, 64, 1))
    small = _rnd(_gen(4), n, 2, 64, dtype=torch.bfloat16)
    kv.copy_(small)
    q = _rnd(_gen(5), 33, 1, 64, dtype=torch.bfloat16)
    qo, ko = (torch.tensor([0, e], dtype=torch.int32, device="cuda") for e in (33, n))
    do = _rnd(_gen(6), 33, 1, 64, dtype=torch.bfloat16)
    res = []
    for t in (kv, small):
        leaves = [x.detach().requires_grad_() for x in (q, t[:, :1], t[:, 1:])]
        out = ops.attention(*leaves, qo, ko)
        res.append((out, *_grads(out, leaves, do)))
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_attention_nan_in_a_visible_row_is_not_hidden(ops):
    q, k, v = (_rnd(_gen(7), 40, 2, 64, dtype=torch.float16) for _ in range(3))
    off = torch.tensor([0, 20, 40], dtype=torch.int32, device="cuda")
    q = q.clone()
    q[5, 1] = float("nan")
    out = ops.attention(q, k, v, off)
    assert bool(out[5, 1].isnan().all())
    out[5, 1] = 0
    assert bool(torch.isfinite(out).all())


# ---- dense layer ---------------------------------------------------------------------------------------------------------
LIN = [
    # rows, inner, outer
    (1, 1, 1), (1, 8, 8), (5, 7, 9), (1, 768, 768), (41, 768, 768), (64, 64, 64), (65, 33, 130), (130, 96, 200), (257, 100, 72), (300, 72, 64),
    (513, 256, 384), (700, 328, 264),
]
FORMS = [
    dict(), dict(gelu=True), dict(gelu=True, checkpoint=True), dict(bias=False), dict(residual=True, drop=0.1), dict(gelu=True, drop=0.3, residual=True),
    dict(gelu=True, drop=0.2, checkpoint=True, bias=False), dict(checkpoint=True),
]


def _linear_inputs(m, k, n, dtype, seed, bias=True, residual=False, drop=0.0, **_):
    g = _gen(seed)
    x, w = _rnd(g, m, k, dtype=dtype), _rnd(g, n, k, dtype=dtype, std=k ** -0.5)
    b = _rnd(g, n, dtype=dtype, std=0.2) if bias else None
    r = _rnd(g, m, n, dtype=dtype) if residual else None
    keep = (torch.rand((m, n), generator=g, device="cuda") >= drop) if drop else None
    return x, w, b, r, keep, _rnd(g, m, n, dtype=dtype, std=0.3)


def _check_linear(ops, x, w, b, r, keep, dy, form, device="cpu"):
    leaves = [t.detach().requires_grad_() for t in (x, w) + ((b,) if b is not None else ())]
    scale = 1 / (1 - form.get("drop", 0.0))
    res = r.detach().requires_grad_() if r is not None else None
    kw = dict(activation="gelu" if form.get("gelu") else None, keep=keep, keep_scale=scale, residual=res, checkpoint="e4m3" if form.get("checkpoint") else None)
    y = ops.linear(leaves[0], leaves[1], leaves[2] if b is not None else None, **kw)
    grads = _grads(y, leaves + ([res] if r is not None else []), dy)
    if r is not None:
        assert torch.equal(grads[-1], dy)
    got = dict(zip(("y", "dx", "dw", "db"), (y, *grads[: len(leaves)])))
    want = train_ref.linear(x, w, b, dy, form.get("gelu", False), keep, scale, r, form.get("checkpoint", False), device)
    for name, (value, bound) in want.items():
        train_ref.check(name, got[name], value, bound)
    return got


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("form", FORMS, ids=["-".join(f"{k}={v}" for k, v in f.items()) or "plain" for f in FORMS])
def test_linear_and_gradients(form, dtype, ops):
    for i, (m, k, n) in enumerate(LIN):
        print(form, dtype, m, k, n, flush=True)
        a = _linear_inputs(m, k, n, DT[dtype], 100 + i, **form)
        got = _check_linear(ops, *a, form)
        again = _check_linear(ops, *a, form)
        assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("form", [FORMS[0], FORMS[2], FORMS[5]], ids=["plain", "checkpoint", "everything"])
@pytest.mark.parametrize("m,k,n", [(6200, 72, 1000), (3104, 2056, 264), (23000, 520, 544), (25601, 96, 256), (256, 6400, 6144),
                                   (6201, 71, 1001), (2049, 2049, 2050), (33001, 129, 131), (21700, 136, 768), (21697, 768, 136)])
def test_linear_and_gradients_of_many_tiles(m, k, n, form, dtype, ops):
    """sizes whose products take the large tiles: ends inside a tile on every side, contractions that end inside a k-tile, split ones"""
    a = _linear_inputs(m, k, n, DT[dtype], 7, **form)
    got = _check_linear(ops, *a, form, "cuda")
    again = _check_linear(ops, *a, form, "cuda")
    assert all(torch.equal(got[x], again[x]) for x in got)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m,k,n", [(5000, 768, 768), (9000, 520, 1304), (700, 72, 264), (301, 100, 30)])
def test_weight_gradient_from_codes_is_that_of_their_values(m, k, n, dtype, ops):
    """the product reads the codes themselves: the same sums over the same values, bit for bit. Values over the whole range of the type, and NaN"""
    g = _gen(51)
    span = {"bf16": 60, "fp16": 6, "fp32": 60}[dtype]
    x = (_rnd(g, m, k, dtype=DT[dtype]).float() * torch.exp2(torch.randint(-span, span, (m, 1), generator=g, device="cuda").float())).to(DT[dtype])
    x[3, 5] = float("nan")
    w = _rnd(g, n, k, dtype=DT[dtype]).requires_grad_()
    dy = _rnd(g, m, n, dtype=DT[dtype], std=1e-3)
    (a,) = _grads(ops.linear(x, w, checkpoint="e4m3"), (w,), dy)
    (b,) = _grads(ops.linear(ops.compress(x).decode(), w), (w,), dy)
    assert bool(a[:, 5].isnan().all()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) and bool(torch.isfinite(a[:, :5]).all())


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_views(dtype, ops):
    """rows of a wider tensor, a transposed weight, an expanded gradient, three dimensions, unaligned storage"""
    g = _gen(9)
    wide = _rnd(g, 90, 200, dtype=DT[dtype])
    w = _rnd(g, 96, 72, dtype=DT[dtype], std=0.1)
    dy = _rnd(g, 90, 72, dtype=DT[dtype])
    for x in (wide[:, 8:104], wide[:, 3:99], wide[::2, :96]):
        _check_linear(ops, x, w.t(), None, None, None, dy[: x.shape[0]], {})
    x3 = _rnd(g, 5, 18, 96, dtype=DT[dtype])
    leaves = [x3.requires_grad_(), w.t().detach().requires_grad_()]
    y = ops.linear(*leaves, checkpoint="e4m3")
    assert y.shape == (5, 18, 72)
    one = torch.ones((), dtype=y.dtype, device="cuda").expand(y.shape)
    a, b = _grads(y, leaves, one)
    c, d = _grads(ops.linear(*leaves, checkpoint="e4m3"), leaves, one.contiguous())
    assert a.shape == x3.shape and torch.equal(a, c) and torch.equal(b, d)


def test_linear_no_rows_and_partial_gradients(ops):
    w, b = torch.randn(24, 16, device="cuda").bfloat16().requires_grad_(), torch.randn(24, device="cuda").bfloat16().requires_grad_()
    x = torch.empty(0, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    for kw in ({}, dict(activation="gelu"), dict(activation="gelu", checkpoint="e4m3")):
        y = ops.linear(x, w, b, **kw)
        assert y.shape == (0, 24)
        gx, gw, gb = _grads(y, (x, w, b), torch.empty_like(y))
        assert gx.shape == (0, 16) and not gw.any() and not gb.any() and gw.shape == w.shape
    x = torch.randn(30, 16, device="cuda").bfloat16()
    dy = torch.randn(30, 24, device="cuda").bfloat16()
    for kw in ({}, dict(activation="gelu"), dict(activation="gelu", checkpoint="e4m3")):
        xr = x.clone().requires_grad_()
        full = _grads(ops.linear(xr, w, b, **kw), (xr, w, b), dy)
        for i, one in enumerate((lambda: (xr, w.detach(), b.detach()), lambda: (x, w, b.detach()), lambda: (x, w.detach(), b))):
            args = one()
            assert torch.equal(_grads(ops.linear(*args, **kw), (args[i],), dy)[0], full[i])


def test_linear_gradient_against_differences(ops):
    g = _gen(15)
    rnd = lambda *s: _rnd(g, *s, dtype=torch.float32)  # noqa: E731
    x, w, b, dy = rnd(70, 33), rnd(45, 33) * 0.2, rnd(45), rnd(70, 45)
    f = lambda *a: (ops.linear(*a, activation="gelu").double() * dy).sum()  # noqa: E731
    req = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = _grads(ops.linear(*req, activation="gelu"), req, dy)
    scale = float((ops.linear(x, w, b, activation="gelu").double() * dy).abs().sum())
    for i in range(3):
        d = rnd(*req[i].shape)
        d /= d.norm()
        h = 2.0 ** -6
        up, down = [x, w, b], [x, w, b]
        up[i], down[i] = up[i] + h * d, down[i] - h * d
        slope = float((f(*up) - f(*down)) / (2 * h))
        assert abs(slope - float((grads[i].double() * d).sum())) <= 1e-4 * (1 + scale / 100), i


# ---- 8-bit activations ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 33), (5, 7), (2, 3, 64), (130, 100), (17, 768), (4, 4100), (96,)])
def test_compress_is_the_definition_bit_for_bit(shape, dtype, ops):
    x = _rnd(_gen(21), *shape, dtype=DT[dtype])
    x = (x.float() * torch.exp(2 * torch.randn(shape[-1], generator=_gen(22), device="cuda"))).to(DT[dtype])
    c = ops.compress(x)
    got = c.decode()
    assert got.dtype == x.dtype and got.shape == x.shape
    want = train_ref.eight_bits(x.double().cpu())
    assert torch.equal(got.double().cpu(), want)                       # four significant bits: exact in every dtype at these magnitudes
    assert torch.equal(c.decode(torch.float32).double().cpu(), want)
    assert torch.equal(ops.compress(got).decode(), got)                # once rounded, always the same


def test_compress_extremes(ops):
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(8, 64, device="cuda")
    x[0, 3], x[0, 40] = inf, 5.0
    x[1, :32], x[1, 33], x[1, 34] = nan, -inf, 3.0
    x[2, 0] = torch.finfo(torch.float32).max
    x[3, 0], x[3, 1] = 2.0 ** -149, -2.0 ** -130
    x[4] = torch.linspace(-448, 448, 64)
    x[5, 0], x[5, 1] = 448.0, 2.0 ** -9
    x[6, 0], x[6, 1], x[6, 2] = 449.0, 2.0 ** -9, 2.0 ** -8
    got = ops.compress(x).decode().double().cpu()
    want = train_ref.eight_bits(x.double().cpu())
    same = (got == want) | (got.isnan() & want.isnan())
    assert bool(same.all()), [(i, j, float(x[i, j]), float(got[i, j]), float(want[i, j])) for i, j in torch.nonzero(~same)[:8].tolist()]
    for dtype in DT.values():                                           # the largest values stay finite
        y = torch.zeros(2, 40, device="cuda", dtype=dtype)
        y[0, 0], y[0, 35], y[1, 1] = torch.finfo(dtype).max, -torch.finfo(dtype).max, torch.finfo(dtype).max * 0.95
        want = train_ref.eight_bits(y.double().cpu(), torch.finfo(dtype).max)
        assert bool(torch.isfinite(want).all()) and torch.equal(ops.compress(y).decode().double().cpu(), want)
    view = _rnd(_gen(23), 20, 100, dtype=torch.float16)[::2, 5:71]
    assert torch.equal(ops.compress(view).decode(), ops.compress(view.contiguous()).decode())
    assert ops.compress(torch.empty(0, 40, device="cuda")).decode().shape == (0, 40)


# ---- layer norm ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m,n", [(1, 1), (1, 768), (3, 7), (41, 768), (130, 100), (257, 264), (9, 4100), (700, 64)])
def test_layer_norm_and_gradients(m, n, dtype, ops):
    g = _gen(31)
    x = (_rnd(g, m, n, dtype=DT[dtype]).float() * torch.exp(torch.randn(n, generator=g, device="cuda")) + 0.3).to(DT[dtype])
    w, b, dy = _rnd(g, n, dtype=DT[dtype], std=0.1) + 1, _rnd(g, n, dtype=DT[dtype], std=0.1), _rnd(g, m, n, dtype=DT[dtype])
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = ops.layer_norm(*leaves, eps=1e-12)
    got = dict(zip(("y", "dx", "dw", "db"), (y, *_grads(y, leaves, dy))))
    for name, (value, bound) in train_ref.layer_norm(x, w, b, dy, 1e-12).items():
        train_ref.check(name, got[name], value, bound)
    again = ops.layer_norm(*leaves, eps=1e-12)
    assert torch.equal(again, y) and all(torch.equal(a, got[k]) for a, k in zip(_grads(again, leaves, dy), ("dx", "dw", "db")))
    if n > 8:                                                           # rows of a wider tensor
        wide = torch.cat([x, x], 1)[:, n:]
        assert torch.equal(ops.layer_norm(wide, w, b, 1e-12).float(), y.float()) or n % 8
    for i in range(3):                                                  # one gradient asked for at a time
        part = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        assert torch.equal(_grads(ops.layer_norm(*part, eps=1e-12), (part[i],), dy)[0], got[("dx", "dw", "db")[i]])


def test_layer_norm_no_rows(ops):
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w, w.detach().requires_grad_())
    gx, gw = _grads(y, (x, w), torch.empty_like(y))
    assert gx.shape == (0, 16) and not gw.any()


# ---- a run of them, as they are used ---------------------------------------------------------------------------------------
def _layer(ops, x, p, off, longest, keeps, checkpoint=None):
    """one encoder layer on packed tokens: attention, output projection with dropout and residual, norm, feed-forward, norm"""
    t = x.shape[0]
    q, k, v = (a.unflatten(1, (4, 64)) for a in ops.linear(x, p["qkv"], p["qkv_b"], checkpoint=checkpoint).split(256, dim=1))
    ctx = ops.attention(q, k, v, off, max_q=longest, max_k=longest, keep=keeps[0], keep_scale=1 / 0.9).reshape(t, 256)
    a = ops.layer_norm(ops.linear(ctx, p["o"], p["o_b"], keep=keeps[1], keep_scale=1 / 0.9, residual=x, checkpoint=checkpoint), p["n1"], p["n1_b"])
    h = ops.linear(a, p["f1"], p["f1_b"], activation="gelu", checkpoint=checkpoint)
    return ops.layer_norm(ops.linear(h, p["f2"], p["f2_b"], keep=keeps[2], keep_scale=1 / 0.9, residual=a, checkpoint=checkpoint), p["n2"], p["n2_b"])


def _layer_inputs(dtype, lens=(37, 5, 90)):
    g = _gen(41)
    rnd = lambda *s, std=1.0: _rnd(g, *s, dtype=dtype, std=std)  # noqa: E731
    t = sum(lens)
    p = {"qkv": rnd(768, 256, std=0.06), "qkv_b": rnd(768, std=0.1), "o": rnd(256, 256, std=0.06), "o_b": rnd(256, std=0.1), "f1": rnd(512, 256, std=0.06),
         "f1_b": rnd(512, std=0.1), "f2": rnd(256, 512, std=0.04), "f2_b": rnd(256, std=0.1)}
    for n in ("n1", "n2"):
        p[n], p[n + "_b"] = 1 + rnd(256, std=0.1), rnd(256, std=0.1)
    keeps = [torch.rand(s, generator=g, device="cuda") >= 0.1 for s in ((t, 4, max(lens)), (t, 256), (t, 256))]
    return rnd(t, 256), p, _offsets(lens)[1], max(lens), keeps, rnd(t, 256, std=0.1)


class _Wide:
    """the operators in float64 torch, on the CPU, for a whole layer"""

    @staticmethod
    def linear(x, w, b, activation=None, keep=None, keep_scale=1.0, residual=None, checkpoint=None):
        y = x @ w.T + b
        y = y * torch.special.ndtr(y) if activation else y
        y = y if keep is None else y * keep.cpu() * keep_scale
        return y if residual is None else y + residual

    @staticmethod
    def layer_norm(x, w, b, eps=1e-12):
        return w * (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) + b

    @staticmethod
    def attention(q, k, v, off, max_q, max_k, keep, keep_scale):
        o = off.tolist()
        outs = []
        for a, b in zip(o, o[1:]):
            s = torch.softmax(torch.matmul(q[a:b].transpose(0, 1), k[a:b].permute(1, 2, 0)) / 8, -1) * keep[a:b, :, : b - a].cpu().transpose(0, 1) * keep_scale
            outs.append(torch.matmul(s, v[a:b].transpose(0, 1)).transpose(0, 1))
        return torch.cat(outs)


@pytest.mark.parametrize("dtype,checkpoint,bound", [("fp32", None, 2e-5), ("fp16", None, 4e-3), ("bf16", None, 3e-2), ("bf16", "e4m3", 8e-2)])
def test_a_layer_forward_and_backward(dtype, checkpoint, bound, ops):
    """Relative 2-norms. A layer is a dozen roundings deep; each is at most u = eps / 2 (fp32 2^-24, fp16 2^-11, bf16 2^-8) of its value and they add at
    worst linearly: 8 u for fp16 and bf16 (2^-8 and 2^-5 = 3e-2); fp32: the sums of up to 768 terms dominate, 2e-5. With 8-bit checkpoints a weight's
    gradient and the activation's slope see values off by up to 2^-4, at random: a root mean square of 2^-4 / sqrt 3 / ... < 5e-2 on top"""
    x, p, off, longest, keeps, dy = _layer_inputs(DT[dtype])
    leaves = {"x": x, **p}
    own = {n: t.detach().requires_grad_() for n, t in leaves.items()}
    y = _layer(ops, own["x"], own, off, longest, keeps, checkpoint)
    got = dict(zip(own, _grads(y, list(own.values()), dy)))
    wide = {n: t.double().cpu().requires_grad_() for n, t in leaves.items()}
    yw = _layer(_Wide, wide["x"], wide, off, longest, keeps)
    want = dict(zip(wide, _grads(yw, list(wide.values()), dy.double().cpu())))
    err = {"y": float((y.double().cpu() - yw).norm() / yw.norm())}
    for n in want:
        err[n] = float((got[n].double().cpu() - want[n]).norm() / want[n].norm())
    assert max(err.values()) <= bound, err


def test_a_layer_on_another_stream_and_in_a_graph(ops):
    x, p, off, longest, keeps, dy = _layer_inputs(torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (x, *p.values())]

    def step():
        own = dict(zip(p, leaves[1:]))
        y = _layer(ops, leaves[0], own, off, longest, keeps, "e4m3")
        return [y.detach(), *_grads(y, leaves, dy)]

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(step(), want):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                                  # two graphs of the same inputs, each with buffers of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    before = x.clone()
    for i in range(4):
        with torch.no_grad():
            leaves[0].copy_(before * (i + 1) * 0.5)
        want = step()
        for g, _ in graphs:
            g.replay()
        eager = step()                                                  # the program's own work between replays
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want)), i
        assert all(torch.equal(a, b) for a, b in zip(eager, want))


def test_attention_off_a_16_byte_border_and_lone_rows(ops):
    g = torch.Generator(device="cuda").manual_seed(3)
    flat = torch.randn(1 + 40 * 2 * 16, generator=g, device="cuda").bfloat16()
    off = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    shifted, plain = flat[1:].view(40, 2, 16), flat[1:].clone().view(40, 2, 16)
    assert shifted.data_ptr() % 16 and shifted.is_contiguous()
    assert torch.equal(ops.attention(shifted, shifted, shifted, off), ops.attention(plain, plain, plain, off))
    # one row, one head: their strides are any number
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for q, kv in ((flat.as_strided((1, 1, 16), (3, 5, 1)), plain[:, :1]), (flat.as_strided((1, 2, 16), (3, 16, 1)), plain)):
        assert q.is_contiguous()
        assert torch.equal(ops.attention(q, kv, kv, one, off), ops.attention(q.clone(memory_format=torch.contiguous_format), kv, kv, one, off))
    leaf = shifted.detach().requires_grad_()
    (got,) = torch.autograd.grad(ops.attention(leaf, plain, plain, off), leaf, plain)
    leaf = plain.detach().requires_grad_()
    (want,) = torch.autograd.grad(ops.attention(leaf, plain, plain, off), leaf, plain)
    assert torch.equal(got, want)


@pytest.mark.parametrize("n,std,vstd,dstd", [(4000, 1.2, 1.2, 3e-3), (700, 1.2, 1.2, 1e-3), (2, 0.02, 4.0, 1e4), (8, 0.02, 20.0, 1e4), (300, 0.02, 1.2, 5e3)])
def test_attention_gradients_in_fp16_beyond_its_range_of_probabilities(n, std, vstd, dstd, ops):
    """dS of small gradients over many keys lie below 2^-14, those of large gradients over few keys above 2^16"""
    g = torch.Generator().manual_seed(n)
    q, k = (torch.randn(n, 1, 64, generator=g).mul(std).half().cuda().requires_grad_() for _ in range(2))
    v, dy = torch.randn(n, 1, 64, generator=g).mul(vstd).half().cuda().requires_grad_(), torch.randn(n, 1, 64, generator=g).mul(dstd).half().cuda()
    off = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    got = torch.autograd.grad(ops.attention(q, k, v, off), (q, k, v), dy)
    q64, k64, v64, d64 = (t.detach().double()[:, 0] for t in (q, k, v, dy))
    p = torch.softmax(q64 @ k64.t() / 8, 1)
    dp = d64 @ v64.t()
    ds = p * (dp - (p * dp).sum(1, keepdim=True))
    for name, a, want in zip("qkv", got, (ds @ k64 / 8, ds.t() @ q64 / 8, p.t() @ d64)):
        # norm-wise three roundings of 2^-11: P or dS, the forward's output in delta, the result (2^-25 absolute where it is below 2^-14); fp32 sums add less than half of one
        off_by, bound = float((a.double()[:, 0] - want).norm()), 3.5 * 2.0**-11 * float(want.norm()) + 2.0**-25 * want.numel() ** 0.5
        assert off_by <= bound, (name, off_by / float(want.norm()))


def test_layer_norm_of_more_rows_than_a_launch_has(ops):
    m = 4 * (1 << 22) + 37
    x = torch.randn(m, 8, device="cuda", dtype=torch.float16)
    w, b = torch.rand(8, device="cuda").half() + 0.5, torch.rand(8, device="cuda").half()
    y = ops.layer_norm(x, w, b)
    for part in (slice(0, 64), slice(m - 64, m)):
        v = x[part].double()
        want = w.double() * (v - v.mean(1, keepdim=True)) / (v.pow(2).mean(1, keepdim=True) + 1e-12).sqrt() + b.double()
        # one rounding of the result (2^-11), and fp32 sums of 8 values with a root: some 20 roundings of 2^-24 of terms below 1.5 * 3 + 1
        assert bool(((y[part].double() - want).abs() <= want.abs() * 2.0**-11 + 20 * 2.0**-24 * 5.5 + 2.0**-25).all())


def test_rows_longer_than_an_int_are_refused(ops):
    from atlas_amd._lib import AtlasHipError

    x, one = torch.zeros(1, device="cuda").expand(1 << 31), torch.zeros(1, device="cuda")
    for call in (lambda: ops.compress(x), lambda: ops.layer_norm(x, x, x), lambda: ops.linear(x, x[None]), lambda: ops.linear(x[:, None], one[None])):
        with pytest.raises(AtlasHipError):
            call()


def test_attention_of_many_short_sequences_whose_longest_is_not_given(ops):
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 30, (3000,), generator=g)
    lens[7] = 700
    off = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).int().cuda()
    x = torch.randn(int(off[-1]), 16, 8, generator=g).half().cuda()
    q, dy = x.detach().requires_grad_(), torch.randn(x.shape, generator=g).half().cuda()
    outs = []
    for longest in ({}, {"max_q": 700, "max_k": 700}, {"max_q": 0, "max_k": 1}):
        y = ops.attention(q, x, x, off, **longest)
        outs.append([y.detach(), *torch.autograd.grad(y, q, dy)])
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_decode_takes_only_what_compress_gives(ops):
    from atlas_amd._lib import AtlasHipError

    x = torch.randn(6, 40, device="cuda")
    c = ops.compress(x)
    assert torch.equal(ops.Compressed(c.codes, c.scales, x.shape, x.dtype).decode(), c.decode())
    for codes, scales, shape in [(c.codes[:5], c.scales, x.shape), (c.codes, c.scales[:5], x.shape), (c.codes, c.scales, (7, 40)), (c.codes, c.scales, (6, 65)),
                                 (c.codes, c.scales, ()), (c.codes, c.scales, (-6, -40)), (c.codes.cpu(), c.scales, x.shape), (c.codes, c.scales.cpu(), x.shape),
                                 (c.codes.int(), c.scales, x.shape), (c.codes.t().contiguous().t(), c.scales, x.shape), (c.codes.flatten(), c.scales, x.shape)]:
        with pytest.raises(AtlasHipError):
            ops.Compressed(codes, scales, shape, x.dtype).decode()
            print("not refused:", codes.shape, scales.shape, shape)


def test_a_captured_call_refuses_leaves_of_a_live_eager_graph(ops):
    """nothing but the forward call is inside the capture: it has to be refused there, and goes through once the eager graph is gone"""
    from atlas_amd._lib import AtlasHipError

    x, w, q = torch.randn(5, 64, device="cuda"), torch.randn(64, 64, device="cuda").requires_grad_(), torch.randn(5, 1, 64, device="cuda").requires_grad_()
    b, off = torch.randn(64, device="cuda").requires_grad_(), torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    calls = [lambda: ops.linear(x, w), lambda: ops.layer_norm(x, b, b), lambda: ops.attention(q, x[:, None], x[:, None], off)]
    eager = [call() for call in calls]
    torch.cuda.synchronize()
    for call in calls:
        with pytest.raises(AtlasHipError, match="default stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = calls[0]()
        again = ops.linear(x, w, residual=y)                            # the same leaf twice in one capture
        (dw,) = torch.autograd.grad(again, w, torch.ones_like(again))
    graph.replay()
    eager = ops.linear(x, w, residual=ops.linear(x, w))
    assert torch.equal(eager, again) and torch.equal(torch.autograd.grad(eager, w, torch.ones_like(eager))[0], dw)


def test_refusals_on_the_gpu(ops):
    from atlas_amd._lib import AtlasHipError

    x = torch.zeros(10, 2, 64, device="cuda", dtype=torch.bfloat16)
    off = torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    bad = [
        lambda: ops.attention(x, x.half(), x, off), lambda: ops.attention(x, x[:, :, :32], x, off), lambda: ops.attention(x[:, :, :60], x[:, :, :60], x[:, :, :60], off),
        lambda: ops.attention(x, x[:5], x[:5], off), lambda: ops.attention(x, x, x, off, off[:1]), lambda: ops.attention(x, x, x, off.float()),
        lambda: ops.attention(x, x, x, off.cpu()), lambda: ops.attention(x, x, x, off, scale=0.0), lambda: ops.attention(x, x, x, off, scale=float("nan")),
        lambda: ops.attention(x, x, x, off, key_mask=torch.ones(9, dtype=torch.bool, device="cuda")),
        lambda: ops.attention(x, x, x, off, key_mask=torch.ones(10, device="cuda")),
        lambda: ops.attention(x, x, x, off, keep=torch.ones(10, 3, 10, dtype=torch.bool, device="cuda")),
        lambda: ops.attention(x.repeat(1, 2, 1)[:, :3], x, x, off), lambda: ops.attention(x.long(), x.long(), x.long(), off),
        lambda: ops.attention(torch.zeros(10, 2, 136, device="cuda"), torch.zeros(10, 2, 136, device="cuda"), torch.zeros(10, 2, 136, device="cuda"), off),
    ]
    a, w = torch.zeros(4, 16, device="cuda"), torch.zeros(8, 16, device="cuda")
    bad += [
        lambda: ops.linear(a, w.half()), lambda: ops.linear(a, w[:, :8]), lambda: ops.linear(a, w, torch.zeros(9, device="cuda")), lambda: ops.linear(a, w[:, :0]),
        lambda: ops.linear(a, w, activation="relu"), lambda: ops.linear(a, w, checkpoint="int8"), lambda: ops.linear(a, w, residual=a),
        lambda: ops.linear(a, w, keep=torch.ones(4, 16, dtype=torch.bool, device="cuda")), lambda: ops.linear(a, w, keep=torch.ones(4, 8, device="cuda")),
        lambda: ops.linear(a.double(), w.double()), lambda: ops.linear(a, w.cpu()), lambda: ops.layer_norm(a, w[0], w[0].half()),
        lambda: ops.layer_norm(a, w[0], w[0][:8]), lambda: ops.layer_norm(a, w[0], w[0], eps=-1.0), lambda: ops.layer_norm(a[:, :0], w[0, :0], w[0, :0]),
        lambda: ops.compress(a.long()), lambda: ops.compress(torch.tensor(1.0, device="cuda")), lambda: ops.compress(a).decode(torch.int8),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AtlasHipError):
            call()
            print("not refused:", i)
    y = ops.linear(a.requires_grad_(), w)
    (gx,) = torch.autograd.grad(y.sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):                                   # once differentiable
        torch.autograd.grad(gx.sum(), a)
