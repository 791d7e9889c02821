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
