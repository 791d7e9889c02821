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
