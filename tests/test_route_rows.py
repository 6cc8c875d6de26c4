"""The weighted return and the sort's gradient where few or no rows belong to
local experts, and maps that leave the rows.

Sums of up to topk fp32 products in a fixed order are exact here: rows and
weights are small integers."""

import ctypes

import pytest
import torch

from int8blockwisegemm_b200 import _lib, permute

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def no_device_error(request):
    if "gpu" not in request.keywords:
        yield
        return
    _lib.device_error(0, clear=True)
    yield
    assert _lib.device_error(0, clear=True) == 0


def integers(*shape, dt=torch.float32, seed=0, most=8):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g).to(dt).to(DEV)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,K,topk", [(1, 8, 1), (5, 64, 3), (40, 2048, 8), (3, 160, 9)])
def test_a_rank_without_rows(T, K, topk, dt):
    """No row belongs to a local expert, and none is there: zeros."""
    out = torch.full((T, K), 7.0, dtype=dt, device=DEV)
    inv = torch.arange(T * topk, dtype=torch.int32, device=DEV)
    eft = torch.zeros(4, dtype=torch.int64, device=DEV)
    empty = torch.empty(0, K, dtype=dt, device=DEV)
    assert empty.data_ptr() == 0
    permute.moe_unpermute(out, empty, torch.ones(T, topk, device=DEV), inv, eft)
    assert not out.any()
    out.fill_(7.0)
    permute.moe_unpermute(out, empty, torch.ones(T, topk, device=DEV), torch.full_like(inv, -1))
    assert not out.any()
    # the sort's gradient with rows of other ranks' experts alone, which are not read
    foreign = torch.full((T * topk, K), float("nan"), dtype=dt, device=DEV)
    assert not permute.moe_permute_backward(foreign, inv, eft, T, topk).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 60])
def test_rows_trimmed_to_the_local_ones(n, dt):
    """A tensor of the local experts' rows alone, n of the 20 * 3."""
    T, topk, K = 20, 3, 64
    inv = torch.randperm(T * topk, generator=torch.Generator().manual_seed(n)).to(torch.int32).to(DEV)
    x, w = integers(n, K, dt=dt), integers(T, topk, seed=1)
    eft = torch.tensor([0, n // 2, n], device=DEV)
    out = torch.empty(T, K, dtype=dt, device=DEV)
    permute.moe_unpermute(out, x, w, inv, eft)
    all_rows = torch.zeros(T * topk, K, device=DEV)
    all_rows[:n] = x.float()
    want = (all_rows[inv.long()].view(T, topk, K) * w[..., None]).sum(1)
    assert torch.equal(out, want.to(dt))
