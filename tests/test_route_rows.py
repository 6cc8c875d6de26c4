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


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_a_map_into_padded_rows(dt):
    """A caller's own layout with gaps between the experts' rows: more rows
    than slots, and every index that the tensor has counts."""
    T, topk, K, rows = 30, 2, 64, 150
    g = torch.Generator().manual_seed(0)
    inv = torch.randperm(rows, generator=g)[:T * topk].to(torch.int32).to(DEV)
    assert int(inv.max()) >= T * topk
    x, w = integers(rows, K, dt=dt), integers(T, topk, seed=1)
    want = (x[inv.long()].float().view(T, topk, K) * w[..., None]).sum(1).to(dt)
    out = torch.empty(T, K, dtype=dt, device=DEV)
    for eft in (None, torch.tensor([0, 70, rows], device=DEV)):
        permute.moe_unpermute(out.fill_(7.0), x, w, inv, eft)
        assert torch.equal(out, want)
    lib, p = _lib.LIB, ctypes.c_void_p
    out.fill_(7.0)
    rc = lib.i8moe_moe_unpermute(p(x.data_ptr()), DTYPES.index(dt), p(w.data_ptr()), p(inv.data_ptr()), None, 0, T,
                                 topk, K, p(out.data_ptr()), p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0 and torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("train", [False, True])
def test_indices_outside_of_the_rows_are_reported(train):
    T, topk, K = 4, 2, 64
    x, w = integers(T * topk, K), integers(T, topk, seed=1)
    inv = i32([0, 1, 2, 8, 4, 5, 6, 7])  # 8 is no row

    def run(inv, eft):
        if train:
            return permute.moe_unpermute_train(x, w, inv, eft)
        out = torch.empty(T, K, device=DEV)
        permute.moe_unpermute(out, x, w, inv, eft)
        return out

    for eft in (None, torch.tensor([0, 9], device=DEV)):
        out = run(inv, eft)
        assert torch.equal(out[1], w[1, 0] * x[2]) and torch.equal(out[0], w[0, 0] * x[0] + w[0, 1] * x[1])
        assert _lib.device_error(0, clear=True) == 1 << 5
    run(inv, torch.tensor([0, 8], device=DEV))  # skipped by the offsets, as rows of other ranks are
    run(i32([0, 1, 2, -1, 4, 5, 6, 7]), None)  # a slot without a row
    assert _lib.device_error(0) == 0


def test_c_argument_errors_before_any_cuda_call():
    one = ctypes.c_void_p(256)  # never read

    def call(rows=4, dtype=0, topk=2, k=64, T=2):
        return _lib.LIB.i8moe_moe_unpermute_rows(one, rows, dtype, one, one, None, 0, T, topk, k, one, None)

    for kw, message in [(dict(rows=-1), "n_rows"), (dict(dtype=3), "dtype"), (dict(topk=0), "topk"),
                        (dict(k=63), "16 bytes"), (dict(T=-1), "n_token")]:
        assert call(**kw) == -1 and message in _lib.last_error(), kw
    assert call(T=0) == 0
