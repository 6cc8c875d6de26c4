"""The RMS norm where its sums leave fp32."""

import pytest
import torch

from int8blockwisegemm_b200 import norm

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [1, 64, 67, 2048, 12289, 40961])
def test_a_norm_that_is_not_finite_says_so(K, dt):
    """Squares that leave fp32 under finite values: the int8 row's scale is
    NaN, as with an infinity, and no scale of a row of zeros."""
    x = torch.ones(5, K, dtype=dt, device=DEV)
    w = torch.ones(K, dtype=dt, device=DEV)
    want = norm.rms_norm_quant_int8(x, w)
    x[1], x[3, K // 2] = 1e25, 3e20
    for residual in (None, torch.zeros_like(x)):
        q, s, y, _ = norm.rms_norm_quant_int8(x, w, 1e-6, residual, return_norm=True)
        assert s.isnan().tolist() == [False, True, False, True, False]
        assert not q[1].any() and not q[3].any()
        assert torch.equal(q[::2], want[0][::2]) and torch.equal(s[::2], want[1][::2])
