"""The compiled torch binding of the norm, the sort and the 4-bit products: what
it refuses because it goes past torch's dispatcher."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

DEV = "cuda:0"


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused():
    """They would be left out without a word."""
    from int8blockwisegemm_b200 import int4, norm, permute
    T, K, topk = 4, 64, 2
    x, w = torch.randn(T, K, device=DEV), torch.randn(K, device=DEV)
    y, tw = torch.randn(T * topk, K, device=DEV), torch.rand(T, topk, device=DEV)
    ids = torch.zeros(T, topk, dtype=torch.int32, device=DEV)
    inv = torch.arange(T * topk, dtype=torch.int32, device=DEV)
    eft = torch.tensor([0, T * topk], device=DEV)
    one = torch.ones(T, device=DEV)
    packed, scale = int4.quantize_weights_int4(torch.randn(1, 32, K, device=DEV), 32, torch.bfloat16)
    eo = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    xb = x.bfloat16()
    calls = [  # the tensors of a call, each of them with a tangent in turn
        (lambda a, b: norm.rms_norm(a, b), (x, w)), (lambda a, b: norm.rms_norm(x, w, 1e-6, a), (x, w)),
        (lambda a, b: norm.rms_norm_quant_int8(a, b), (x, w)),
        (lambda a, b: norm.rms_norm_backward(a, x, b, one), (x, w)),
        (lambda a, b: norm.rms_norm_backward(x, a, b, one, None, x), (x, w)),
        (lambda a, b: permute.moe_permute_train(a, ids, 1), (x, w)),
        (lambda a, b: permute.moe_unpermute_train(a, b, inv, eft), (y, tw)),
        (lambda a, b: permute.moe_permute_backward(a, inv, eft, T, topk), (y, tw)),
        (lambda a, b: permute.moe_unpermute_backward(x, a, b, inv, eft), (y, tw)),
        (lambda a, b: int4.int4_grouped_mv(a, packed, b, eo, 32), (xb, scale))]
    for call, args in calls:
        want = call(*args)
        with fwd.dual_level():
            call(*args)
            refused = 0
            for i in range(2):
                dual = [fwd.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)]
                try:
                    call(*dual)
                except RuntimeError as e:
                    assert "forward-mode" in str(e)
                    refused += 1
            assert refused >= 1
        again = call(*args)
        want, again = (t if isinstance(t, tuple) else (t,) for t in (want, again))
        assert all(a is b or torch.equal(a, b) for a, b in zip(want, again))
