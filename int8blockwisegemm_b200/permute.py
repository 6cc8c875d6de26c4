"""MoE permute / unpermute wrappers with the reference's signatures and
allocations (int8_hybrid_moe/permute.py:9-134): permuted_idx is pre-filled
with the sentinel n_token*topk, token_expert_indices is arange."""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import BF16, FP16, FP32, LIB, launch

_DT = {torch.bfloat16: BF16, torch.float16: FP16, torch.float32: FP32}


def _alloc(n_token: int, topk: int, n_local_expert: int, device):
    rows = n_token * topk
    tei = torch.arange(rows, dtype=torch.int32, device=device).reshape(n_token, topk)
    eft = torch.empty(n_local_expert + 1, dtype=torch.int64, device=device)
    pidx = torch.full((rows,), rows, dtype=torch.int32, device=device)
    inv = torch.empty((n_token, topk), dtype=torch.int32, device=device)
    return tei, eft, pidx, inv


def moe_permute(hidden_states, a1q_scale, topk_ids, n_expert: int, n_local_expert: int = -1,
                expert_map=None, permuted_hidden_states=None):
    """Expand and permute activation rows into expert-contiguous order."""
    n_token, n_hidden = hidden_states.size()
    topk = topk_ids.size(1)
    if n_local_expert == -1:
        n_local_expert = n_expert
    if permuted_hidden_states is None:
        permuted_hidden_states = torch.empty((n_token * topk, n_hidden),
                                             dtype=hidden_states.dtype,
                                             device=hidden_states.device)
    tei, eft, pidx, inv = _alloc(n_token, topk, n_local_expert, hidden_states.device)
    ops.moe_permute(hidden_states, topk_ids.to(torch.int32), tei, expert_map, n_expert,
                    n_local_expert, topk, permuted_hidden_states, eft, inv, pidx)
    if a1q_scale is not None and a1q_scale.dim() > 1:
        a1q_scale = a1q_scale[pidx.clamp(max=n_token * topk - 1) // topk]
    return permuted_hidden_states, a1q_scale, eft, inv.flatten(), pidx


def moe_permute_metadata(hidden_states, topk_ids, n_expert: int, n_local_expert: int = -1,
                         expert_map=None):
    """Routing metadata only (no row copy)."""
    n_token = hidden_states.size(0)
    topk = topk_ids.size(1)
    if n_local_expert == -1:
        n_local_expert = n_expert
    tei, eft, pidx, inv = _alloc(n_token, topk, n_local_expert, hidden_states.device)
    ops.moe_permute_metadata(topk_ids.to(torch.int32), tei, expert_map, n_expert,
                             n_local_expert, topk, eft, inv, pidx)
    return eft, inv.flatten(), pidx


def moe_route_for_gemm(topk_ids, n_token: int, n_expert: int, n_local_expert: int, expert_map,
                       n_out1: int, k1: int, n_out2: int, k2: int, tile_m: int, inv_out=None):
    """Extension: routing metadata plus the int32 expert offsets, both GEMMs'
    problem sizes and the quant scale offsets, from one set of kernels.
    ``inv_out`` (int32, n_token * topk elements, contiguous) receives the
    inverse map instead of a new tensor.

    Returns (expert_first_token_offset, inv_permuted_idx (flat), permuted_idx,
             expert_offsets_i32 [E+1], problem_sizes13, problem_sizes2,
             scale_offsets_i32 [E+1])."""
    topk = topk_ids.size(1)
    dev = topk_ids.device
    # the routing kernels write every permuted_idx slot (sentinel included)
    # and take token_expert_indices as arange when it is omitted: no
    # pre-fill launches on this path
    rows = n_token * topk
    eft = torch.empty(n_local_expert + 1, dtype=torch.int64, device=dev)
    pidx = torch.empty(rows, dtype=torch.int32, device=dev)
    if inv_out is None:
        inv = torch.empty((n_token, topk), dtype=torch.int32, device=dev)
    else:
        assert (inv_out.dtype == torch.int32 and inv_out.is_contiguous()
                and inv_out.numel() == rows and inv_out.device == dev)
        inv = inv_out.view(n_token, topk)
    eo = torch.empty(n_local_expert + 1, dtype=torch.int32, device=dev)
    ps1 = torch.empty((n_local_expert, 3), dtype=torch.int32, device=dev)
    ps2 = torch.empty((n_local_expert, 3), dtype=torch.int32, device=dev)
    so = torch.empty(n_local_expert + 1, dtype=torch.int32, device=dev)
    torch.ops.int8_hybrid_moe.moe_route_for_gemm(
        topk_ids.to(torch.int32), None, expert_map, n_expert, n_local_expert, topk, eft, inv,
        pidx, eo, ps1, ps2, so, n_out1, k1, n_out2, k2, tile_m)
    return eft, inv.flatten(), pidx, eo, ps1, ps2, so


def router_topk(logits, topk: int, bias=None):
    """Extension (the router upstream of the runner): top-k experts of each
    token by logits + bias, weights = softmax of their unbiased logits.
    Returns (topk_weights fp32 [T, k], topk_ids int32 [T, k])."""
    from ._lib import call
    assert logits.dtype == torch.float32 and logits.is_contiguous() and logits.is_cuda
    T, E = logits.shape
    ids = torch.empty(T, topk, dtype=torch.int32, device=logits.device)
    w = torch.empty(T, topk, dtype=torch.float32, device=logits.device)
    if bias is not None:
        assert bias.dtype == torch.float32 and bias.numel() == E and bias.is_contiguous()
    with torch.cuda.device(logits.device):
        call("i8moe_router_topk", logits.data_ptr(),
             bias.data_ptr() if bias is not None else None, T, E, topk, ids.data_ptr(),
             w.data_ptr(), torch.cuda.current_stream(logits.device).cuda_stream)
    return w, ids


def router_route_for_gemm(logits, topk: int, n_local_expert: int, expert_map, n_out1: int,
                          k1: int, n_out2: int, k2: int, tile_m: int, bias=None):
    """Extension: ``router_topk`` and ``moe_route_for_gemm`` in one pass (the
    router kernel also builds the routing histogram).  Returns
    (topk_weights, topk_ids, expert_first_token_offset, inv_permuted_idx
    (flat), permuted_idx, expert_offsets_i32, problem_sizes13,
    problem_sizes2, scale_offsets_i32)."""
    from ._lib import call
    assert logits.dtype == torch.float32 and logits.is_contiguous() and logits.is_cuda
    T, E = logits.shape
    dev = logits.device
    ids = torch.empty(T, topk, dtype=torch.int32, device=dev)
    w = torch.empty(T, topk, dtype=torch.float32, device=dev)
    eft = torch.empty(n_local_expert + 1, dtype=torch.int64, device=dev)
    pidx = torch.empty(T * topk, dtype=torch.int32, device=dev)
    inv = torch.empty((T, topk), dtype=torch.int32, device=dev)
    eo = torch.empty(n_local_expert + 1, dtype=torch.int32, device=dev)
    ps1 = torch.empty((n_local_expert, 3), dtype=torch.int32, device=dev)
    ps2 = torch.empty((n_local_expert, 3), dtype=torch.int32, device=dev)
    so = torch.empty(n_local_expert + 1, dtype=torch.int32, device=dev)
    from ._lib import LIB
    ws = torch.empty(max(1, LIB.i8moe_route_workspace_size(T * topk, E)), dtype=torch.uint8,
                     device=dev)
    emap = expert_map.to(torch.int32).contiguous() if expert_map is not None else None
    with torch.cuda.device(dev):
        call("i8moe_router_route_for_gemm", logits.data_ptr(),
             bias.data_ptr() if bias is not None else None, T, E, topk, ids.data_ptr(),
             w.data_ptr(), None, emap.data_ptr() if emap is not None else None,
             n_local_expert, eft.data_ptr(), inv.data_ptr(), pidx.data_ptr(), eo.data_ptr(),
             ps1.data_ptr(), ps2.data_ptr(), so.data_ptr(), n_out1, k1, n_out2, k2, tile_m,
             ws.data_ptr(), ws.numel(), torch.cuda.current_stream(dev).cuda_stream)
    return w, ids, eft, inv.flatten(), pidx, eo, ps1, ps2, so


def moe_unpermute(out, permuted_hidden_states, topk_weights, inv_permuted_idx,
                  expert_first_token_offset=None) -> None:
    """Top-k weighted reduction back to token order."""
    topk = topk_weights.size(1)
    ops.moe_unpermute(permuted_hidden_states, topk_weights, inv_permuted_idx,
                      expert_first_token_offset, topk, out)


# ---------------------------------------------------------------------------
# Differentiable sort and return (extension).  Both passes can be captured into
# a CUDA graph; as for every autograd graph, drop eager graphs that hold the
# same leaves before capturing a backward pass.
# ---------------------------------------------------------------------------

def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _check_rows(what: str, name: str, t) -> None:
    _check(t.is_cuda and t.dim() == 2, f"{what}: {name} must be a CUDA tensor [rows, hidden]")
    _check(t.dtype in _DT, f"{what}: {name} must be bfloat16, float16 or float32")
    _check(t.size(1) * t.element_size() % 16 == 0,
           f"{what}: hidden row must be a multiple of 16 bytes")


def _check_maps(what: str, inv, eft, rows: int, device) -> None:
    _check(inv.dtype == torch.int32 and inv.is_contiguous() and inv.device == device
           and inv.numel() == rows,
           f"{what}: inv_permuted_idx must be contiguous int32 with n_token * topk elements")
    if eft is not None:
        _check(eft.dtype == torch.int64 and eft.is_contiguous() and eft.device == device
               and eft.dim() == 1 and eft.numel() >= 1,
               f"{what}: expert_first_token_offset must be contiguous int64 [n_local_expert + 1]")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and 16-byte aligned, copied when it is not."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _eft_args(eft):
    return (None, 0) if eft is None else (eft.data_ptr(), eft.numel() - 1)


def moe_permute_backward(permuted_grad, inv_permuted_idx, expert_first_token_offset, n_token: int,
                         topk: int):
    """Gradient of the row copy: [n_token, hidden], the sum of each token's
    rows of ``permuted_grad`` that belong to local experts."""
    what = "moe_permute_backward"
    _check_rows(what, "permuted_grad", permuted_grad)
    _check(n_token >= 0 and topk >= 1 and permuted_grad.size(0) == n_token * topk,
           f"{what}: permuted_grad must have n_token * topk rows")
    dev = permuted_grad.device
    _check_maps(what, inv_permuted_idx, expert_first_token_offset, n_token * topk, dev)
    g = _aligned(permuted_grad)
    out = torch.empty((n_token, g.size(1)), dtype=g.dtype, device=dev)
    launch("i8moe_moe_permute_backward", dev, g.data_ptr(), _DT[g.dtype],
           inv_permuted_idx.data_ptr(), *_eft_args(expert_first_token_offset), n_token, topk,
           g.size(1), out.data_ptr())
    return out


def moe_unpermute_backward(out_grad, permuted_hidden_states, topk_weights, inv_permuted_idx,
                           expert_first_token_offset=None):
    """Gradients of ``moe_unpermute``: (of permuted_hidden_states, of
    topk_weights in fp32); zero for rows of no local expert."""
    what = "moe_unpermute_backward"
    _check_rows(what, "permuted_hidden_states", permuted_hidden_states)
    dev = permuted_hidden_states.device
    _check(topk_weights.dim() == 2 and topk_weights.dtype == torch.float32
           and topk_weights.device == dev, f"{what}: topk_weights must be float32 [n_token, topk]")
    n_token, topk = topk_weights.shape
    _check(topk >= 1 and permuted_hidden_states.size(0) == n_token * topk,
           f"{what}: permuted_hidden_states must have n_token * topk rows")
    _check(out_grad.shape == (n_token, permuted_hidden_states.size(1))
           and out_grad.dtype == permuted_hidden_states.dtype and out_grad.device == dev,
           f"{what}: out_grad must be [n_token, hidden] of permuted_hidden_states' dtype")
    _check_maps(what, inv_permuted_idx, expert_first_token_offset, n_token * topk, dev)
    g, y, w = _aligned(out_grad), _aligned(permuted_hidden_states), topk_weights.contiguous()
    dy = torch.empty_like(y)
    dw = torch.empty_like(w)
    launch("i8moe_moe_unpermute_backward", dev, g.data_ptr(), y.data_ptr(), _DT[y.dtype],
           w.data_ptr(), inv_permuted_idx.data_ptr(), *_eft_args(expert_first_token_offset),
           n_token, topk, y.size(1), dy.data_ptr(), dw.data_ptr())
    return dy, dw


def _sort_rows(x, ids, emap, n_expert, n_local_expert):
    T, topk = ids.shape
    dev, rows = x.device, T * topk
    eft = torch.empty(n_local_expert + 1, dtype=torch.int64, device=dev)
    inv = torch.empty(rows, dtype=torch.int32, device=dev)
    pidx = torch.empty(rows, dtype=torch.int32, device=dev)
    out = torch.empty((rows, x.size(1)), dtype=x.dtype, device=dev)
    nbytes = LIB.i8moe_route_workspace_size(rows, n_expert)
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
    launch("i8moe_moe_permute_metadata", dev, ids.data_ptr(), None,
           emap.data_ptr() if emap is not None else None, T, topk, n_expert, n_local_expert,
           eft.data_ptr(), inv.data_ptr(), pidx.data_ptr(), ws.data_ptr(), nbytes)
    launch("i8moe_moe_scatter_rows", dev, x.data_ptr(), _DT[x.dtype], inv.data_ptr(),
           eft.data_ptr(), n_local_expert, T, topk, x.size(1), out.data_ptr())
    return out, eft, inv, pidx


class _SortRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, emap, n_expert, n_local_expert):
        out, eft, inv, pidx = _sort_rows(x, ids, emap, n_expert, n_local_expert)
        ctx.save_for_backward(eft, inv)
        ctx.tokens = tuple(ids.shape)
        ctx.mark_non_differentiable(eft, inv, pidx)
        ctx.set_materialize_grads(False)
        return out, eft, inv, pidx

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, *_):
        if grad is None:
            return (None,) * 5
        eft, inv = ctx.saved_tensors
        return moe_permute_backward(grad, inv, eft, *ctx.tokens), None, None, None, None


class _ReturnRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, inv, eft):
        out = torch.empty((weights.size(0), rows.size(1)), dtype=rows.dtype, device=rows.device)
        launch("i8moe_moe_unpermute", rows.device, rows.data_ptr(), _DT[rows.dtype],
               weights.data_ptr(), inv.data_ptr(), *_eft_args(eft), weights.size(0),
               weights.size(1), rows.size(1), out.data_ptr())
        ctx.save_for_backward(rows, weights, inv, eft)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, weights, inv, eft = ctx.saved_tensors
        dy, dw = moe_unpermute_backward(grad, rows, weights, inv, eft)
        return (dy if ctx.needs_input_grad[0] else None,
                dw if ctx.needs_input_grad[1] else None, None, None)


def moe_permute_train(hidden_states, topk_ids, n_expert: int, n_local_expert: int = -1,
                      expert_map=None):
    """``moe_permute`` for training: differentiable in hidden_states (once).

    Returns (permuted_hidden_states [T * topk, hidden],
    expert_first_token_offset, inv_permuted_idx (flat), permuted_idx); rows of
    no local expert are zero and give no gradient."""
    what = "moe_permute_train"
    _check_rows(what, "hidden_states", hidden_states)
    dev = hidden_states.device
    _check(topk_ids.dim() == 2 and topk_ids.size(0) == hidden_states.size(0)
           and topk_ids.size(1) >= 1 and topk_ids.device == dev,
           f"{what}: topk_ids must have shape [n_token, topk] on hidden_states' device")
    _check(not topk_ids.is_floating_point(), f"{what}: topk_ids must be integers")
    if n_local_expert == -1:
        n_local_expert = n_expert
    _check(1 <= n_expert <= 2048 and 0 <= n_local_expert <= n_expert,
           f"{what}: n_expert must be in [1, 2048] and n_local_expert in [0, n_expert]")
    if expert_map is not None:
        _check(expert_map.dtype == torch.int32 and expert_map.is_contiguous()
               and expert_map.device == dev and expert_map.shape == (n_expert,),
               f"{what}: expert_map must be contiguous int32 [n_expert] on hidden_states' device")
    ids = topk_ids.to(torch.int32).contiguous()
    return _SortRows.apply(_aligned(hidden_states), ids, expert_map, n_expert, n_local_expert)


def moe_unpermute_train(permuted_hidden_states, topk_weights, inv_permuted_idx,
                        expert_first_token_offset=None):
    """``moe_unpermute`` for training: returns [n_token, hidden],
    differentiable in permuted_hidden_states and topk_weights (once)."""
    what = "moe_unpermute_train"
    _check_rows(what, "permuted_hidden_states", permuted_hidden_states)
    dev = permuted_hidden_states.device
    _check(topk_weights.dim() == 2 and topk_weights.size(1) >= 1 and topk_weights.device == dev
           and permuted_hidden_states.size(0) == topk_weights.numel(),
           f"{what}: permuted_hidden_states must have one row per element of topk_weights "
           "[n_token, topk]")
    _check_maps(what, inv_permuted_idx, expert_first_token_offset, topk_weights.numel(), dev)
    return _ReturnRows.apply(_aligned(permuted_hidden_states),
                             topk_weights.to(torch.float32).contiguous(), inv_permuted_idx,
                             expert_first_token_offset)
