"""Expert layers with 4-bit weights and group scales for decoding (no
reference counterpart): the weights' quantisation, the products of each
expert's few rows, and the layer's forward.

Weights are kept as ``packed`` uint8 [E, N, K/2], column k in byte k // 2 (low
half for even k) as q + 8 with q in [-8, 7], and ``scale`` [E, N,
ceil(K / group_size)]; a weight is scale * q.  Activations are bf16 or fp16.
The kernels read the weights of the experts that have rows once per eight
rows, so they are for few rows per expert.  64 experts of 1024 x 2048: up to 8
rows each take 22 us, where the INT8 grouped GEMM takes 31; from 12 on (36) the
INT8 product is the faster one, with 64 rows 34 against 117 us.
"""

from __future__ import annotations

import torch

from ._lib import BF16, FP16, FP32, TORCH_OPS, launch
from .permute import moe_route_for_gemm, moe_unpermute

_DT = {torch.bfloat16: BF16, torch.float16: FP16, torch.float32: FP32}


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def quantize_weights_int4(w: torch.Tensor, group_size: int = 128, scale_dtype=None):
    """(packed, scale) of w [E, N, K] (bf16, fp16 or fp32): per group
    scale = max|w| / 7 rounded to ``scale_dtype`` (w's type when omitted) and
    q = clamp(rint(w / scale), -8, 7).  K must be a multiple of 32,
    group_size 32, 64 or 128; the last group of a row may be shorter.  The
    products take scales of the activations' type: give ``scale_dtype`` for
    fp32 weights.  A group with a NaN gets scale NaN, one whose scale leaves
    its type inf; their q is 0 and products by them are NaN.  No gradients."""
    scale_dtype = w.dtype if scale_dtype is None else scale_dtype
    _check(w.is_cuda and w.dim() == 3, "quantize_weights_int4: w must be a CUDA tensor [E, N, K]")
    _check(w.dtype in _DT and scale_dtype in _DT, "quantize_weights_int4: unsupported dtype")
    _check(group_size in (32, 64, 128),
           "quantize_weights_int4: group_size must be 32, 64 or 128")
    E, N, K = w.shape
    _check(K % 32 == 0, "quantize_weights_int4: K must be divisible by 32")
    w = w.contiguous()
    packed = torch.empty((E, N, K // 2), dtype=torch.uint8, device=w.device)
    scale = torch.empty((E, N, -(-K // group_size)), dtype=scale_dtype, device=w.device)
    launch("i8moe_quantize_weights_int4", w.device, w.data_ptr(), _DT[w.dtype], E, N, K,
           group_size, packed.data_ptr(), scale.data_ptr(), _DT[scale_dtype])
    return packed, scale


def int4_grouped_mv(x, w_packed, w_scale, expert_offsets, group_size: int = 128,
                    permuted_idx=None, topk: int = 1, silu: bool = False, out=None):
    """Rows r in [expert_offsets[e], expert_offsets[e+1]) times the transposed
    weights of expert e.

    x [rows, K] holds the sorted rows; with ``permuted_idx`` (int32 [rows])
    row r is x[permuted_idx[r] // topk] instead.  ``silu``: w_packed holds N/2
    gate rows and then N/2 up rows, and the result is silu(gate) * up.
    Returns ``out`` [rows, N] (N/2 with silu) in x's type, allocated when not
    given; rows outside every expert keep what it held.  Sums are fp32,
    rounded once; a group's sum comes before its scale, of up to 128 terms of
    up to 8 |x| (bf16 values above 2^117 may leave fp32).  No gradients."""
    return TORCH_OPS.int4_grouped_mv(x, w_packed, w_scale, expert_offsets, group_size, permuted_idx,
                                     topk, silu, out)


def run_int4_moe(output, hidden_states, w1_packed, w1_scale, w2_packed, w2_scale, topk_ids,
                 topk_weights, global_num_experts: int, expert_map=None,
                 group_size: int = 128) -> None:
    """MoE forward of a decoding step with 4-bit weights; writes ``output``
    [T, K].  w1 [E, 2N, K] (gate rows, then up rows) and w2 [E, K, N] as
    ``quantize_weights_int4`` packs them, E being the local experts;
    ``expert_map`` as in the INT8 forward.  Four launches for up to
    2048 rows, six for more, no host synchronisation; it can be captured into
    a CUDA graph."""
    _check(hidden_states.dim() == 2 and w1_packed.dim() == 3 and w2_packed.dim() == 3,
           "run_int4_moe: hidden_states must be [T, K], the weights [E, rows, columns / 2]")
    _check(hidden_states.is_cuda and topk_ids.device == hidden_states.device
           and topk_weights.device == hidden_states.device,
           "run_int4_moe: hidden_states, topk_ids and topk_weights must be on one CUDA device")
    T, K = hidden_states.shape
    E, two_n, _ = w1_packed.shape
    _check(2 * w1_packed.size(2) == K and w2_packed.shape == (E, K, two_n // 4) and two_n % 4 == 0,
           "run_int4_moe: w1 must be [E, 2N, K] and w2 [E, K, N]")
    _check(expert_map is None or (expert_map.dtype == torch.int32 and expert_map.is_contiguous()
                                  and expert_map.shape == (global_num_experts,)
                                  and expert_map.device == hidden_states.device),
           "run_int4_moe: expert_map must be contiguous int32 [global_num_experts]")
    _check(topk_ids.dim() == 2 and topk_ids.size(0) == T and topk_weights.shape == topk_ids.shape,
           "run_int4_moe: topk_ids and topk_weights must have shape [T, topk]")
    _check(output.shape == hidden_states.shape and output.dtype == hidden_states.dtype
           and output.is_contiguous() and output.device == hidden_states.device,
           "run_int4_moe: output must be contiguous [T, K] of hidden_states' dtype and device")
    topk = topk_ids.size(1)
    eft, inv, pidx, eo, _, _, _ = moe_route_for_gemm(
        topk_ids.contiguous(), T, global_num_experts, E, expert_map, two_n, K, K, two_n // 2, 64)
    act = int4_grouped_mv(hidden_states, w1_packed, w1_scale, eo, group_size, permuted_idx=pidx,
                          topk=topk, silu=True)
    mm2 = int4_grouped_mv(act, w2_packed, w2_scale, eo, group_size)
    moe_unpermute(output, mm2, topk_weights.contiguous(), inv, eft)
