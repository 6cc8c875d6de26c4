// The rows' way to the experts and back for training: the row scatter in
// expert order, and the gradients of the scatter and of the top-k weighted
// return (i8moe_moe_unpermute).  No reference counterpart.
//
// With d = inv[t, j] the sorted row of token t's j-th expert, and rows past
// expert_first_token_offset[n_local] (no local expert) counting as zero:
//   scatter:             P[d] = x[t]
//   its gradient:        dx[t] = sum_j dP[d]
//   gradient of the return out[t] = sum_j w[t, j] Y[d]:
//                        dY[d] = w[t, j] dout[t],  dw[t, j] = <dout[t], Y[d]>
// inv is a permutation of the n_token * topk rows, so every row of P and dY
// is written exactly once, and nothing is added in an order that varies.
#include <algorithm>

#include "common.cuh"

namespace i8moe {

static __device__ unsigned g_err_route_grad;

int read_route_grad_error(uint32_t* w, int clear) {
  unsigned v = 0;
  I8_CUDA(cudaMemcpyFromSymbol(&v, g_err_route_grad, sizeof(v)));
  if (clear) {
    unsigned z = 0;
    I8_CUDA(cudaMemcpyToSymbol(g_err_route_grad, &z, sizeof(z)));
  }
  *w = v;
  return I8MOE_OK;
}

namespace {

struct RowArgs {
  const int32_t* inv;  // [n_token * topk]
  const int64_t* eft;  // nullable: every row is valid
  int n_local;
  int n_token, topk;
  int vpr;  // 16-byte vectors per row
};

__device__ __forceinline__ int64_t valid_rows(const RowArgs& a) {
  const int64_t total = static_cast<int64_t>(a.n_token) * a.topk;
  if (a.eft == nullptr) return total;
  const int64_t v = __ldg(a.eft + a.n_local);
  return v < total ? v : total;
}

// Sorted row of slot s, or -1 (and the error bit) when the map is no map.
__device__ __forceinline__ int64_t sorted_row(const RowArgs& a, int64_t s) {
  const int64_t d = __ldg(a.inv + s);
  if (d >= 0 && d < static_cast<int64_t>(a.n_token) * a.topk) return d;
  atomicOr(&g_err_route_grad, kErrBadIndex);
  return -1;
}

__global__ void __launch_bounds__(256) scatter_rows_kernel(RowArgs a, const uint4* __restrict__ x,
                                                           uint4* __restrict__ out) {
  const int64_t valid = valid_rows(a);
  for (int64_t t = blockIdx.x; t < a.n_token; t += gridDim.x)
    for (int v = threadIdx.x; v < a.vpr; v += blockDim.x) {
      const uint4 row = __ldg(x + t * a.vpr + v);
      for (int j = 0; j < a.topk; ++j) {
        const int64_t d = sorted_row(a, t * a.topk + j);
        if (d >= 0) out[d * a.vpr + v] = d < valid ? row : make_uint4(0, 0, 0, 0);
      }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) gather_sum_kernel(RowArgs a, const uint4* __restrict__ rows,
                                                         uint4* __restrict__ out) {
  constexpr int EPV = 16 / sizeof(T);
  const int64_t valid = valid_rows(a);
  for (int64_t t = blockIdx.x; t < a.n_token; t += gridDim.x)
    for (int v = threadIdx.x; v < a.vpr; v += blockDim.x) {
      float acc[EPV];
#pragma unroll
      for (int e = 0; e < EPV; ++e) acc[e] = 0.f;
      for (int j = 0; j < a.topk; ++j) {
        const int64_t d = sorted_row(a, t * a.topk + j);
        if (d < 0 || d >= valid) continue;
        const uint4 raw = __ldg(rows + d * a.vpr + v);
        const T* p = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int e = 0; e < EPV; ++e) acc[e] += Num<T>::to_f(p[e]);
      }
      uint4 o;
      T* ov = reinterpret_cast<T*>(&o);
#pragma unroll
      for (int e = 0; e < EPV; ++e) ov[e] = Num<T>::from_f(acc[e]);
      out[t * a.vpr + v] = o;
    }
}

// One warp per slot (t, j).
template <typename T>
__global__ void __launch_bounds__(256) return_grad_kernel(RowArgs a, const uint4* __restrict__ dout,
                                                          const uint4* __restrict__ rows,
                                                          const float* __restrict__ w,
                                                          uint4* __restrict__ drows,
                                                          float* __restrict__ dw) {
  constexpr int EPV = 16 / sizeof(T);
  const int64_t valid = valid_rows(a);
  const int64_t slots = static_cast<int64_t>(a.n_token) * a.topk;
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t s = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
       s < slots; s += warps) {
    const int64_t t = s / a.topk;
    const int64_t d = sorted_row(a, s);
    const bool on = d >= 0 && d < valid;
    const float wt = on ? __ldg(w + s) : 0.f;
    float dot = 0.f;
    for (int v = lane; v < a.vpr && d >= 0; v += 32) {
      uint4 o = make_uint4(0, 0, 0, 0);
      if (on) {
        const uint4 g = __ldg(dout + t * a.vpr + v);
        const uint4 y = __ldg(rows + d * a.vpr + v);
        const T* gp = reinterpret_cast<const T*>(&g);
        const T* yp = reinterpret_cast<const T*>(&y);
        T* op = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
          const float ge = Num<T>::to_f(gp[e]);
          dot = fmaf(ge, Num<T>::to_f(yp[e]), dot);
          op[e] = Num<T>::from_f(wt * ge);
        }
      }
      drows[d * a.vpr + v] = o;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane == 0) dw[s] = dot;
  }
}

// Checks shared by the entry points; fills `a`.
int row_args(const char* what, int dtype, const int32_t* inv, const int64_t* eft, int64_t n_local,
             int64_t n_token, int64_t topk, int64_t n_hidden, uintptr_t pointers, RowArgs* a) {
  I8_REQUIRE(dtype == I8MOE_BF16 || dtype == I8MOE_FP16 || dtype == I8MOE_FP32,
             "%s: unsupported dtype", what);
  I8_REQUIRE(topk >= 1, "%s: topk must be positive", what);
  I8_REQUIRE(n_token >= 0 && n_token <= INT32_MAX / topk, "%s: n_token * topk must fit in int32",
             what);
  I8_REQUIRE(n_hidden >= 0 && n_hidden < (int64_t(1) << 31), "%s: bad n_hidden", what);
  const int64_t row_bytes = n_hidden * (dtype == I8MOE_FP32 ? 4 : 2);
  I8_REQUIRE(row_bytes % 16 == 0, "%s: hidden row must be a multiple of 16 bytes", what);
  I8_REQUIRE(pointers % 16 == 0, "%s: tensors must be 16-byte aligned", what);
  I8_REQUIRE(eft == nullptr || n_local >= 0, "%s: bad n_local_expert", what);
  *a = RowArgs{inv, eft, static_cast<int>(n_local), static_cast<int>(n_token),
               static_cast<int>(topk), static_cast<int>(row_bytes / 16)};
  return I8MOE_OK;
}

uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

unsigned row_grid(int64_t n, int per_sm) {
  return static_cast<unsigned>(std::min<int64_t>(n, int64_t(num_sms(current_device())) * per_sm));
}

}  // namespace
}  // namespace i8moe

using namespace i8moe;

extern "C" {

int i8moe_moe_scatter_rows(const void* input, int dtype, const int32_t* inv_permuted_idx,
                           const int64_t* expert_first_token_offset, int64_t n_local_expert,
                           int64_t n_token, int64_t topk, int64_t n_hidden, void* permuted_input,
                           i8moe_stream_t stream) {
  RowArgs a;
  const int rc = row_args("moe_scatter_rows", dtype, inv_permuted_idx, expert_first_token_offset,
                          n_local_expert, n_token, topk, n_hidden,
                          bits(input) | bits(permuted_input), &a);
  if (rc != I8MOE_OK) return rc;
  if (n_token == 0 || n_hidden == 0) return I8MOE_OK;
  scatter_rows_kernel<<<row_grid(n_token, 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      a, static_cast<const uint4*>(input), static_cast<uint4*>(permuted_input));
  return check_launch("moe_scatter_rows");
}

int i8moe_moe_permute_backward(const void* permuted_grad, int dtype,
                               const int32_t* inv_permuted_idx,
                               const int64_t* expert_first_token_offset, int64_t n_local_expert,
                               int64_t n_token, int64_t topk, int64_t n_hidden, void* input_grad,
                               i8moe_stream_t stream) {
  RowArgs a;
  const int rc = row_args("moe_permute_backward", dtype, inv_permuted_idx,
                          expert_first_token_offset, n_local_expert, n_token, topk, n_hidden,
                          bits(permuted_grad) | bits(input_grad), &a);
  if (rc != I8MOE_OK) return rc;
  if (n_token == 0 || n_hidden == 0) return I8MOE_OK;
  const uint4* in = static_cast<const uint4*>(permuted_grad);
  uint4* out = static_cast<uint4*>(input_grad);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = row_grid(n_token, 8);
  if (dtype == I8MOE_BF16) gather_sum_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a, in, out);
  else if (dtype == I8MOE_FP16) gather_sum_kernel<__half><<<grid, 256, 0, st>>>(a, in, out);
  else gather_sum_kernel<float><<<grid, 256, 0, st>>>(a, in, out);
  return check_launch("moe_permute_backward");
}

int i8moe_moe_unpermute_backward(const void* out_grad, const void* permuted_hidden, int dtype,
                                 const float* topk_weights, const int32_t* inv_permuted_idx,
                                 const int64_t* expert_first_token_offset, int64_t n_local_expert,
                                 int64_t n_token, int64_t topk, int64_t n_hidden,
                                 void* permuted_grad, float* weights_grad, i8moe_stream_t stream) {
  RowArgs a;
  const int rc =
      row_args("moe_unpermute_backward", dtype, inv_permuted_idx, expert_first_token_offset,
               n_local_expert, n_token, topk, n_hidden,
               bits(out_grad) | bits(permuted_hidden) | bits(permuted_grad), &a);
  if (rc != I8MOE_OK) return rc;
  if (n_token == 0) return I8MOE_OK;
  const uint4* g = static_cast<const uint4*>(out_grad);
  const uint4* y = static_cast<const uint4*>(permuted_hidden);
  uint4* dy = static_cast<uint4*>(permuted_grad);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = row_grid((n_token * topk + 7) / 8, 8);
  if (dtype == I8MOE_BF16)
    return_grad_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a, g, y, topk_weights, dy, weights_grad);
  else if (dtype == I8MOE_FP16)
    return_grad_kernel<__half><<<grid, 256, 0, st>>>(a, g, y, topk_weights, dy, weights_grad);
  else
    return_grad_kernel<float><<<grid, 256, 0, st>>>(a, g, y, topk_weights, dy, weights_grad);
  return check_launch("moe_unpermute_backward");
}

}  // extern "C"
