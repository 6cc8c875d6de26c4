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
#include <initializer_list>

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

// Rows of local experts; the entry points bound n_token * topk by 2^31.
__device__ __forceinline__ int valid_rows(const RowArgs& a) {
  const int total = a.n_token * a.topk;
  if (a.eft == nullptr) return total;
  const int64_t v = __ldg(a.eft + a.n_local);
  return v < total ? static_cast<int>(v) : total;
}

// Vector v of row r.
template <typename V>
__device__ __forceinline__ V* vec(V* rows, const RowArgs& a, int64_t r, int v) {
  return rows + r * a.vpr + v;
}

// Sorted row of slot s, or -1 (and the error bit) when the map is no map.
__device__ __forceinline__ int sorted_row(const RowArgs& a, int64_t s) {
  const int d = __ldg(a.inv + s);
  if (d >= 0 && d < a.n_token * a.topk) return d;
  atomicOr(&g_err_route_grad, kErrBadIndex);
  return -1;
}


// Sorted rows of up to kSlots of token t's slots from j0 on; -1 for none.
template <int kSlots>
__device__ __forceinline__ void sorted_rows(const RowArgs& a, int64_t t, int j0, int* d) {
#pragma unroll
  for (int j = 0; j < kSlots; ++j) d[j] = j0 + j < a.topk ? sorted_row(a, t * a.topk + j0 + j) : -1;
}

// One token per CTA: its row is read once and written topk times.
__global__ void __launch_bounds__(256) scatter_rows_kernel(RowArgs a, const uint4* __restrict__ x,
                                                           uint4* __restrict__ out) {
  constexpr int kSlots = 8;
  const int valid = valid_rows(a);
  const int64_t t = blockIdx.x;
  for (int v = threadIdx.x; v < a.vpr; v += blockDim.x) {
    const uint4 row = __ldg(x + t * a.vpr + v);
    for (int j0 = 0; j0 < a.topk; j0 += kSlots) {
      int d[kSlots];
      sorted_rows<kSlots>(a, t, j0, d);
#pragma unroll
      for (int j = 0; j < kSlots; ++j)
        if (d[j] >= 0) *vec(out, a, d[j], v) = d[j] < valid ? row : make_uint4(0, 0, 0, 0);
    }
  }
}

// One token per CTA, four of its rows in flight by predicated loads; rows that do
// not count are not read.  Bound by memory: 8192 x 2048 bf16, top 8 (302 MB) takes
// 47 us right after the kernel that wrote the rows, 55 with other data in L2, 45
// replayed over three inputs, and 16384 x 4096 fp16 175; replayed without the
// loads' evict-first hint 48, without the stores' 43 and 184.
template <typename T>
__global__ void __launch_bounds__(256, 6) gather_sum_kernel(RowArgs a,
                                                            const uint4* __restrict__ rows,
                                                            uint4* __restrict__ out) {
  constexpr int EPV = 16 / sizeof(T), kSlots = 4;
  const int valid = valid_rows(a);
  const int64_t t = blockIdx.x;
  for (int v = threadIdx.x; v < a.vpr; v += blockDim.x) {
    float acc[EPV];
#pragma unroll
    for (int e = 0; e < EPV; ++e) acc[e] = 0.f;
    for (int j0 = 0; j0 < a.topk; j0 += kSlots) {
      int d[kSlots];
      uint4 raw[kSlots];
      sorted_rows<kSlots>(a, t, j0, d);
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (d[j] >= valid) d[j] = -1;
        raw[j] = load_if(d[j], vec(rows, a, d[j], v));
      }
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        const T* p = reinterpret_cast<const T*>(&raw[j]);
#pragma unroll
        for (int e = 0; e < EPV; ++e) acc[e] += d[j] < 0 ? 0.f : Num<T>::to_f(p[e]);
      }
    }
    uint4 o;
    T* ov = reinterpret_cast<T*>(&o);
#pragma unroll
    for (int e = 0; e < EPV; ++e) ov[e] = Num<T>::from_f(acc[e]);
    __stcs(out + t * a.vpr + v, o);
  }
}

// One token per CTA: its gradient is read once for all of its rows, four of
// which are in flight, and their dot products are reduced together.  Bound by
// memory: 8192 x 2048 bf16, top 8 (570 MB, half of it written) takes 100 us, 5.7
// TB/s where a copy has 6.6; with eight rows in flight 125 us (registers for two
// CTAs an SM only), with two 101.
template <typename T>
__global__ void __launch_bounds__(256, 4) return_grad_kernel(RowArgs a, const uint4* __restrict__ dout,
                                                          const uint4* __restrict__ rows,
                                                          const float* __restrict__ w,
                                                          uint4* __restrict__ drows,
                                                          float* __restrict__ dw) {
  constexpr int EPV = 16 / sizeof(T), kSlots = 4;
  __shared__ float s_dot[8][kSlots];
  const int valid = valid_rows(a);
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int j0 = 0; j0 < a.topk; j0 += kSlots) {
    int d[kSlots];
    float wt[kSlots], dot[kSlots];
    sorted_rows<kSlots>(a, t, j0, d);
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      wt[j] = d[j] >= 0 && d[j] < valid ? __ldg(w + t * a.topk + j0 + j) : 0.f;
      dot[j] = 0.f;
    }
    for (int v = threadIdx.x; v < a.vpr; v += blockDim.x) {
      const uint4 g = __ldg(dout + t * a.vpr + v);
      uint4 raw[kSlots];
#pragma unroll
      for (int j = 0; j < kSlots; ++j)
        raw[j] = d[j] >= 0 && d[j] < valid ? __ldg(vec(rows, a, d[j], v)) : make_uint4(0, 0, 0, 0);
      float gf[EPV];
      const T* gp = reinterpret_cast<const T*>(&g);
#pragma unroll
      for (int e = 0; e < EPV; ++e) gf[e] = Num<T>::to_f(gp[e]);
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (d[j] < 0) continue;
        const bool on = d[j] < valid;
        const T* yp = reinterpret_cast<const T*>(&raw[j]);
        uint4 o = make_uint4(0, 0, 0, 0);
        if (on) {
          T* op = reinterpret_cast<T*>(&o);
#pragma unroll
          for (int e = 0; e < EPV; ++e) {
            dot[j] = fmaf(gf[e], Num<T>::to_f(yp[e]), dot[j]);
            op[e] = Num<T>::from_f(wt[j] * gf[e]);
          }
        }
        *vec(drows, a, d[j], v) = o;
      }
    }
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], o);
      if (lane == 0) s_dot[warp][j] = dot[j];
    }
    __syncthreads();
    if (threadIdx.x < kSlots && j0 + static_cast<int>(threadIdx.x) < a.topk) {
      float sum = 0.f;
      for (int i = 0; i < warps; ++i) sum += s_dot[i][threadIdx.x];
      dw[t * a.topk + j0 + threadIdx.x] = sum;
    }
    if (j0 + kSlots < a.topk) __syncthreads();  // s_dot is written again
  }
}

// Checks shared by the entry points; fills `a`.
int row_args(const char* what, int dtype, const int32_t* inv, const int64_t* eft, int64_t n_local,
             int64_t n_token, int64_t topk, int64_t n_hidden,
             std::initializer_list<const void*> rows, RowArgs* a) {
  I8_REQUIRE(dtype == I8MOE_BF16 || dtype == I8MOE_FP16 || dtype == I8MOE_FP32,
             "%s: unsupported dtype", what);
  I8_REQUIRE(topk >= 1, "%s: topk must be positive", what);
  I8_REQUIRE(n_token >= 0 && n_token <= INT32_MAX / topk, "%s: n_token * topk must fit in int32",
             what);
  I8_REQUIRE(n_hidden >= 0 && n_hidden < (int64_t(1) << 31), "%s: bad n_hidden", what);
  const int64_t row_bytes = n_hidden * (dtype == I8MOE_FP32 ? 4 : 2);
  I8_REQUIRE(row_bytes % 16 == 0, "%s: hidden row must be a multiple of 16 bytes", what);
  if (n_token > 0 && n_hidden > 0)
    for (const void* p : rows) {
      I8_REQUIRE(p != nullptr, "%s: every tensor must be given", what);
      I8_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0,
                 "%s: tensors must be 16-byte aligned", what);
    }
  I8_REQUIRE(n_token == 0 || inv != nullptr, "%s: every tensor must be given", what);
  I8_REQUIRE(eft == nullptr || n_local >= 0, "%s: bad n_local_expert", what);
  *a = RowArgs{inv, eft, static_cast<int>(n_local), static_cast<int>(n_token),
               static_cast<int>(topk), static_cast<int>(row_bytes / 16)};
  return I8MOE_OK;
}

// Threads of a CTA for rows of that many vectors.
int row_threads(int vpr) { return std::min(256, (vpr + 31) / 32 * 32); }

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
                          {input, permuted_input}, &a);
  if (rc != I8MOE_OK) return rc;
  if (n_token == 0 || n_hidden == 0) return I8MOE_OK;
  scatter_rows_kernel<<<static_cast<unsigned>(n_token), row_threads(a.vpr), 0,
                        static_cast<cudaStream_t>(stream)>>>(
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
                          {permuted_grad, input_grad}, &a);
  if (rc != I8MOE_OK) return rc;
  if (n_token == 0 || n_hidden == 0) return I8MOE_OK;
  const uint4* in = static_cast<const uint4*>(permuted_grad);
  uint4* out = static_cast<uint4*>(input_grad);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(n_token);
  const int threads = row_threads(a.vpr);
  if (dtype == I8MOE_BF16) gather_sum_kernel<__nv_bfloat16><<<grid, threads, 0, st>>>(a, in, out);
  else if (dtype == I8MOE_FP16) gather_sum_kernel<__half><<<grid, threads, 0, st>>>(a, in, out);
  else gather_sum_kernel<float><<<grid, threads, 0, st>>>(a, in, out);
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
               {out_grad, permuted_hidden, permuted_grad}, &a);
  if (rc != I8MOE_OK) return rc;
  if (n_token == 0) return I8MOE_OK;
  I8_REQUIRE(topk_weights && weights_grad, "moe_unpermute_backward: every tensor must be given");
  const uint4* g = static_cast<const uint4*>(out_grad);
  const uint4* y = static_cast<const uint4*>(permuted_hidden);
  uint4* dy = static_cast<uint4*>(permuted_grad);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(n_token);
  const int threads = std::max(32, row_threads(a.vpr));
  if (dtype == I8MOE_BF16)
    return_grad_kernel<__nv_bfloat16><<<grid, threads, 0, st>>>(a, g, y, topk_weights, dy, weights_grad);
  else if (dtype == I8MOE_FP16)
    return_grad_kernel<__half><<<grid, threads, 0, st>>>(a, g, y, topk_weights, dy, weights_grad);
  else
    return_grad_kernel<float><<<grid, threads, 0, st>>>(a, g, y, topk_weights, dy, weights_grad);
  return check_launch("moe_unpermute_backward");
}

}  // extern "C"
