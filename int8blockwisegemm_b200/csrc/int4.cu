// Experts' products of a few tokens with 4-bit weights and group scales
// (weights as they are kept for decoding), and the weights' quantisation.  No
// reference counterpart: beside the INT8 grouped GEMM, it reads half the
// bytes of weights per token.
//
//   out[r, n] = sum_k x[src(r), k] * scale[e, n, k / G] * (u[e, n, k] - 8)
//
// for the rows expert_offsets[e] <= r < expert_offsets[e + 1] of expert e,
// src(r) = r or permuted_idx[r] / topk.  u is the nibble of column k: byte
// k / 2 of the weight's row, low half for even k.  With `silu` the first half
// of the n rows is a gate and the second half its factor:
//   out[r, n] = silu(gate[r, n]) * up[r, n],  n < N / 2.
// Sums are fp32 and rounded once, after the activation.
#include <algorithm>

#include "common.cuh"

namespace i8moe {

static __device__ unsigned g_err_int4;

int read_int4_error(uint32_t* w, int clear) {
  unsigned v = 0;
  I8_CUDA(cudaMemcpyFromSymbol(&v, g_err_int4, sizeof(v)));
  if (clear) {
    unsigned z = 0;
    I8_CUDA(cudaMemcpyToSymbol(g_err_int4, &z, sizeof(z)));
  }
  *w = v;
  return I8MOE_OK;
}

namespace {

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == I8MOE_BF16) return Num<__nv_bfloat16>::to_f(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == I8MOE_FP16) return Num<__half>::to_f(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

struct MvArgs {
  const void* x;
  int64_t x_stride;  // elements
  int64_t x_rows;
  const int32_t* pidx;  // nullable
  int topk;
  const uint8_t* w;  // [E, N, K / 2]
  const void* scale;  // [E, N, groups]
  int scale_dtype;
  int group, groups;
  const int32_t* eo;  // [E + 1]
  int n_expert;
  int64_t rows;
  int n, k;
  void* out;  // [rows, N] or [rows, N / 2]
};

// Rows of expert e, clipped to the output: empty (and the error bit) when the
// offsets are out of order.
__device__ __forceinline__ void expert_rows(const MvArgs& a, int e, int64_t* r0, int64_t* r1) {
  *r0 = __ldg(a.eo + e);
  *r1 = __ldg(a.eo + e + 1);
  if (*r0 < 0 || *r1 < *r0 || *r1 > a.rows) {
    atomicOr(&g_err_int4, kErrBadProblem);
    *r1 = *r0;
  }
}

__device__ __forceinline__ int64_t source_row(const MvArgs& a, int64_t r) {
  if (a.pidx == nullptr) return r;
  const int32_t p = __ldg(a.pidx + r);
  const int64_t t = p / a.topk;
  if (p >= 0 && t < a.x_rows) return t;
  atomicOr(&g_err_int4, kErrBadIndex);
  return -1;  // counts as a row of zeros
}

__device__ __forceinline__ float silu_mul(float gate, float up) {
  return __fdiv_rn(gate, 1.f + expf(-gate)) * up;
}

// One warp per output column of an expert and eight of its rows at a time;
// lane l takes the 8-column words l, l + 32, ... of the weight's row.
template <typename T, bool kSilu>
__global__ void __launch_bounds__(256) mv_warp_kernel(MvArgs a) {
  constexpr int kRows = 8;
  const int e = blockIdx.y;
  int64_t r0, r1;
  expert_rows(a, e, &r0, &r1);
  if (r0 == r1) return;
  const int lane = threadIdx.x & 31;
  const int n_out = kSilu ? a.n / 2 : a.n;
  const int n = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (n >= n_out) return;
  const T* x = static_cast<const T*>(a.x);
  for (int64_t r = r0; r < r1; r += kRows) {
    float acc[2][kRows];
#pragma unroll
    for (int half = 0; half < (kSilu ? 2 : 1); ++half) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) acc[half][i] = 0.f;
      const int64_t wn = static_cast<int64_t>(e) * a.n + n + half * n_out;
      const uint32_t* w = reinterpret_cast<const uint32_t*>(a.w) + wn * (a.k / 8);
      for (int word = lane; word < a.k / 8; word += 32) {
        const uint32_t u = __ldg(w + word);
        const float s = load_any(a.scale, a.scale_dtype, wn * a.groups + word * 8 / a.group);
        for (int i = 0; i < kRows && r + i < r1; ++i) {
          const int64_t src = source_row(a, r + i);
          if (src < 0) continue;
          const T* xr = x + src * a.x_stride + word * 8;
          float part = 0.f;
#pragma unroll
          for (int c = 0; c < 8; ++c)
            part = fmaf(Num<T>::to_f(xr[c]), static_cast<float>((u >> (4 * c)) & 15u) - 8.f, part);
          acc[half][i] = fmaf(part, s, acc[half][i]);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          acc[half][i] += __shfl_xor_sync(0xffffffffu, acc[half][i], o);
    }
    if (lane == 0)
      for (int i = 0; i < kRows && r + i < r1; ++i)
        static_cast<T*>(a.out)[(r + i) * n_out + n] =
            Num<T>::from_f(kSilu ? silu_mul(acc[0][i], acc[1][i]) : acc[0][i]);
  }
}

template <typename T>
int launch_mv(const MvArgs& a, bool silu, cudaStream_t st) {
  const int n_out = silu ? a.n / 2 : a.n;
  const dim3 grid((n_out + 7) / 8, a.n_expert);
  if (silu) mv_warp_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else mv_warp_kernel<T, false><<<grid, 256, 0, st>>>(a);
  return check_launch("int4_grouped_mv");
}

// One warp per group: scale = max|w| / 7 rounded to the scale's type, and
// u = clamp(rint(w / scale), -8, 7) + 8 by that rounded scale, so that its
// rounding shifts no weight twice.  A group of zeros (or one whose scale
// rounds to zero) gets scale 0 and u = 8.
template <typename T, typename S>
__global__ void __launch_bounds__(256) quantize_int4_kernel(const T* __restrict__ w, int64_t rows,
                                                            int k, int group, int groups,
                                                            uint8_t* __restrict__ packed,
                                                            S* __restrict__ scale) {
  const int lane = threadIdx.x & 31;
  const int64_t total = rows * groups;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
       i < total; i += warps) {
    const int64_t row = i / groups;
    const int g = static_cast<int>(i - row * groups);
    const int k0 = g * group;
    const int k1 = min(k, k0 + group);
    const T* src = w + row * k;
    float m = 0.f;
    for (int c = k0 + lane; c < k1; c += 32) m = fmaxf(m, fabsf(Num<T>::to_f(src[c])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const S s = Num<S>::from_f(__fdiv_rn(m, 7.f));
    const float sf = Num<S>::to_f(s);
    if (lane == 0) scale[i] = s;
    for (int c = k0 + 2 * lane; c < k1; c += 64) {
      int u[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float v = Num<T>::to_f(src[c + b]);
        const int q = sf > 0.f ? __float2int_rn(__fdiv_rn(v, sf)) : 0;
        u[b] = max(-8, min(7, q)) + 8;
      }
      packed[row * (k / 2) + c / 2] = static_cast<uint8_t>(u[0] | (u[1] << 4));
    }
  }
}

template <typename T>
int launch_quantize(const void* w, int64_t rows, int k, int group, int groups, uint8_t* packed,
                    void* scale, int scale_dtype, cudaStream_t st) {
  const int64_t warps = rows * groups;
  const unsigned grid = static_cast<unsigned>(
      std::min<int64_t>((warps + 7) / 8, int64_t(num_sms(current_device())) * 16));
  const T* src = static_cast<const T*>(w);
  if (scale_dtype == I8MOE_BF16)
    quantize_int4_kernel<<<grid, 256, 0, st>>>(src, rows, k, group, groups, packed,
                                               static_cast<__nv_bfloat16*>(scale));
  else if (scale_dtype == I8MOE_FP16)
    quantize_int4_kernel<<<grid, 256, 0, st>>>(src, rows, k, group, groups, packed,
                                               static_cast<__half*>(scale));
  else
    quantize_int4_kernel<<<grid, 256, 0, st>>>(src, rows, k, group, groups, packed,
                                               static_cast<float*>(scale));
  return check_launch("quantize_weights_int4");
}

bool float_dtype(int d) { return d == I8MOE_BF16 || d == I8MOE_FP16 || d == I8MOE_FP32; }

uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

}  // namespace
}  // namespace i8moe

using namespace i8moe;

extern "C" {

int i8moe_quantize_weights_int4(const void* w, int dtype, int64_t n_expert, int64_t n, int64_t k,
                                int64_t group_size, uint8_t* packed, void* scale, int scale_dtype,
                                i8moe_stream_t stream) {
  I8_REQUIRE(float_dtype(dtype) && float_dtype(scale_dtype),
             "quantize_weights_int4: unsupported dtype");
  I8_REQUIRE(n_expert >= 0 && n >= 0 && k >= 0 && k < (int64_t(1) << 31),
             "quantize_weights_int4: bad shape");
  I8_REQUIRE(k % 32 == 0, "quantize_weights_int4: K must be divisible by 32");
  I8_REQUIRE(group_size == 32 || group_size == 64 || group_size == 128,
             "quantize_weights_int4: group_size must be 32, 64 or 128");
  if (n_expert == 0 || n == 0 || k == 0) return I8MOE_OK;
  const int groups = static_cast<int>((k + group_size - 1) / group_size);
  const int g = static_cast<int>(group_size);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t rows = n_expert * n;
  const int ki = static_cast<int>(k);
  if (dtype == I8MOE_BF16)
    return launch_quantize<__nv_bfloat16>(w, rows, ki, g, groups, packed, scale, scale_dtype, st);
  if (dtype == I8MOE_FP16)
    return launch_quantize<__half>(w, rows, ki, g, groups, packed, scale, scale_dtype, st);
  return launch_quantize<float>(w, rows, ki, g, groups, packed, scale, scale_dtype, st);
}

int i8moe_int4_grouped_mv(const void* x, int64_t x_stride, int64_t x_rows, int dtype,
                          const int32_t* permuted_idx, int64_t topk, const uint8_t* w_packed,
                          const void* w_scale, int scale_dtype, int64_t group_size,
                          const int32_t* expert_offsets, int64_t n_expert, int64_t n_rows,
                          int64_t n, int64_t k, int silu, void* out, i8moe_stream_t stream) {
  I8_REQUIRE(dtype == I8MOE_BF16 || dtype == I8MOE_FP16,
             "int4_grouped_mv: x must be bfloat16 or float16");
  I8_REQUIRE(scale_dtype == dtype || scale_dtype == I8MOE_FP32,
             "int4_grouped_mv: w_scale must have x's dtype or float32");
  I8_REQUIRE(group_size == 32 || group_size == 64 || group_size == 128,
             "int4_grouped_mv: group_size must be 32, 64 or 128");
  I8_REQUIRE(k >= 32 && k % 32 == 0 && k < (int64_t(1) << 31) - 128,
             "int4_grouped_mv: K must be positive and divisible by 32");
  I8_REQUIRE(n >= 0 && n < (int64_t(1) << 31) - 128 && (!silu || n % 2 == 0),
             "int4_grouped_mv: bad N (even with silu)");
  I8_REQUIRE(n_expert >= 0 && n_expert <= 2048, "int4_grouped_mv: n_expert must be in [0, 2048]");
  I8_REQUIRE(n_rows >= 0 && n_rows < (int64_t(1) << 31) && x_rows >= 0,
             "int4_grouped_mv: bad n_rows");
  I8_REQUIRE(topk >= 1 && topk < (int64_t(1) << 31), "int4_grouped_mv: topk must be positive");
  I8_REQUIRE(permuted_idx != nullptr || x_rows >= n_rows,
             "int4_grouped_mv: x has fewer rows than the output");
  if (n_rows == 0 || n == 0 || n_expert == 0) return I8MOE_OK;
  I8_REQUIRE(x_stride >= k && x_stride % 8 == 0 && bits(x) % 16 == 0 && bits(w_packed) % 16 == 0,
             "int4_grouped_mv: x rows and w_packed must be 16-byte aligned");
  MvArgs a{x, x_stride, x_rows, permuted_idx, static_cast<int>(topk), w_packed, w_scale,
           scale_dtype, static_cast<int>(group_size),
           static_cast<int>((k + group_size - 1) / group_size), expert_offsets,
           static_cast<int>(n_expert), n_rows, static_cast<int>(n), static_cast<int>(k), out};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == I8MOE_BF16) return launch_mv<__nv_bfloat16>(a, silu != 0, st);
  return launch_mv<__half>(a, silu != 0, st);
}

}  // extern "C"
