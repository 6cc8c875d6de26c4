// RMS norm with the residual's addition, an int8 output with a scale per
// token, and the gradients.  No reference counterpart: it is the step in
// front of the MoE layer, whose int8 output is what i8moe_int8_grouped_mm
// takes with a_row_scale.
//
//   h = x + residual                       (stored rounded to the row type)
//   rstd = 1 / sqrt(mean(h^2) + eps)       (from the unrounded fp32 sum h)
//   y = h * rstd * weight                  (rounded once)
//   scale = max(max|y|, 1e-10) / 127, q = rint(y / scale)   (from fp32 y)
//
// and, with n = h * rstd and a = dy * weight,
//   dx = dresidual = rstd * (a - n * mean(a * n)) + dh
//   dweight = sum over rows of dy * n.
// Everything between the loads and the stores is fp32.
#include <algorithm>

#include "common.cuh"

namespace i8moe {
namespace {

struct NormArgs {
  const void* x;
  const void* residual;  // nullable
  const void* weight;
  int64_t x_stride, residual_stride;  // elements
  int weight_dtype;
  int64_t rows;
  int k;
  float eps;
  void* h;      // nullable
  void* y;      // nullable
  float* rstd;  // nullable
  int8_t* q;    // nullable
  float* scale;
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == I8MOE_BF16) return Num<__nv_bfloat16>::to_f(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == I8MOE_FP16) return Num<__half>::to_f(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}

__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == I8MOE_BF16) static_cast<__nv_bfloat16*>(p)[i] = Num<__nv_bfloat16>::from_f(v);
  else if (dtype == I8MOE_FP16) static_cast<__half*>(p)[i] = Num<__half>::from_f(v);
  else static_cast<float*>(p)[i] = v;
}

// max that keeps NaN, so that a row without a finite norm gets a NaN scale
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Sum {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct MaxNan {
  static __device__ __forceinline__ float of(float a, float b) { return max_nan(a, b); }
};

// Reduction over a CTA of whole warps; every thread gets the result.
template <typename Op>
__device__ __forceinline__ float block_reduce(float v, float* s_part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = Op::of(v, __shfl_xor_sync(0xffffffffu, v, o));
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  __syncthreads();  // s_part may still be read by the reduction before
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s_part[0];
  for (int w = 1; w < warps; ++w) v = Op::of(v, s_part[w]);
  return v;
}

__device__ __forceinline__ int8_t to_int8(float y, float scale) {
  // |y / scale| <= 127 but for its last bit, which rint takes back to 127; a
  // NaN becomes 0 (the row's scale is NaN too)
  return static_cast<int8_t>(__float2int_rn(__fdiv_rn(y, scale)));
}

// Rows of any width and alignment: one CTA per row, which it reads up to
// three times (sum of squares, absmax, output); the repeats hit L1/L2.
template <typename T>
__global__ void __launch_bounds__(256) norm_any_kernel(NormArgs a) {
  __shared__ float s_part[8];
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
    const T* res =
        a.residual ? static_cast<const T*>(a.residual) + r * a.residual_stride : nullptr;
    auto h_at = [&](int i) {
      const float v = Num<T>::to_f(x[i]);
      return res ? v + Num<T>::to_f(res[i]) : v;
    };
    float ss = 0.f;
    for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
      const float h = h_at(i);
      ss = fmaf(h, h, ss);
    }
    ss = block_reduce<Sum>(ss, s_part);
    const float rstd = __frsqrt_rn(ss / static_cast<float>(a.k) + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[r] = rstd;
    float scale = 0.f;
    if (a.q) {
      float m = 0.f;
      for (int i = threadIdx.x; i < a.k; i += blockDim.x)
        m = max_nan(m, fabsf(h_at(i) * rstd * load_any(a.weight, a.weight_dtype, i)));
      scale = max_nan(block_reduce<MaxNan>(m, s_part), 1e-10f) / 127.f;
      if (threadIdx.x == 0) a.scale[r] = scale;
    }
    for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
      const float h = h_at(i);
      const float y = h * rstd * load_any(a.weight, a.weight_dtype, i);
      if (a.h) static_cast<T*>(a.h)[r * a.k + i] = Num<T>::from_f(h);
      if (a.y) static_cast<T*>(a.y)[r * a.k + i] = Num<T>::from_f(y);
      if (a.q) a.q[r * a.k + i] = to_int8(y, scale);
    }
  }
}

struct NormGradArgs {
  const void* dy;  // nullable
  const void* dh;  // nullable
  const void* h;
  const void* weight;
  int64_t dy_stride, dh_stride, h_stride;
  int weight_dtype;
  const float* rstd;
  int64_t rows;
  int k;
  void* dx;
  float* part;  // [n_part, k], nullable: no weight gradient is wanted
  int n_part;
};

// Partial sums of the weight's gradient that a backward pass writes (one row
// of k each) before they are added up in a fixed order.
constexpr int kNormParts = 296;

template <typename T>
__global__ void __launch_bounds__(256) norm_grad_any_kernel(NormGradArgs a) {
  __shared__ float s_part[8];
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* h = static_cast<const T*>(a.h) + r * a.h_stride;
    const T* dy = static_cast<const T*>(a.dy) + r * a.dy_stride;
    const T* dh = a.dh ? static_cast<const T*>(a.dh) + r * a.dh_stride : nullptr;
    const float rstd = a.rstd[r];
    float dot = 0.f;
    for (int i = threadIdx.x; i < a.k; i += blockDim.x)
      dot += Num<T>::to_f(dy[i]) * load_any(a.weight, a.weight_dtype, i) *
             (Num<T>::to_f(h[i]) * rstd);
    const float mean = block_reduce<Sum>(dot, s_part) / static_cast<float>(a.k);
    for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
      const float n = Num<T>::to_f(h[i]) * rstd;
      const float g = Num<T>::to_f(dy[i]) * load_any(a.weight, a.weight_dtype, i);
      float d = rstd * (g - n * mean);
      if (dh) d += Num<T>::to_f(dh[i]);
      static_cast<T*>(a.dx)[r * a.k + i] = Num<T>::from_f(d);
    }
  }
}

// part[p, i] = sum of dy * n over the rows p, p + n_part, ...
template <typename T>
__global__ void __launch_bounds__(256) norm_weight_part_kernel(NormGradArgs a) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.k) return;
  float s = 0.f;
  for (int64_t r = blockIdx.y; r < a.rows; r += a.n_part)
    s = fmaf(Num<T>::to_f(static_cast<const T*>(a.dy)[r * a.dy_stride + i]),
             Num<T>::to_f(static_cast<const T*>(a.h)[r * a.h_stride + i]) * a.rstd[r], s);
  a.part[static_cast<int64_t>(blockIdx.y) * a.k + i] = s;
}

__global__ void __launch_bounds__(256) norm_weight_sum_kernel(const float* part, int n_part, int k,
                                                              void* dweight, int dtype) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= k) return;
  float s = 0.f;
  for (int p = 0; p < n_part; ++p) s += part[static_cast<int64_t>(p) * k + i];
  store_any(dweight, dtype, i, s);
}

bool float_dtype(int d) { return d == I8MOE_BF16 || d == I8MOE_FP16 || d == I8MOE_FP32; }

template <typename T>
int launch_norm(const NormArgs& a, cudaStream_t st) {
  const int sms = num_sms(current_device());
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, sms * 8));
  norm_any_kernel<T><<<grid, 256, 0, st>>>(a);
  return check_launch("rms_norm");
}

template <typename T>
int launch_norm_grad(const NormGradArgs& a, cudaStream_t st) {
  const int sms = num_sms(current_device());
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, sms * 8));
  norm_grad_any_kernel<T><<<grid, 256, 0, st>>>(a);
  if (a.part)
    norm_weight_part_kernel<T><<<dim3((a.k + 255) / 256, a.n_part), 256, 0, st>>>(a);
  return check_launch("rms_norm_backward");
}

}  // namespace
}  // namespace i8moe

using namespace i8moe;

extern "C" {

int i8moe_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                   int dtype, const void* weight, int weight_dtype, int64_t n_rows,
                   int64_t n_hidden, float eps, void* residual_out, void* y, float* rstd,
                   int8_t* q, float* q_scale, i8moe_stream_t stream) {
  I8_REQUIRE(float_dtype(dtype), "rms_norm: unsupported dtype");
  I8_REQUIRE(weight_dtype == dtype || weight_dtype == I8MOE_FP32,
             "rms_norm: weight must have the rows' dtype or float32");
  I8_REQUIRE(n_rows >= 0 && n_hidden >= 1 && n_hidden < (int64_t(1) << 31) - 1024,
             "rms_norm: bad n_rows / n_hidden");
  I8_REQUIRE(eps >= 0.f && eps < 3.0e38f, "rms_norm: eps must be finite and not negative");
  if (n_rows == 0) return I8MOE_OK;
  I8_REQUIRE((residual == nullptr) == (residual_out == nullptr),
             "rms_norm: residual and residual_out go together");
  I8_REQUIRE((q == nullptr) == (q_scale == nullptr), "rms_norm: q and q_scale go together");
  I8_REQUIRE(y != nullptr || q != nullptr, "rms_norm: no output given");
  I8_REQUIRE(x != nullptr && weight != nullptr, "rms_norm: x and weight must be given");
  NormArgs a{x, residual, weight, x_stride, residual_stride, weight_dtype, n_rows,
             static_cast<int>(n_hidden), eps, residual_out, y, rstd, q, q_scale};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == I8MOE_BF16) return launch_norm<__nv_bfloat16>(a, st);
  if (dtype == I8MOE_FP16) return launch_norm<__half>(a, st);
  return launch_norm<float>(a, st);
}

size_t i8moe_rms_norm_backward_workspace_size(int64_t n_rows, int64_t n_hidden) {
  if (n_rows < 1 || n_hidden < 1) return 0;
  return static_cast<size_t>(std::min<int64_t>(n_rows, kNormParts)) *
         static_cast<size_t>(n_hidden) * sizeof(float);
}

int i8moe_rms_norm_backward(const void* dy, int64_t dy_stride, const void* residual_grad,
                            int64_t residual_grad_stride, const void* h, int64_t h_stride,
                            int dtype, const void* weight, int weight_dtype, const float* rstd,
                            int64_t n_rows, int64_t n_hidden, void* dx, void* dweight,
                            void* workspace, size_t workspace_bytes, i8moe_stream_t stream) {
  I8_REQUIRE(float_dtype(dtype), "rms_norm_backward: unsupported dtype");
  I8_REQUIRE(weight_dtype == dtype || weight_dtype == I8MOE_FP32,
             "rms_norm_backward: weight must have the rows' dtype or float32");
  I8_REQUIRE(n_rows >= 0 && n_hidden >= 1 && n_hidden < (int64_t(1) << 31) - 1024,
             "rms_norm_backward: bad n_rows / n_hidden");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n_rows == 0) {
    if (dweight)
      I8_CUDA(cudaMemsetAsync(dweight, 0, n_hidden * (weight_dtype == I8MOE_FP32 ? 4 : 2), st));
    return I8MOE_OK;
  }
  I8_REQUIRE(dy && h && weight && rstd && dx,
             "rms_norm_backward: dy, h, weight, rstd and dx must be given");
  NormGradArgs a{dy, residual_grad, h, weight, dy_stride, residual_grad_stride, h_stride,
                 weight_dtype, rstd, n_rows, static_cast<int>(n_hidden), dx, nullptr, 0};
  if (dweight) {
    I8_REQUIRE(workspace != nullptr && workspace_bytes >= i8moe_rms_norm_backward_workspace_size(
                                                              n_rows, n_hidden),
               "rms_norm_backward: the workspace is too small");
    a.part = static_cast<float*>(workspace);
    a.n_part = static_cast<int>(std::min<int64_t>(n_rows, kNormParts));
  }
  int rc;
  if (dtype == I8MOE_BF16) rc = launch_norm_grad<__nv_bfloat16>(a, st);
  else if (dtype == I8MOE_FP16) rc = launch_norm_grad<__half>(a, st);
  else rc = launch_norm_grad<float>(a, st);
  if (rc != I8MOE_OK || !dweight) return rc;
  norm_weight_sum_kernel<<<(a.k + 255) / 256, 256, 0, st>>>(a.part, a.n_part, a.k, dweight,
                                                            weight_dtype);
  return check_launch("rms_norm_backward: weight");
}

}  // extern "C"
