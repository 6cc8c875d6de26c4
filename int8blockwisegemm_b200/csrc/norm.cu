// RMS norm with the residual's addition, an int8 output with a scale per
// token, and the gradients.  No reference counterpart: it is the step in
// front of the MoE layer, whose int8 output, sorted by expert, is what
// i8moe_int8_grouped_mm takes with a_row_scale.
//
//   h = x + residual                       (stored rounded to the row type)
//   rstd = 1 / sqrt(mean(h^2) + eps)       (from the unrounded fp32 sum h)
//   y = h * rstd * weight                  (rounded once)
//   scale = max(max|y|, 1e-10) / 127, q = rint(y / scale)   (from fp32 y)
//
// and, with n = h * rstd and a = dy * weight,
//   dx = dresidual = rstd * (a - n * mean(a * n)) + dh
//   dweight = sum over rows of dy * n.
// Everything between the loads and the stores is fp32.  The backward pass adds x
// and the residual again instead of reading the stored h: its rounding would be
// the larger half of dweight's error.
#include <algorithm>

#include "common.cuh"
#include "norm_index.cuh"

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
  float inv_k;  // 1 / k
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

template <typename T, int kVec>
__device__ __forceinline__ void load_weight(const void* w, int dtype, int i, float* out) {
  if constexpr (sizeof(T) < 4) {
    if (dtype != I8MOE_FP32) {
      struct alignas(sizeof(T) * kVec) Raw {
        T v[kVec];
      };
      const Raw raw = *reinterpret_cast<const Raw*>(static_cast<const T*>(w) + i);
#pragma unroll
      for (int e = 0; e < kVec; ++e) out[e] = Num<T>::to_f(raw.v[e]);
      return;
    }
  }
  if constexpr (kVec % 4 == 0) {
#pragma unroll
    for (int e = 0; e < kVec; e += 4) {
      const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + i + e);
      out[e] = f.x;
      out[e + 1] = f.y;
      out[e + 2] = f.z;
      out[e + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) out[e] = static_cast<const float*>(w)[i + e];
  }
}

// The same one by one, 0 outside of the row, of k >= 1 elements.
template <int kVec, typename W>
__device__ __forceinline__ void load_elements(const W* w, int i, int k, float* out) {
  if (i >= 0 && i + kVec <= k) {
    w += i;
#pragma unroll
    for (int e = 0; e < kVec; ++e) out[e] = Num<W>::to_f(w[e]);
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      out[e] = Num<W>::to_f(w[nearest_element(i + e, k)]);
      if (i + e < 0 || i + e >= k) out[e] = 0.f;
    }
  }
}
// The elements from i on, shift elements before a 16-byte boundary: cut out of
// the two packs that hold them (8192 x 1001: 21 instead of 25 us one by one).
template <typename T, int kVec>
__device__ __forceinline__ void load_weight_at(const void* w, int dtype, int i, int shift, int k,
                                               float* out) {
  if constexpr (sizeof(T) < 4) {
    if (dtype != I8MOE_FP32) {
      const T* p = static_cast<const T*>(w);
      const int up = i + shift;  // of the two packs that hold the elements, the second
      if (up + kVec > k || reinterpret_cast<uintptr_t>(w) % 16 != 0) {
        load_elements<kVec>(p, i, k, out);
        return;
      }
      const uint4 hi = *reinterpret_cast<const uint4*>(p + up);
      uint4 lo = make_uint4(0, 0, 0, 0);
      if (up > 0) lo = *reinterpret_cast<const uint4*>(p + up - kVec);
      uint32_t d[9] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w, 0};
      const int at = kVec - shift;  // the first element's place in both
#pragma unroll
      for (int step = 8; step >= 2; step /= 2)
#pragma unroll
        for (int j = 0; j < 9; ++j)
          if (at & step) d[j] = j + step / 2 < 9 ? d[j + step / 2] : 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t v = __funnelshift_r(d[j], d[j + 1], at & 1 ? 16 : 0);
        out[2 * j] = Num<T>::to_f(reinterpret_cast<const T*>(&v)[0]);
        out[2 * j + 1] = Num<T>::to_f(reinterpret_cast<const T*>(&v)[1]);
      }
      return;
    }
  }
  load_elements<kVec>(static_cast<const float*>(w), i, k, out);
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

// rint(y * inv) as int8, for |y * inv| <= 127 up to its last bits: adding 1.5 *
// 2^23 rounds to the nearest integer, ties to even, and leaves it in the low
// bits.
__device__ __forceinline__ int8_t to_int8(float y, float inv) {
  return static_cast<int8_t>(__float_as_uint(fmaf(y, inv, 12582912.f)));
}

// The largest |y| of a row, for its scale: NaN where the sum of squares is not
// finite (it may leave fp32 where no value does, and every y is 0 then).
__device__ __forceinline__ float largest_of(float largest, float sum) {
  const bool finite = sum < __int_as_float(0x7f800000);
  return finite ? max_nan(largest, 1e-10f) : __int_as_float(0x7fffffff);
}

// What the int8 values of a row are multiplied by: 127 over its largest |y|.
// Non-finite rows give 0 and a mask of zeros, which makes their values 0.
struct Int8Row {
  float inv;
  uint8_t mask;
};
__device__ __forceinline__ Int8Row int8_row(float largest) {
  const bool finite = largest < __int_as_float(0x7f800000);
  // scaled, because the fast division gives 0 for a divisor above 2^126
  return {finite ? __fdividef(127.f / 256, largest * (1.f / 256)) : 0.f, static_cast<uint8_t>(finite ? 0xff : 0)};
}

// kVec elements that one thread reads or writes at once.
template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Pack {
  T v[kVec];
};

// Zeros the elements outside of the row.
template <typename T, int kVec>
__device__ __forceinline__ void trim(Pack<T, kVec>& v, int i, int k) {
#pragma unroll
  for (int e = 0; e < kVec; ++e)
    if (i + e < 0 || i + e >= k) v.v[e] = Num<T>::from_f(0.f);
}

// row[i, i + kVec), of which only what lies in [0, k)
template <bool kShift, typename T, int kVec>
__device__ __forceinline__ void store_pack(T* row, int i, int k, const Pack<T, kVec>& v) {
  if (!kShift || (i >= 0 && i + kVec <= k)) {
    *reinterpret_cast<Pack<T, kVec>*>(row + i) = v;
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      if (i + e >= 0 && i + e < k) row[i + e] = v.v[e];
  }
}

// Rows in registers: blockDim.x threads hold a row, kPer packs each (a CTA has
// several rows where a row takes less than a warp), so that it is read once,
// and the sum of squares and the largest |h * weight| (from which the int8
// scale follows, rstd being one factor of the row) are reduced together.  kVec
// is 16 bytes' worth when width, strides and pointers allow it, with kShift or
// without, else 1.
// Bound by memory: 8192 x 2048 bf16 with a residual takes 24 us, 5.6 TB/s of
// the 6.6 that a copy has; two packs a thread take 1 us more, four 4, and CTAs
// that stay and load the next row ahead 4.
template <typename T, int kVec, int kPer, bool kShift, bool kQuant>
__global__ void __launch_bounds__(1024) norm_row_kernel(NormArgs a) {
  using P = Pack<T, kVec>;
  __shared__ float s_sum[32], s_max[32];
  const int64_t r = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int tid = threadIdx.x, stride = blockDim.x * kVec;
  const RowPart part = row_part<kVec, kShift>(r, a.rows, a.k, tid);
  const int k = part.k, first = part.first, shift = tid * kVec - first;
  const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
  const T* res = static_cast<const T*>(a.residual) + r * a.residual_stride;
  P xv[kPer], rv[kPer];
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int i = p * stride + first;
    if (i < k) {
      // what lies before a row, or behind one that is not the last, belongs to the tensor too
      if (!kShift || i + kVec <= k || r + 1 < a.rows) {
        xv[p] = *reinterpret_cast<const P*>(x + i);
        if (a.residual) rv[p] = *reinterpret_cast<const P*>(res + i);
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          if (i + e >= 0 && i + e < k) {
            xv[p].v[e] = x[i + e];
            if (a.residual) rv[p].v[e] = res[i + e];
          }
        }
      }
    }
  }
  float w[kPer][kVec];
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int i = p * stride + first;
    if (i < k) {
      if constexpr (kShift) load_weight_at<T, kVec>(a.weight, a.weight_dtype, i, shift, k, w[p]);
      else load_weight<T, kVec>(a.weight, a.weight_dtype, i, w[p]);
    }
  }
  float h[kPer][kVec];
  float ss = 0.f, m = 0.f;
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int i = p * stride + first;
    if (i < k) {
      if (kShift && (i < 0 || i + kVec > k)) {
        trim(xv[p], i, k);
        if (a.residual) trim(rv[p], i, k);
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        h[p][e] = Num<T>::to_f(xv[p].v[e]);
        if (a.residual) h[p][e] += Num<T>::to_f(rv[p].v[e]);
        ss = fmaf(h[p][e], h[p][e], ss);
        if constexpr (kQuant) m = max_nan(m, fabsf(h[p][e] * w[p][e]));
      }
      if (a.h) {
        P o;
#pragma unroll
        for (int e = 0; e < kVec; ++e) o.v[e] = Num<T>::from_f(h[p][e]);
        store_pack<kShift>(static_cast<T*>(a.h) + r * a.k, i, k, o);
      }
    }
  }
  for (int o = min(32, static_cast<int>(blockDim.x)) >> 1; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if constexpr (kQuant) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  if (blockDim.x > 32) {  // one row
    if ((tid & 31) == 0) {
      s_sum[tid >> 5] = ss;
      if constexpr (kQuant) s_max[tid >> 5] = m;
    }
    __syncthreads();
    const bool on = (tid & 31) < (blockDim.x >> 5);
    ss = on ? s_sum[tid & 31] : 0.f;
    if constexpr (kQuant) m = on ? s_max[tid & 31] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if constexpr (kQuant) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
  }
  const float rstd = rsqrtf(fmaf(ss, a.inv_k, a.eps));
  const float largest = largest_of(m * rstd, ss);
  const Int8Row row = int8_row(largest);
  if (tid == 0 && k > 0) {
    if (a.rstd) a.rstd[r] = rstd;
    if constexpr (kQuant) a.scale[r] = largest / 127.f;
  }
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int i = p * stride + first;
    if (i < k) {
      P o;
#pragma unroll
      for (int e = 0; e < kVec; ++e) h[p][e] = h[p][e] * rstd * w[p][e];
      if (!kQuant || a.y) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) o.v[e] = Num<T>::from_f(h[p][e]);
        store_pack<kShift>(static_cast<T*>(a.y) + r * a.k, i, k, o);
      }
      if constexpr (kQuant) {
        Pack<int8_t, kVec> q;
#pragma unroll
        for (int e = 0; e < kVec; ++e) q.v[e] = to_int8(h[p][e], row.inv) & row.mask;
        store_pack<kShift>(a.q + r * a.k, i, k, q);
      }
    }
  }
}

// Rows too wide for the registers of a CTA: read up to three times (sum of
// squares, absmax, output); the repeats hit L1/L2.
template <typename T>
__global__ void __launch_bounds__(256) norm_wide_kernel(NormArgs a) {
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
    const float rstd = rsqrtf(fmaf(ss, a.inv_k, a.eps));
    if (a.rstd && threadIdx.x == 0) a.rstd[r] = rstd;
    Int8Row row{};
    if (a.q) {
      float m = 0.f;
      for (int i = threadIdx.x; i < a.k; i += blockDim.x)
        m = max_nan(m, fabsf(h_at(i) * rstd * load_any(a.weight, a.weight_dtype, i)));
      const float largest = largest_of(block_reduce<MaxNan>(m, s_part), ss);
      row = int8_row(largest);
      if (threadIdx.x == 0) a.scale[r] = largest / 127.f;
    }
    for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
      const float h = h_at(i);
      const float y = h * rstd * load_any(a.weight, a.weight_dtype, i);
      if (a.h) static_cast<T*>(a.h)[r * a.k + i] = Num<T>::from_f(h);
      if (a.y) static_cast<T*>(a.y)[r * a.k + i] = Num<T>::from_f(y);
      if (a.q) a.q[r * a.k + i] = to_int8(y, row.inv) & row.mask;
    }
  }
}

struct NormGradArgs {
  const void* x;
  const void* residual;  // nullable
  const void* dy;
  const void* dh;  // nullable: the gradient of the residual stream
  const void* weight;
  int64_t x_stride, residual_stride, dy_stride, dh_stride;
  int weight_dtype;
  const float* rstd;
  int64_t rows;
  int k;
  float inv_k;  // 1 / k
  void* dx;
  float* part;  // [n_part, k], nullable: no weight gradient is wanted
  int n_part;
};

template <int kPer>
constexpr int kGradStages = kPer > 2 ? 1 : 2;  // rows of a group in shared memory
// Threads of a CTA whose groups have that many, and CTAs resident on an SM:
// 768 threads of 80 registers (1024 of 64 spilled: 52 instead of 36 us), for
// one group of 512 threads 1024, for more packs a thread 512, and for shifted
// rows, which take more registers, 512 (8192 x 1001: 28 instead of 38 us).
template <int kThreads>
constexpr int kGradThreads = kThreads > 256 ? kThreads : 256;
template <int kVec, int kPer, int kThreads, bool kShift>
constexpr int kGradCtas = kThreads <= 256 ? (kShift ? 2 : 3) : kPer <= (kVec == 1 ? 4 : 1) ? 2 : 1;
// The most CTAs of a backward pass, and partial sums of the weight's gradient
// that it writes (one row of k each) before they are added up.
constexpr int kNormParts = 444;

// The kThreads threads of a group hold a row's columns, kPer packs each, for
// all rows that the group takes, and add up their share of the weight's
// gradient in registers.  Rows come through a ring of kGradStages in shared
// memory, of which every thread reads what it copied itself, so that the next
// rows are on their way during a row's one reduction (one barrier of the
// group; the halves of s_part take turns) without holding registers: with the
// next row in registers instead, the default size took 48 us, spills and all;
// a third row in the ring costs 1 us.
// Single elements (kVec 1) do wait in registers, of which they take few.  A
// CTA's groups meet at its end.  The grid is what is resident at once; with
// kShift a multiple of 8, so that all rows of a CTA have the same shift.
template <typename T, int kVec, int kPer, int kThreads, bool kWeight, bool kShift>
__global__ void __launch_bounds__(kGradThreads<kThreads>, kGradCtas<kVec, kPer, kThreads, kShift>)
    norm_grad_row_kernel(NormGradArgs a) {
  using P = Pack<T, kVec>;
  constexpr int kCta = kGradThreads<kThreads>;
  constexpr bool kRing = kVec > 1;
  constexpr int kGroups = kCta / kThreads, kWarps = kThreads / 32;
  constexpr int kStages = kGradStages<kPer>;
  extern __shared__ uint4 s_ring[];  // [stage][x, dy, residual, dh][kPer][thread of the CTA]
  __shared__ float s_part[2][kCta / 32];
  const int group = threadIdx.x / kThreads, tid = threadIdx.x % kThreads;
  const int lane = tid & 31;
  const int64_t rows_at_once = static_cast<int64_t>(gridDim.x) * kGroups;
  int64_t r = static_cast<int64_t>(group) * gridDim.x + blockIdx.x;
  const int shift = kShift ? shift_of<kVec>(r, a.k) : 0, first = tid * kVec - shift;
  auto row_of = [&](int which, int64_t row) {
    return which == 0   ? static_cast<const T*>(a.x) + row * a.x_stride
           : which == 1 ? static_cast<const T*>(a.dy) + row * a.dy_stride
           : which == 2 ? static_cast<const T*>(a.residual) + row * a.residual_stride
                        : static_cast<const T*>(a.dh) + row * a.dh_stride;
  };
  auto there = [&](int which) {
    return which < 2 || (which == 2 ? a.residual : a.dh) != nullptr;
  };
  auto ring = [&](int stage, int which, int p) {
    return s_ring + ((stage * 4 + which) * kPer + p) * kCta + threadIdx.x;
  };
  auto copy = [&](int64_t row, int stage) {
    if (row < a.rows)
#pragma unroll
      for (int which = 0; which < 4; ++which)
        if (there(which))
#pragma unroll
          for (int p = 0; p < kPer; ++p) {
            const int i = p * (kThreads * kVec) + first;
            if (i < a.k)  // zeros behind the row; what lies before it belongs to the tensor too
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                               smem_u32(ring(stage, which, p))),
                           "l"(row_of(which, row) + i),
                           "r"(kShift ? min(kVec, a.k - i) * static_cast<int>(sizeof(T)) : 16)
                           : "memory");
          }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  P now[kRing ? 1 : 4][kPer] = {}, next[kRing ? 1 : 4][kPer] = {};
  auto load = [&](int64_t row) {
#pragma unroll
    for (int which = 0; which < 4; ++which)
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        const int i = p * (kThreads * kVec) + first;
        if (i < a.k && there(which))
          next[kRing ? 0 : which][p] = *reinterpret_cast<const P*>(row_of(which, row) + i);
      }
  };
  auto get = [&](int stage, int which, int p) {
    if constexpr (kRing) return *reinterpret_cast<const P*>(ring(stage, which, p));
    else return now[which][p];
  };

  if constexpr (kRing) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) copy(r + s * rows_at_once, s);
  } else if (r < a.rows) {
    load(r);
  }
  float w[kPer][kVec], dw[kPer][kVec];
#pragma unroll
  for (int p = 0; p < kPer; ++p) {
    const int i = p * (kThreads * kVec) + first;
    if (i < a.k) {
      if constexpr (kShift) load_weight_at<T, kVec>(a.weight, a.weight_dtype, i, shift, a.k, w[p]);
      else load_weight<T, kVec>(a.weight, a.weight_dtype, i, w[p]);
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) dw[p][e] = 0.f;
  }
  float rstd_next = r < a.rows ? a.rstd[r] : 0.f;
  for (int turn = 0, stage = 0; r < a.rows; turn ^= 1) {
    const float rstd = rstd_next;
    if (r + rows_at_once < a.rows) rstd_next = a.rstd[r + rows_at_once];
    if constexpr (kRing) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      if (kShift && first < 0) {
#pragma unroll
        for (int which = 0; which < 3; ++which)
          if (there(which)) trim(*reinterpret_cast<P*>(ring(stage, which, 0)), first, a.k);
      }
    } else {
#pragma unroll
      for (int which = 0; which < 4; ++which)
#pragma unroll
        for (int p = 0; p < kPer; ++p) now[which][p] = next[which][p];
      if (r + rows_at_once < a.rows) load(r + rows_at_once);
    }
    float dot = 0.f;  // of dy * weight and h
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int i = p * (kThreads * kVec) + first;
      if (i < a.k) {
        const P x = get(stage, 0, p), g = get(stage, 1, p);
        P res;
        if (a.residual) res = get(stage, 2, p);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          float hf = Num<T>::to_f(x.v[e]);
          if (a.residual) hf += Num<T>::to_f(res.v[e]);
          const float gf = Num<T>::to_f(g.v[e]);
          if constexpr (kWeight) dw[p][e] = fmaf(gf * rstd, hf, dw[p][e]);
          dot = fmaf(gf * w[p][e], hf, dot);
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if constexpr (kWarps > 1) {
      float* part = s_part[turn] + group * kWarps;
      if (lane == 0) part[tid >> 5] = dot;
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(kThreads) : "memory");
      dot = part[lane % kWarps];
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    }
    // dx = rstd * (a - n * mean(a * n)) with n = h * rstd
    const float back = -(rstd * rstd) * (rstd * (dot * a.inv_k));
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int i = p * (kThreads * kVec) + first;
      if (i < a.k) {
        const P x = get(stage, 0, p), g = get(stage, 1, p);
        P o, res, add;
        if (a.residual) res = get(stage, 2, p);
        if (a.dh) add = get(stage, 3, p);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          float d = Num<T>::to_f(x.v[e]);
          if (a.residual) d += Num<T>::to_f(res.v[e]);
          d *= back;
          d = fmaf(Num<T>::to_f(g.v[e]) * w[p][e], rstd, d);
          if (a.dh) d += Num<T>::to_f(add.v[e]);
          o.v[e] = Num<T>::from_f(d);
        }
        store_pack<kShift>(static_cast<T*>(a.dx) + r * a.k, i, a.k, o);
      }
    }
    if constexpr (kRing) {
      copy(r + kStages * rows_at_once, stage);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    r += rows_at_once;
  }
  if constexpr (kWeight) {
    float* s_dw = reinterpret_cast<float*>(s_ring);  // [group - 1][kPer * kVec][kThreads]
    if constexpr (kGroups > 1) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();
      if (group > 0)
#pragma unroll
        for (int p = 0; p < kPer; ++p)
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            s_dw[((group - 1) * kPer * kVec + p * kVec + e) * kThreads + tid] = dw[p][e];
      __syncthreads();
      if (group > 0) return;
    }
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int i = p * (kThreads * kVec) + first;
      if (i < a.k)
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          float v = dw[p][e];
          for (int o = 0; o < kGroups - 1; ++o)
            v += s_dw[(o * kPer * kVec + p * kVec + e) * kThreads + tid];
          if (!kShift || (i + e >= 0 && i + e < a.k))
            a.part[static_cast<int64_t>(blockIdx.x) * a.k + i + e] = v;
        }
    }
  }
}

// h of one row, element by element
template <typename T>
struct SumRow {
  const T* x;
  const T* residual;
  __device__ __forceinline__ SumRow(const NormGradArgs& a, int64_t r)
      : x(static_cast<const T*>(a.x) + r * a.x_stride),
        residual(a.residual ? static_cast<const T*>(a.residual) + r * a.residual_stride : nullptr) {}
  __device__ __forceinline__ float operator[](int i) const {
    const float v = Num<T>::to_f(x[i]);
    return residual ? v + Num<T>::to_f(residual[i]) : v;
  }
};

// Rows too wide for the registers of a CTA: read twice, and once more for the
// weight's gradient.
template <typename T>
__global__ void __launch_bounds__(256) norm_grad_wide_kernel(NormGradArgs a) {
  __shared__ float s_part[8];
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const SumRow<T> h(a, r);
    const T* dy = static_cast<const T*>(a.dy) + r * a.dy_stride;
    const T* dh = a.dh ? static_cast<const T*>(a.dh) + r * a.dh_stride : nullptr;
    const float rstd = a.rstd[r];
    float dot = 0.f;
    for (int i = threadIdx.x; i < a.k; i += blockDim.x)
      dot += Num<T>::to_f(dy[i]) * load_any(a.weight, a.weight_dtype, i) * (h[i] * rstd);
    const float mean = block_reduce<Sum>(dot, s_part) * a.inv_k;
    for (int i = threadIdx.x; i < a.k; i += blockDim.x) {
      const float g = Num<T>::to_f(dy[i]) * load_any(a.weight, a.weight_dtype, i);
      float d = rstd * (g - h[i] * rstd * mean);
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
             SumRow<T>(a, r)[i] * a.rstd[r], s);
  a.part[static_cast<int64_t>(blockIdx.y) * a.k + i] = s;
}

// Adds up the partial sums: 32 columns a CTA, its 32 warps a share of the parts
// each, in a fixed order.
__global__ void __launch_bounds__(1024) norm_weight_sum_kernel(const float* part, int n_part, int k,
                                                               void* dweight, int dtype) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (i < k)
    for (int p = warp; p < n_part; p += 32) v += part[static_cast<int64_t>(p) * k + i];
  s[warp][lane] = v;
  __syncthreads();
  v = s[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int c = blockIdx.x * 32 + warp;
  if (lane == 0 && c < k) store_any(dweight, dtype, c, v);
}

bool float_dtype(int d) { return d == I8MOE_BF16 || d == I8MOE_FP16 || d == I8MOE_FP32; }

uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Whether rows can be read by shifted packs: k and the strides leave the same
// remainder, and a row's ends lie inside the rows beside it.
template <int kVec>
bool same_shift(int k, int64_t stride) { return stride >= k && stride % kVec == k % kVec; }

template <typename T, int kVec, int kPer, bool kShift>
void launch_norm_row(const NormArgs& a, cudaStream_t st) {
  const auto [x, y] = row_block<kVec, kPer, kShift>(a.k);
  auto kernel = a.q ? norm_row_kernel<T, kVec, kPer, kShift, true>
                    : norm_row_kernel<T, kVec, kPer, kShift, false>;
  kernel<<<static_cast<unsigned>((a.rows + y - 1) / y), dim3(x, y), 0, st>>>(a);
}

// One pack a thread while that makes no CTA of more than 512 threads; elements
// one by one come eight to a thread (4096 x 2047 bf16: 33 us with four, 41
// with two).
template <typename T, int kVec, bool kShift>
bool launch_norm_rows(const NormArgs& a, cudaStream_t st) {
  const int k = covered<kVec, kShift>(a.k);
  if constexpr (kVec == 1) {
    if (k > 8 * 1024) return false;
    launch_norm_row<T, 1, 8, false>(a, st);
  } else if (k <= kVec * 512) {
    launch_norm_row<T, kVec, 1, kShift>(a, st);
  } else if (k <= kVec * 2 * 1024) {
    launch_norm_row<T, kVec, 2, kShift>(a, st);
  } else {
    return false;
  }
  return true;
}

template <typename T>
int launch_norm(const NormArgs& a, cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);
  const bool aligned = (bits(a.x) | bits(a.residual) | bits(a.h) | bits(a.y)) % 16 == 0 && bits(a.q) % 8 == 0;
  const bool packs = aligned && bits(a.weight) % 16 == 0 && a.k % kVec == 0 && a.x_stride % kVec == 0 &&
                     (!a.residual || a.residual_stride % kVec == 0);
  const bool shift = aligned && a.k >= kVec && same_shift<kVec>(a.k, a.x_stride) &&
                     (!a.residual || same_shift<kVec>(a.k, a.residual_stride));
  if (!(packs   ? launch_norm_rows<T, kVec, false>(a, st)
        : shift ? launch_norm_rows<T, kVec, true>(a, st)
                : launch_norm_rows<T, 1, false>(a, st))) {
    const int sms = num_sms(current_device());
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, sms * 8));
    norm_wide_kernel<T><<<grid, 256, 0, st>>>(a);
  }
  return check_launch("rms_norm");
}

template <typename T, int kVec, bool kShift, int kPer, int kThreads>
int launch_norm_grad_kernel(NormGradArgs& a, cudaStream_t st) {
  constexpr int kCta = kGradThreads<kThreads>, kGroups = kCta / kThreads;
  const int64_t most = int64_t(num_sms(current_device())) * kGradCtas<kVec, kPer, kThreads, kShift>;
  a.n_part = static_cast<int>(
      std::min({(a.rows + kGroups - 1) / kGroups, most, int64_t(kNormParts)}));
  if (kShift) a.n_part -= a.n_part % 8;
  constexpr int kRing = kVec > 1 ? kGradStages<kPer> * 4 * kPer * kCta * 16 : 0;
  constexpr int kMeet = (kGroups - 1) * kPer * kVec * kThreads * 4;
  constexpr int kSmem = kRing > kMeet ? kRing : kMeet;
  auto kernel = a.part ? norm_grad_row_kernel<T, kVec, kPer, kThreads, true, kShift>
                       : norm_grad_row_kernel<T, kVec, kPer, kThreads, false, kShift>;
  if (kSmem > 40 * 1024)  // with the static part, more than every kernel may have
    I8_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  kernel<<<a.n_part, kCta, kSmem, st>>>(a);
  return check_launch("rms_norm_backward");
}

// Widths that fit a CTA's registers; `*wide` says that this one does not.
template <typename T, int kVec, bool kShift>
int launch_norm_grad_rows(NormGradArgs& a, cudaStream_t st, bool* wide) {
  constexpr int kMost = kVec == 1 ? 8 : kVec == 4 ? 4 : 2;  // what the registers hold
  const int packs = (covered<kVec, kShift>(a.k) + kVec - 1) / kVec;
  if (packs <= 32) return launch_norm_grad_kernel<T, kVec, kShift, 1, 32>(a, st);
  if (packs <= 64) return launch_norm_grad_kernel<T, kVec, kShift, 1, 64>(a, st);
  if (packs <= 128) return launch_norm_grad_kernel<T, kVec, kShift, 1, 128>(a, st);
  if (packs <= 256) return launch_norm_grad_kernel<T, kVec, kShift, 1, 256>(a, st);
  if (packs <= 512) return launch_norm_grad_kernel<T, kVec, kShift, 1, 512>(a, st);
  if (packs <= 1024) return launch_norm_grad_kernel<T, kVec, kShift, 2, 512>(a, st);
  if (packs <= 512 * kMost) return launch_norm_grad_kernel<T, kVec, kShift, kMost, 512>(a, st);
  *wide = true;
  return I8MOE_OK;
}

template <typename T>
int launch_norm_grad(NormGradArgs& a, cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);
  const bool aligned =
      (bits(a.x) | bits(a.residual) | bits(a.dy) | bits(a.dh) | bits(a.dx)) % 16 == 0;
  const bool packs = aligned && bits(a.weight) % 16 == 0 && a.k % kVec == 0 &&
                     a.x_stride % kVec == 0 && a.dy_stride % kVec == 0 &&
                     (!a.residual || a.residual_stride % kVec == 0) &&
                     (!a.dh || a.dh_stride % kVec == 0);
  // 64 rows: eight CTAs, each with a row for the most groups that it may have
  const bool shift = aligned && a.rows >= 64 && a.k >= kVec && same_shift<kVec>(a.k, a.x_stride) &&
                     same_shift<kVec>(a.k, a.dy_stride) &&
                     (!a.residual || same_shift<kVec>(a.k, a.residual_stride)) &&
                     (!a.dh || same_shift<kVec>(a.k, a.dh_stride));
  bool wide = false;
  const int rc = packs   ? launch_norm_grad_rows<T, kVec, false>(a, st, &wide)
                 : shift ? launch_norm_grad_rows<T, kVec, true>(a, st, &wide)
                         : launch_norm_grad_rows<T, 1, false>(a, st, &wide);
  if (!wide) return rc;
  a.n_part = static_cast<int>(std::min<int64_t>(a.rows, kNormParts));
  norm_grad_wide_kernel<T><<<a.n_part, 256, 0, st>>>(a);
  if (a.part) norm_weight_part_kernel<T><<<dim3((a.k + 255) / 256, a.n_part), 256, 0, st>>>(a);
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
  I8_REQUIRE(n_rows >= 0 && n_rows < (int64_t(1) << 31) && n_hidden >= 1 &&
                 n_hidden < (int64_t(1) << 31) - 1024,
             "rms_norm: bad n_rows / n_hidden");
  I8_REQUIRE(eps >= 0.f && eps < 3.0e38f, "rms_norm: eps must be finite and not negative");
  if (n_rows == 0) return I8MOE_OK;
  I8_REQUIRE((residual == nullptr) == (residual_out == nullptr),
             "rms_norm: residual and residual_out go together");
  I8_REQUIRE((q == nullptr) == (q_scale == nullptr), "rms_norm: q and q_scale go together");
  I8_REQUIRE(y != nullptr || q != nullptr, "rms_norm: no output given");
  I8_REQUIRE(x != nullptr && weight != nullptr, "rms_norm: x and weight must be given");
  NormArgs a{x, residual, weight, x_stride, residual_stride, weight_dtype, n_rows,
             static_cast<int>(n_hidden), 1.f / static_cast<float>(n_hidden), eps, residual_out, y,
             rstd, q, q_scale};
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
                            int64_t residual_grad_stride, const void* x, int64_t x_stride,
                            const void* residual, int64_t residual_stride, int dtype,
                            const void* weight, int weight_dtype, const float* rstd,
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
  I8_REQUIRE(dy && x && weight && rstd && dx,
             "rms_norm_backward: dy, x, weight, rstd and dx must be given");
  NormGradArgs a{x, residual, dy, residual_grad, weight, x_stride, residual_stride, dy_stride,
                 residual_grad_stride, weight_dtype, rstd, n_rows, static_cast<int>(n_hidden),
                 1.f / static_cast<float>(n_hidden), dx, nullptr, 0};
  if (dweight) {
    I8_REQUIRE(workspace != nullptr && workspace_bytes >= i8moe_rms_norm_backward_workspace_size(
                                                              n_rows, n_hidden),
               "rms_norm_backward: the workspace is too small");
    a.part = static_cast<float*>(workspace);
  }
  int rc;
  if (dtype == I8MOE_BF16) rc = launch_norm_grad<__nv_bfloat16>(a, st);
  else if (dtype == I8MOE_FP16) rc = launch_norm_grad<__half>(a, st);
  else rc = launch_norm_grad<float>(a, st);
  if (rc != I8MOE_OK || !dweight) return rc;
  norm_weight_sum_kernel<<<(a.k + 31) / 32, 1024, 0, st>>>(a.part, a.n_part, a.k, dweight,
                                                           weight_dtype);
  return check_launch("rms_norm_backward: weight");
}

}  // extern "C"
