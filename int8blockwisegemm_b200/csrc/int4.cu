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

// ---------------------------------------------------------------------------
// The products on the tensor cores
// ---------------------------------------------------------------------------
// Weights are the m16 operand of mma.m16n8k16 and a chunk of an expert's rows
// (8 per n8 tile) the other one, so that each weight is read and unpacked once
// for all rows of the chunk.  A nibble u becomes the 16-bit float base + u by
// one AND-OR and u - 8 by one subtraction, both exact; products with x are
// exact in the fp32 accumulators, which are scaled per group, so that no
// weight is rounded.
//
// A sum over k may take the k's in any order, so each lane loads what lies
// together: lane (g, q) = (lane / 4, lane % 4) takes rows g and g + 8 of a tile
// and, of every group of G columns, the G / 4 columns from q * G / 4 on.  A
// word's nibbles j and j + 4 are the pair that one AND leaves in a register,
// and x is paired the same way.
template <typename T>
struct Mma;

template <>
struct Mma<__nv_bfloat16> {
  static constexpr uint32_t kBase = 0x43004300u;  // 128 + u: 7 bits of fraction hold u
  static __device__ __forceinline__ uint32_t minus(uint32_t v) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                     __nv_bfloat162{__ushort_as_bfloat16(0x4308),
                                                    __ushort_as_bfloat16(0x4308)});  // 136
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

template <>
struct Mma<__half> {
  static constexpr uint32_t kBase = 0x64006400u;  // 1024 + u
  static __device__ __forceinline__ uint32_t minus(uint32_t v) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v),
                              __half2{__ushort_as_half(0x6408), __ushort_as_half(0x6408)});  // 1032
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// Weights are read once: they pass by L1, which holds the rows of x.
template <int kWords>
__device__ __forceinline__ void load_words(const uint32_t* p, uint32_t* w) {
  if constexpr (kWords == 4)
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
        : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  else if constexpr (kWords == 2)
    asm("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  else
    asm("ld.global.nc.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
}

constexpr int kMvThreads = 256;
constexpr int kMvWarps = kMvThreads / 32;
constexpr int kMvTiles = 4;       // m16 tiles of a warp
constexpr int kMvStep = 128;      // columns of a step
constexpr int kMvMaxExperts = 2048;

// One CTA takes a contiguous range of units, a unit being a chunk of 8 * kNt
// rows of an expert times a block of output columns; its 8 warps are 1, 2, 4
// or 8 shares of K times the rest in column blocks, and the shares' sums meet
// in shared memory.  Loads of a tile's next words are issued as soon as its
// present ones are unpacked, across units too.
template <typename T, int G, int kNt, bool kSilu>
__global__ void __launch_bounds__(kMvThreads, 2) mv_mma_kernel(MvArgs a, int k_shares) {
  constexpr int kGroups = kMvStep / G;  // groups of a step
  constexpr int kWords = G / 32;        // words of a lane in a group's row
  constexpr int kChunk = 8 * kNt;
  constexpr int kCols = kSilu ? kMvTiles * 8 : kMvTiles * 16;  // output columns of a warp
  __shared__ int s_first[kMvMaxExperts + 1];  // an expert's first chunk
  __shared__ int s_warp[kMvWarps];
  extern __shared__ float4 s_sum[];  // [2][warp][tile][kNt][lane]

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, q = lane & 3;

  // every expert's number of chunks, and their running sum
  {
    const int per = (a.n_expert + kMvThreads - 1) / kMvThreads;
    const int e0 = tid * per;
    int own = 0;
    for (int e = e0; e < min(a.n_expert, e0 + per); ++e) {
      int64_t r0, r1;
      expert_rows(a, e, &r0, &r1);
      const int n = static_cast<int>((r1 - r0 + kChunk - 1) / kChunk);
      s_first[e + 1] = n;
      own += n;
    }
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) s_warp[warp] = sum;
    __syncthreads();
    int at = sum - own;
    for (int w = 0; w < warp; ++w) at += s_warp[w];
    for (int e = e0; e < min(a.n_expert, e0 + per); ++e) {
      at += s_first[e + 1];
      s_first[e + 1] = at;
    }
    if (tid == 0) s_first[0] = 0;
    __syncthreads();
  }

  const int n_out = kSilu ? a.n / 2 : a.n;
  const int col_shares = kMvWarps / k_shares;
  const int ks = warp % k_shares, cs = warp / k_shares;
  const int blocks = (n_out + kCols * col_shares - 1) / (kCols * col_shares);
  const int64_t total = static_cast<int64_t>(s_first[a.n_expert]) * blocks;
  const int64_t u0 = total * blockIdx.x / gridDim.x, u1 = total * (blockIdx.x + 1) / gridDim.x;
  if (u0 == u1) return;
  const int steps = (a.k + kMvStep - 1) / kMvStep;
  const int st0 = steps * ks / k_shares, st1 = steps * (ks + 1) / k_shares;
  const int row_words = a.k / 8;

  // where a unit's rows and weights lie
  struct Unit {
    int chunk, block, expert;
    int64_t row0;
    int rows;
  };
  auto find = [&](int64_t u, const Unit& before) {
    Unit n;
    n.chunk = static_cast<int>(u / blocks);
    n.block = static_cast<int>(u - static_cast<int64_t>(n.chunk) * blocks);
    if (n.chunk == before.chunk) {
      n.expert = before.expert;
      n.row0 = before.row0;
      n.rows = before.rows;
      return n;
    }
    int lo = 0, hi = a.n_expert;  // the expert with s_first[lo] <= chunk < s_first[lo + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_first[mid] <= n.chunk) lo = mid;
      else hi = mid;
    }
    n.expert = lo;
    n.row0 = __ldg(a.eo + lo) + static_cast<int64_t>(n.chunk - s_first[lo]) * kChunk;
    n.rows = static_cast<int>(min(static_cast<int64_t>(kChunk), __ldg(a.eo + lo + 1) - n.row0));
    return n;
  };
  const T* x_row[kNt];
  auto find_rows = [&](const Unit& n) {
#pragma unroll
    for (int t = 0; t < kNt; ++t) {
      x_row[t] = nullptr;
      if (t * 8 + g < n.rows) {
        const int64_t src = source_row(a, n.row0 + t * 8 + g);
        if (src >= 0) x_row[t] = static_cast<const T*>(a.x) + src * a.x_stride;
      }
    }
  };

  uint32_t w[kMvTiles][2][4];  // [tile][row g / g + 8][word]
  float s[kMvTiles][2][kGroups];
  auto weight_row = [&](const Unit& n, int tile, int half) {
    int row = (n.block * col_shares + cs) * kCols + (kSilu ? tile >> 1 : tile) * 16 + half * 8 + g;
    row = min(row, n_out - 1);  // columns past the end are computed and not stored
    return kSilu && (tile & 1) ? row + n_out : row;
  };
  auto load_tile = [&](const Unit& n, int step, int tile) {
    const uint32_t* base =
        reinterpret_cast<const uint32_t*>(a.w) + static_cast<int64_t>(n.expert) * a.n * row_words;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t* row = base + static_cast<int64_t>(weight_row(n, tile, half)) * row_words;
#pragma unroll
      for (int gi = 0; gi < kGroups; ++gi) {
        const int word = step * (kMvStep / 8) + gi * (G / 8) + q * kWords;
        if (word < row_words) {
          load_words<kWords>(row + word, &w[tile][half][gi * kWords]);
        } else {
#pragma unroll
          for (int i = 0; i < kWords; ++i) w[tile][half][gi * kWords + i] = 0x88888888u;
        }
      }
    }
  };
  auto load_scale = [&](const Unit& n, int step, int tile) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int64_t row = static_cast<int64_t>(n.expert) * a.n + weight_row(n, tile, half);
#pragma unroll
      for (int gi = 0; gi < kGroups; ++gi) {
        const int64_t at = row * a.groups + min(step * kGroups + gi, a.groups - 1);
        s[tile][half][gi] = a.scale_dtype == I8MOE_FP32
                                ? __ldg(static_cast<const float*>(a.scale) + at)
                                : Num<T>::to_f(__ldg(static_cast<const T*>(a.scale) + at));
      }
    }
  };
  uint4 xr[kNt][4];  // [word] eight values of x each
  auto load_x = [&](int step) {
#pragma unroll
    for (int t = 0; t < kNt; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int word =
            step * (kMvStep / 8) + (i / kWords) * (G / 8) + q * kWords + i % kWords;
        xr[t][i] = x_row[t] != nullptr && word < row_words
                       ? __ldg(reinterpret_cast<const uint4*>(x_row[t]) + word)
                       : make_uint4(0, 0, 0, 0);
      }
  };

  Unit cur{-1, 0, 0, 0, 0};
  cur = find(u0, cur);
  find_rows(cur);
#pragma unroll
  for (int i = 0; i < kMvTiles; ++i) {
    load_tile(cur, st0, i);
    load_scale(cur, st0, i);
  }
  load_x(st0);

  for (int64_t u = u0; u < u1; ++u) {
    float acc[kMvTiles][kNt][4];
#pragma unroll
    for (int i = 0; i < kMvTiles; ++i)
#pragma unroll
      for (int t = 0; t < kNt; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][t][c] = 0.f;
    const Unit next = u + 1 < u1 ? find(u + 1, cur) : cur;
    for (int step = st0; step < st1; ++step) {
      // x in the weights' pairing: b[word][j] = (x[j], x[j + 4])
      uint32_t b[kNt][4][4];
#pragma unroll
      for (int t = 0; t < kNt; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          b[t][i][0] = __byte_perm(xr[t][i].x, xr[t][i].z, 0x5410);
          b[t][i][1] = __byte_perm(xr[t][i].x, xr[t][i].z, 0x7632);
          b[t][i][2] = __byte_perm(xr[t][i].y, xr[t][i].w, 0x5410);
          b[t][i][3] = __byte_perm(xr[t][i].y, xr[t][i].w, 0x7632);
        }
      const bool last = step + 1 == st1;
      const Unit& n = last ? next : cur;
      const int n_step = last ? st0 : step + 1;
      const bool more = !last || u + 1 < u1;
      if (more) {
        if (last && next.chunk != cur.chunk) find_rows(next);
        load_x(n_step);
      }
#pragma unroll
      for (int i = 0; i < kMvTiles; ++i) {
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) {
          float part[kNt][4];
#pragma unroll
          for (int t = 0; t < kNt; ++t)
#pragma unroll
            for (int c = 0; c < 4; ++c) part[t][c] = 0.f;
#pragma unroll
          for (int j = 0; j < kWords; ++j) {
            const int wi = gi * kWords + j;
            uint32_t f[2][4];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int p = 0; p < 4; ++p)
                f[half][p] =
                    Mma<T>::minus(((w[i][half][wi] >> (4 * p)) & 0x000f000fu) | Mma<T>::kBase);
#pragma unroll
            for (int t = 0; t < kNt; ++t) {
              Mma<T>::mma(part[t], f[0][0], f[1][0], f[0][1], f[1][1], b[t][wi][0], b[t][wi][1]);
              Mma<T>::mma(part[t], f[0][2], f[1][2], f[0][3], f[1][3], b[t][wi][2], b[t][wi][3]);
            }
          }
#pragma unroll
          for (int t = 0; t < kNt; ++t)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              acc[i][t][c] = fmaf(part[t][c], s[i][c >> 1][gi], acc[i][t][c]);
        }
        if (more) {
          load_tile(n, n_step, i);
          load_scale(n, n_step, i);
        }
      }
    }

    // the shares of K meet; the two halves of s_sum take turns, so that one
    // barrier a unit is enough
    float4* sum = s_sum + ((u - u0) & 1) * (kMvWarps * kMvTiles * kNt * 32);
#pragma unroll
    for (int i = 0; i < kMvTiles; ++i)
#pragma unroll
      for (int t = 0; t < kNt; ++t)
        sum[((warp * kMvTiles + i) * kNt + t) * 32 + lane] =
            make_float4(acc[i][t][0], acc[i][t][1], acc[i][t][2], acc[i][t][3]);
    __syncthreads();
    constexpr int kItems = kMvTiles * kNt / (kSilu ? 2 : 1);  // of a column share
    for (int item = warp; item < col_shares * kItems; item += kMvWarps) {
      const int c = item / kItems, t = item % kNt;
      const int i = item % kItems / kNt;  // tile, or pair of a gate's and a factor's
      float v[kSilu ? 2 : 1][4];
#pragma unroll
      for (int h = 0; h < (kSilu ? 2 : 1); ++h) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[h][j] = 0.f;
        for (int k = 0; k < k_shares; ++k) {
          const float4 p = sum[(((c * k_shares + k) * kMvTiles + (kSilu ? 2 * i + h : i)) * kNt +
                                t) * 32 + lane];
          v[h][0] += p.x;
          v[h][1] += p.y;
          v[h][2] += p.z;
          v[h][3] += p.w;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = t * 8 + 2 * q + (j & 1);
        const int col = (cur.block * col_shares + c) * kCols + i * 16 + g + 8 * (j >> 1);
        if (row < cur.rows && col < n_out)
          static_cast<T*>(a.out)[(cur.row0 + row) * n_out + col] =
              Num<T>::from_f(kSilu ? silu_mul(v[0][j], v[kSilu ? 1 : 0][j]) : v[0][j]);
      }
    }
    cur = next;
  }
}

template <typename T, int G, int kNt, bool kSilu>
int launch_mv_kernel(const MvArgs& a, cudaStream_t st) {
  const int steps = (a.k + kMvStep - 1) / kMvStep;
  int k_shares = 1;
  while (k_shares < kMvWarps && 2 * k_shares <= steps) k_shares *= 2;
  constexpr int kSmem = 2 * kMvWarps * kMvTiles * kNt * 32 * static_cast<int>(sizeof(float4));
  auto kernel = mv_mma_kernel<T, G, kNt, kSilu>;
  I8_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  const int64_t cols = (kSilu ? kMvTiles * 8 : kMvTiles * 16) * (kMvWarps / k_shares);
  const int64_t units =
      (((kSilu ? a.n / 2 : a.n) + cols - 1) / cols) *
      std::min<int64_t>(a.rows, (a.rows + 8 * kNt - 1) / (8 * kNt) + a.n_expert);
  const unsigned grid =
      static_cast<unsigned>(std::min<int64_t>(units, int64_t(num_sms(current_device())) * 2));
  kernel<<<grid, kMvThreads, kSmem, st>>>(a, k_shares);
  return check_launch("int4_grouped_mv");
}

template <typename T, int kNt, bool kSilu>
int launch_mv_group(const MvArgs& a, cudaStream_t st) {
  if (a.group == 128) return launch_mv_kernel<T, 128, kNt, kSilu>(a, st);
  if (a.group == 64) return launch_mv_kernel<T, 64, kNt, kSilu>(a, st);
  return launch_mv_kernel<T, 32, kNt, kSilu>(a, st);
}

template <typename T>
int launch_mv(const MvArgs& a, bool silu, cudaStream_t st) {
  return silu ? launch_mv_group<T, 1, true>(a, st) : launch_mv_group<T, 1, false>(a, st);
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
