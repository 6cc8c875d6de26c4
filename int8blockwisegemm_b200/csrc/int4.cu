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
  const void* scale;  // [E, N, groups], x's type
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
  return -1;
}

// The quotient's two last bits are below the rounding of the 16-bit result.
__device__ __forceinline__ float silu_mul(float gate, float up) {
  return __fdividef(gate, 1.f + expf(-gate)) * up;
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
  // d = a * b + (first ? 0 : d)
  static __device__ __forceinline__ void mma(bool first, float (&d)[4], uint32_t a0, uint32_t a1,
                                             uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (first)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
          "{%8,%9}, {%10,%10,%10,%10};"
          : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
          : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
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
  static __device__ __forceinline__ void mma(bool first, float (&d)[4], uint32_t a0, uint32_t a1,
                                             uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (first)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
          "{%8,%9}, {%10,%10,%10,%10};"
          : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
          : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
          "{%8,%9}, {%0,%1,%2,%3};"
          : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
          : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// (w >> shift) & 0x000f000f | base: the pair of nibbles `shift / 4` of both
// halves, each in the low bits of a float.  As one three-input operation (the
// compiler made two of it: 102 against 90 us for the decode case's first
// product).
template <typename T>
__device__ __forceinline__ uint32_t nibble_pair(uint32_t w, int shift) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;"  // (a & b) | c
      : "=r"(r) : "r"(w >> shift), "r"(0x000f000fu), "r"(Mma<T>::kBase));
  return Mma<T>::minus(r);
}

// 16 bytes to shared memory past L1; `bytes` 0 fills with zeros and reads
// nothing.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copies_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kPending>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
template <int kWords>
__device__ __forceinline__ void load_shared(uint32_t at, uint32_t* w) {
  if constexpr (kWords == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
  else if constexpr (kWords == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at));
}

constexpr int kMvThreads = 256;
constexpr int kMvWarps = kMvThreads / 32;
constexpr int kMvTiles = 4;          // m16 tiles of a warp
constexpr int kMvStep = 128;         // columns of a step
constexpr int kMvSlots = 2;          // steps of weights in flight; more would leave L1 too small
constexpr int kMvSlotBytes = 64 * kMvStep / 2;

// A unit is a chunk of 8 * kNt rows of an expert times a block of columns: two
// sets of 32 weight rows, 64 columns or, with silu, 32 gates and their 32
// factors.  A CTA takes a contiguous range of units, and its 8 warps take equal
// contiguous shares of the range's steps of 128 columns of K, wherever units
// begin: a warp stores the units that are its own, and the sums of those that
// it shares with the next warps meet in shared memory, once, at the end (one
// barrier per unit cost a third of the decode case's time).
//
// A warp's weights (64 rows x 128 columns, 4 KB a step) come through its own
// ring of slots in shared memory, steps ahead and across units, so that no
// registers wait for memory; x (which stays in L1) and the scales come one
// step ahead in registers.  In a slot, 16-byte piece c of row r lies at
// c ^ turn(r), which spreads the reads of every group size over the banks.
template <typename T, int G, int kNt, bool kSilu>
__global__ void __launch_bounds__(kMvThreads, 2) mv_mma_kernel(MvArgs a) {
  constexpr int kGroups = kMvStep / G;  // groups of a step
  constexpr int kWords = G / 32;        // words of a lane in a group's row
  constexpr int kChunk = 8 * kNt;
  constexpr int kCols = kSilu ? 32 : 64;  // output columns of a unit
  extern __shared__ __align__(128) unsigned char s_mem[];
  unsigned char* s_slots = s_mem;  // [warp][kMvSlots][kMvSlotBytes]
  float4* s_sum =                  // [warp - 1][tile][kNt][lane]
      reinterpret_cast<float4*>(s_mem + kMvWarps * kMvSlots * kMvSlotBytes);
  int* s_first = reinterpret_cast<int*>(s_sum + (kMvWarps - 1) * kMvTiles * kNt * 32);
  __shared__ int s_warp[kMvWarps];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, q = lane & 3;

  // s_first[e]: expert e's first chunk
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
  const int blocks = (n_out + kCols - 1) / kCols;
  const int64_t total = static_cast<int64_t>(s_first[a.n_expert]) * blocks;
  const int64_t u0 = total * blockIdx.x / gridDim.x, u1 = total * (blockIdx.x + 1) / gridDim.x;
  if (u0 == u1) return;
  const int steps = (a.k + kMvStep - 1) / kMvStep;
  const int row_bytes = a.k / 2;
  // this warp's steps of the CTA's
  const int64_t all = (u1 - u0) * steps;
  auto share = [&](int w) { return all * w / kMvWarps; };
  const int64_t i0 = share(warp), i1 = share(warp + 1);

  // A unit: the rows of a chunk and a block of columns
  struct Unit {
    int chunk, block, expert, rows;
    int64_t row0;
  };
  auto find_chunk = [&](Unit& n) {
    int lo = 0, hi = a.n_expert;  // the expert with s_first[lo] <= chunk < s_first[lo + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_first[mid] <= n.chunk) lo = mid;
      else hi = mid;
    }
    n.expert = lo;
    n.row0 = __ldg(a.eo + lo) + static_cast<int64_t>(n.chunk - s_first[lo]) * kChunk;
    n.rows = static_cast<int>(min(static_cast<int64_t>(kChunk), __ldg(a.eo + lo + 1) - n.row0));
  };
  auto advance = [&](Unit& n) {
    if (++n.block < blocks) return false;
    n.block = 0;
    ++n.chunk;
    find_chunk(n);
    return true;
  };

  // Weights: the lane copies piece q of rows g, g + 8, g + 16 and g + 24 of
  // both sets; rows past the expert's last repeat it and are not stored.
  const uint32_t slots =
      smem_u32(s_slots) + static_cast<uint32_t>(warp) * (kMvSlots * kMvSlotBytes);
  const int turn = ((g >> 1) & 1) * 2 + (g >> 2);
  const uint32_t copy_at = slots + g * 64 + ((q ^ turn) << 4);
  uint32_t read_at[kGroups];
#pragma unroll
  for (int gi = 0; gi < kGroups; ++gi) {
    const int piece = kGroups == 1 ? q : kGroups == 2 ? 2 * gi + (q >> 1) : gi;
    const int byte = kGroups == 1 ? 0 : kGroups == 2 ? (q & 1) * 8 : q * 4;
    read_at[gi] = slots + g * 64 + ((piece ^ turn) << 4) + byte;
  }
  const uint8_t* w_set[2];  // piece q of row g of a set
  int64_t w_left = 0;       // rows of the tensor from the second set's row g on
  const uint32_t w_stride = 8 * row_bytes;
  auto find_weights = [&](const Unit& n) {
    const int64_t row = static_cast<int64_t>(n.expert) * a.n + n.block * kCols + g;
    w_set[0] = a.w + row * row_bytes + q * 16;
    w_set[1] = w_set[0] + static_cast<int64_t>(kSilu ? n_out : 32) * row_bytes;
    w_left = static_cast<int64_t>(a.n_expert) * a.n - (row + (kSilu ? n_out : 32));
  };
  // Rows past an expert's last are the next expert's, and not stored; only the
  // tensor's end is checked.
  auto copy_weights = [&](int step, int slot) {
    const uint32_t dst = copy_at + slot * kMvSlotBytes;
    const int byte = step * (kMvStep / 2);
    if (byte + kMvStep / 2 <= row_bytes && w_left >= 32) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          copy16(dst + (h * 4 + m) * 512,
                 w_set[h] + byte + static_cast<uint64_t>(w_stride) * m, 16);
    } else {
      const bool in = byte + q * 16 < row_bytes;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const bool on = in && 8 * m < w_left + (h ? 0 : kSilu ? n_out : 32);
          copy16(dst + (h * 4 + m) * 512,
                 on ? w_set[h] + byte + static_cast<uint64_t>(w_stride) * m : a.w, on ? 16 : 0);
        }
    }
  };
  const T* s_set[2];  // the scales of row `lane` of a set
  auto find_scales = [&](const Unit& n) {
    const int first = n.block * kCols;
    const int64_t base = static_cast<int64_t>(n.expert) * a.n;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = kSilu ? first : first + 32 * h;
      s_set[h] = static_cast<const T*>(a.scale) +
                 (base + (kSilu ? h * n_out : 0) + min(c + lane, n_out - 1)) * a.groups;
    }
  };
  T s_next[2][kGroups];
  auto load_scales = [&](int step) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int gi = 0; gi < kGroups; ++gi) {
        const int at = step * kGroups + gi;
        s_next[h][gi] =
            kGroups == 1 || at < a.groups ? __ldg(s_set[h] + at) : Num<T>::from_f(0.f);
      }
  };

  // x: eight values of each of the lane's words, through L1.  Rows that the
  // chunk does not have are not loaded, and what their registers hold is not
  // stored; rows whose index is bad and columns past K are zeros.
  uint4 xr[kNt][4];
#pragma unroll
  for (int t = 0; t < kNt; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) xr[t][i] = make_uint4(0, 0, 0, 0);
  const T* x_row[kNt];
  bool x_on[kNt];
  auto find_rows = [&](const Unit& n) {
#pragma unroll
    for (int t = 0; t < kNt; ++t) {
      const int r = t * 8 + g;
      const int64_t src = r < n.rows ? source_row(a, n.row0 + r) : -1;
      x_on[t] = src >= 0;
      x_row[t] = static_cast<const T*>(a.x) + (src < 0 ? 0 : src) * a.x_stride + q * kWords * 8;
      if (src < 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) xr[t][i] = make_uint4(0, 0, 0, 0);
      }
    }
  };
  auto load_x = [&](int step) {
    const int k0 = step * kMvStep;
    const bool tail = k0 + kMvStep > a.k;
#pragma unroll
    for (int t = 0; t < kNt; ++t)
      if (x_on[t]) {
        const uint4* p = reinterpret_cast<const uint4*>(x_row[t] + k0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = (i / kWords) * (G / 8) + i % kWords;
          if (!tail || k0 + (at + q * kWords) * 8 < a.k) xr[t][i] = __ldg(p + at);
          else xr[t][i] = make_uint4(0, 0, 0, 0);
        }
      }
  };

  float acc[kMvTiles][kNt][4];
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < kMvTiles; ++i)
#pragma unroll
      for (int t = 0; t < kNt; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][t][c] = 0.f;
  };
  // acc[i][t] holds rows 2 q, 2 q + 1 of n8 tile t, columns g and g + 8 of tile
  // i; a transpose gives each lane one row and two neighbouring columns
  auto store = [&](const Unit& n) {
#pragma unroll
    for (int t = 0; t < kNt; ++t) {
      const int row = t * 8 + g;
      T* out = static_cast<T*>(a.out) + (n.row0 + row) * n_out;
#pragma unroll
      for (int i = 0; i < (kSilu ? 2 : 4); ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          __align__(4) T v[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float y = acc[i][t][half * 2 + j];
            v[j] = Num<T>::from_f(kSilu ? silu_mul(y, acc[kSilu ? i + 2 : i][t][half * 2 + j]) : y);
          }
          uint32_t pair = *reinterpret_cast<const uint32_t*>(v);
          asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(pair));
          const int col = n.block * kCols + i * 16 + half * 8 + 2 * q;
          if (row < n.rows) {
            const T* p = reinterpret_cast<const T*>(&pair);
            if (n_out % 2 == 0) {
              if (col < n_out) *reinterpret_cast<uint32_t*>(out + col) = pair;
            } else {
              if (col < n_out) out[col] = p[0];
              if (col + 1 < n_out) out[col + 1] = p[1];
            }
          }
        }
    }
  };

  // `cur` is the unit that is computed, `ahead` the one whose weights are
  // copied next
  Unit cur, done;
  int step = 0, from = 0;  // the step at hand, the unit's first one of this warp
  bool open = false;       // acc holds a unit's first steps, not its last
  clear();
  if (i0 < i1) {
    const int64_t u = u0 + i0 / steps;
    step = from = static_cast<int>(i0 % steps);
    cur.chunk = static_cast<int>(u / blocks);
    cur.block = static_cast<int>(u - static_cast<int64_t>(cur.chunk) * blocks);
    find_chunk(cur);
    find_rows(cur);
    find_scales(cur);
    Unit ahead = cur;
    find_weights(ahead);
    int st_ahead = step;
    int64_t i_ahead = i0;
    auto copy_next = [&](int slot) {
      if (i_ahead < i1) {
        copy_weights(st_ahead, slot);
        if (++i_ahead < i1 && ++st_ahead == steps) {
          st_ahead = 0;
          advance(ahead);
          find_weights(ahead);
        }
      }
      copies_commit();
    };
#pragma unroll
    for (int s = 0; s < kMvSlots; ++s) copy_next(s);
    load_x(step);
    load_scales(step);

    int slot = 0;
    for (int64_t i1_left = i1 - i0; i1_left > 0; --i1_left) {
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
      float s_row[2][kGroups];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) s_row[h][gi] = Num<T>::to_f(s_next[h][gi]);
      const bool last = step + 1 == steps;
      if (last) done = cur;
      if (i1_left > 1) {
        if (last) {
          if (advance(cur)) find_rows(cur);
          find_scales(cur);
        }
        load_x(last ? 0 : step + 1);
        load_scales(last ? 0 : step + 1);
      }
      copies_wait<kMvSlots - 1>();
      __syncwarp();
      const uint32_t base = slot * kMvSlotBytes;
#pragma unroll
      for (int i = 0; i < kMvTiles; ++i) {  // tile i: rows 16 (i % 2) of set i / 2
        uint32_t w[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int gi = 0; gi < kGroups; ++gi)
            load_shared<kWords>(read_at[gi] + base + (i * 2 + half) * 512, &w[half][gi * kWords]);
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) {
          float part[kNt][4];
#pragma unroll
          for (int j = 0; j < kWords; ++j) {
            const int wi = gi * kWords + j;
            uint32_t f[2][4];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int p = 0; p < 4; ++p) f[half][p] = nibble_pair<T>(w[half][wi], 4 * p);
#pragma unroll
            for (int t = 0; t < kNt; ++t) {
              Mma<T>::mma(j == 0, part[t], f[0][0], f[1][0], f[0][1], f[1][1], b[t][wi][0],
                          b[t][wi][1]);
              Mma<T>::mma(false, part[t], f[0][2], f[1][2], f[0][3], f[1][3], b[t][wi][2],
                          b[t][wi][3]);
            }
          }
          const float s0 = __shfl_sync(0xffffffffu, s_row[i >> 1][gi], (i & 1) * 16 + g);
          const float s1 = __shfl_sync(0xffffffffu, s_row[i >> 1][gi], (i & 1) * 16 + 8 + g);
#pragma unroll
          for (int t = 0; t < kNt; ++t)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              acc[i][t][c] = fmaf(part[t][c], c < 2 ? s0 : s1, acc[i][t][c]);
        }
      }
      __syncwarp();
      copy_next(slot);
      slot = slot + 1 == kMvSlots ? 0 : slot + 1;

      if (last) {
        if (from == 0) {
          store(done);
        } else {  // an earlier warp has the unit's first steps
#pragma unroll
          for (int i = 0; i < kMvTiles; ++i)
#pragma unroll
            for (int t = 0; t < kNt; ++t)
              s_sum[(((warp - 1) * kMvTiles + i) * kNt + t) * 32 + lane] =
                  make_float4(acc[i][t][0], acc[i][t][1], acc[i][t][2], acc[i][t][3]);
        }
        clear();
        from = 0;
        step = 0;
      } else {
        ++step;
      }
    }
    copies_wait<0>();
    open = step != 0;
    if (open && from != 0) {  // neither the unit's first steps nor its last
#pragma unroll
      for (int i = 0; i < kMvTiles; ++i)
#pragma unroll
        for (int t = 0; t < kNt; ++t)
          s_sum[(((warp - 1) * kMvTiles + i) * kNt + t) * 32 + lane] =
              make_float4(acc[i][t][0], acc[i][t][1], acc[i][t][2], acc[i][t][3]);
      open = false;
    }
  }
  __syncthreads();
  if (!open) return;
  // the warps after this one that have steps of its last unit
  const int64_t end = i1 + (steps - step);
  for (int v = warp + 1; v < kMvWarps && share(v) < end; ++v) {
    if (share(v) == share(v + 1)) continue;
#pragma unroll
    for (int i = 0; i < kMvTiles; ++i)
#pragma unroll
      for (int t = 0; t < kNt; ++t) {
        const float4 p = s_sum[(((v - 1) * kMvTiles + i) * kNt + t) * 32 + lane];
        acc[i][t][0] += p.x;
        acc[i][t][1] += p.y;
        acc[i][t][2] += p.z;
        acc[i][t][3] += p.w;
      }
  }
  store(cur);
}

template <typename T, int G, int kNt, bool kSilu>
int launch_mv_kernel(const MvArgs& a, cudaStream_t st) {
  const int smem = kMvWarps * kMvSlots * kMvSlotBytes +
                   (kMvWarps - 1) * kMvTiles * kNt * 32 * static_cast<int>(sizeof(float4)) +
                   (a.n_expert + 1) * static_cast<int>(sizeof(int));
  auto kernel = mv_mma_kernel<T, G, kNt, kSilu>;
  I8_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int64_t cols = kSilu ? 32 : 64;
  const int64_t units =
      (((kSilu ? a.n / 2 : a.n) + cols - 1) / cols) *
      std::min<int64_t>(a.rows, (a.rows + 8 * kNt - 1) / (8 * kNt) + a.n_expert);
  const unsigned grid =
      static_cast<unsigned>(std::min<int64_t>(units, int64_t(num_sms(current_device())) * 2));
  kernel<<<grid, kMvThreads, smem, st>>>(a);
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
                          const void* w_scale, int64_t group_size, const int32_t* expert_offsets,
                          int64_t n_expert, int64_t n_rows, int64_t n, int64_t k, int silu,
                          void* out, i8moe_stream_t stream) {
  I8_REQUIRE(dtype == I8MOE_BF16 || dtype == I8MOE_FP16,
             "int4_grouped_mv: x must be bfloat16 or float16");
  I8_REQUIRE(group_size == 32 || group_size == 64 || group_size == 128,
             "int4_grouped_mv: group_size must be 32, 64 or 128");
  I8_REQUIRE(k >= 32 && k % 32 == 0 && k < (int64_t(1) << 26),
             "int4_grouped_mv: K must be positive, divisible by 32 and below 2^26");
  I8_REQUIRE(n >= 0 && n < (int64_t(1) << 31) - 128 && (!silu || n % 2 == 0),
             "int4_grouped_mv: bad N (even with silu)");
  I8_REQUIRE(n_expert >= 0 && n_expert <= 2048, "int4_grouped_mv: n_expert must be in [0, 2048]");
  I8_REQUIRE(n_rows >= 0 && n_rows < (int64_t(1) << 31) && x_rows >= 0,
             "int4_grouped_mv: bad n_rows");
  I8_REQUIRE(topk >= 1 && topk < (int64_t(1) << 31), "int4_grouped_mv: topk must be positive");
  I8_REQUIRE(permuted_idx != nullptr || x_rows >= n_rows,
             "int4_grouped_mv: x has fewer rows than the output");
  if (n_rows == 0 || n == 0 || n_expert == 0) return I8MOE_OK;
  I8_REQUIRE(x_stride >= k && x_stride % 8 == 0 && bits(x) % 16 == 0 && bits(w_packed) % 16 == 0 &&
                 bits(out) % 16 == 0,
             "int4_grouped_mv: x rows, w_packed and out must be 16-byte aligned");
  MvArgs a{x, x_stride, x_rows, permuted_idx, static_cast<int>(topk), w_packed, w_scale,
           static_cast<int>(group_size),
           static_cast<int>((k + group_size - 1) / group_size), expert_offsets,
           static_cast<int>(n_expert), n_rows, static_cast<int>(n), static_cast<int>(k), out};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == I8MOE_BF16) return launch_mv<__nv_bfloat16>(a, silu != 0, st);
  return launch_mv<__half>(a, silu != 0, st);
}

}  // extern "C"
