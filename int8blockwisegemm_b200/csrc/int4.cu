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
#include <atomic>

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
  bool scale_packs;  // rows of scales hold whole steps, and start on 8 bytes
  const int32_t* eo;  // [E + 1]
  int n_expert;
  int64_t rows;
  int n, k;
  void* out;  // [rows, N] or [rows, N / 2]
};

// Rows of expert e, or -1 (and the error bit) when the offsets are out of order
// or leave the output.
__device__ __forceinline__ int64_t expert_rows(const MvArgs& a, int e) {
  const int64_t r0 = __ldg(a.eo + e), r1 = __ldg(a.eo + e + 1);
  if (r0 >= 0 && r0 <= r1 && r1 <= a.rows) return r1 - r0;
  atomicOr(&g_err_int4, kErrBadProblem);
  return -1;
}

__device__ __forceinline__ int64_t source_row(const MvArgs& a, int64_t r) {
  if (a.pidx == nullptr) return r;
  const int32_t p = __ldg(a.pidx + r);
  const int64_t t = p / a.topk;
  if (p >= 0 && t < a.x_rows) return t;
  atomicOr(&g_err_int4, kErrBadIndex);
  return -1;
}

// gate / (1 + exp(-gate)) * up, the exponential of the negative value on either
// side, so that it cannot overflow and the divisor is in [1, 2]: the fast
// division, whose two last bits are below the rounding of the 16-bit result,
// gives 0 for divisors above 2^126.
__device__ __forceinline__ float silu_mul(float gate, float up) {
  const float e = expf(-fabsf(gate));
  return __fdividef(gate < 0.f ? gate * e : gate, 1.f + e) * up;
}

// ---------------------------------------------------------------------------
// The products on the tensor cores
// ---------------------------------------------------------------------------
// Weights are the m16 operand of mma.m16n8k16 and a chunk of an expert's rows
// (8 per n8 tile) the other one, so that each weight is read and unpacked once
// for all rows of the chunk.  A nibble u becomes the 16-bit float u - 8, exactly;
// products are exact in the fp32 accumulators, which are scaled per group, so
// that no weight is rounded and nothing but x (u - 8) enters a sum.  (Sums that
// start at minus the offset's part, in place of an operation per pair of weights,
// carry the offset times x: a large x under a zero weight then costs the result
// its last bits, for 62 instead of 65 us in bf16, and 64 instead of 59 in fp16.)
//
// A sum over k may take the k's in any order, so each lane loads what lies
// together: lane (g, q) = (lane / 4, lane % 4) takes rows g and g + 8 of a tile
// and, of every group of G columns, the G / 4 columns from q * G / 4 on.  A
// word's nibbles j and j + 4 are the pair that one AND leaves in a register,
// and x is paired the same way.
template <typename T>
struct Mma;

#define I8_MMA(TYPE)                                                                          \
  asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE                                  \
      ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"                        \
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                        \
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), \
        "f"(c[3]))

// u - 8 of nibbles p and p + 4, as a pair of 16-bit floats: one AND-OR (a single
// three-input operation; the compiler made two of it) puts the nibbles into the
// fraction of a base, and one operation takes base and offset off again.  Both
// are exact.
__device__ __forceinline__ uint32_t masked(uint32_t w, uint32_t mask, uint32_t base) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;"  // (a & b) | c
      : "=r"(r) : "r"(w), "r"(mask), "r"(base));
  return r;
}
template <>
struct Mma<__nv_bfloat16> {
  // 7 bits of fraction: 128 + u
  static __device__ __forceinline__ uint32_t weights(uint32_t w, int p) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;"
        : "=r"(r) : "r"(masked(w >> (4 * p), 0x000f000fu, 0x43004300u)), "r"(0x43084308u));
    return r;
  }
  // d = a * b + c
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1,
                                             const float* c) {
    I8_MMA("bf16");
  }
};

template <>
struct Mma<__half> {
  // 10 bits of fraction: 1024 + u, or 1024 + 16 u
  static __device__ __forceinline__ uint32_t weights(uint32_t w, int p) {
    uint32_t r;
    if (p >= 2) w >>= 8;
    if (p % 2 == 0)
      asm("sub.rn.f16x2 %0, %1, %2;"
          : "=r"(r) : "r"(masked(w, 0x000f000fu, 0x64006400u)), "r"(0x64086408u));
    else
      asm("fma.rn.f16x2 %0, %1, %2, %3;"  // / 16 - (64 + 8)
          : "=r"(r) : "r"(masked(w, 0x00f000f0u, 0x64006400u)), "r"(0x2c002c00u), "r"(0xd480d480u));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1,
                                             const float* c) {
    I8_MMA("f16");
  }
};
#undef I8_MMA

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

template <typename T, int kCount>
struct alignas(sizeof(T) * kCount) ScalePack {
  T v[kCount];
};

// One CTA an SM: 12 warps of 160 registers take 65 us for the decode case's
// first product, 14 of 128 70 and 13 of 128 74.
constexpr int kMvThreads = 384;
constexpr int kMvWarps = kMvThreads / 32;
constexpr int kMvChunk = 8;          // rows of a chunk, one n8 tile: two took 103 us in that case
                                     // (62 then), and 49 instead of 43 with 16 rows an expert
constexpr int kMvStep = 128;         // columns of a step
constexpr int kMvSlots = 2;          // steps of weights in flight: three take 66 us
constexpr int kMvTileBytes = 16 * kMvStep / 2;
constexpr int kMvMaxExperts = 2048;

// A unit is a chunk of kMvChunk rows of an expert times a block of columns: two
// sets of weight rows of kTiles / 2 tiles each, neighbouring columns or, with
// silu, gates and their factors.  A CTA takes a contiguous range of units, and
// its warps take equal contiguous shares of the range's steps of 128 columns of
// K, wherever units begin: a warp stores the units that are its own, and the
// sums of those that it shares with the next warps meet in shared memory, once,
// at the end.
//
// Bound by latencies that three warps a scheduler leave open: 128 tokens' first
// product (256 experts, K 2048, 2 x 512 columns, 274 MB) takes 65 us, 4.2 TB/s,
// with 59 % of the issue slots busy, the ALU pipe 57 and the tensor pipe 25 %; the
// loads alone take 49 us.
//
// A warp's weights (16 kTiles rows x 128 columns a step) come through its own
// ring of slots in shared memory, steps ahead and across units, so that no
// registers wait for memory; x (which stays in L1) and the scales come one
// step ahead in registers.  In a slot, 16-byte piece c of row r lies at
// c ^ turn(r), which spreads the reads of every group size over the banks.
template <typename T, int G, int kTiles, bool kSilu>
__global__ void __launch_bounds__(kMvThreads, 1) mv_mma_kernel(MvArgs a) {
  constexpr int kGroups = kMvStep / G;  // groups of a step
  constexpr int kWords = G / 32;        // words of a lane in a group's row
  constexpr int kSetTiles = kTiles / 2, kSetRows = 16 * kSetTiles;
  constexpr int kCols = kSilu ? kSetRows : 2 * kSetRows;  // output columns of a unit
  constexpr int kSlotBytes = kTiles * kMvTileBytes;
  extern __shared__ __align__(128) unsigned char s_mem[];
  unsigned char* s_slots = s_mem;  // [warp][kMvSlots][kSlotBytes]
  float4* s_sum =                  // [warp - 1][tile][lane]
      reinterpret_cast<float4*>(s_mem + kMvWarps * kMvSlots * kSlotBytes);
  int* s_first = reinterpret_cast<int*>(s_sum + (kMvWarps - 1) * kTiles * 32);
  __shared__ int s_warp[kMvWarps];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, q = lane & 3;

  // s_first[e]: expert e's first chunk.  Offsets that are not in order are
  // refused as a whole, so that the chunks are as many as the launch allowed for.
  {
    bool bad = false;
    const int per = (a.n_expert + kMvThreads - 1) / kMvThreads;
    const int e0 = tid * per;
    int own = 0;
    for (int e = e0; e < min(a.n_expert, e0 + per); ++e) {
      const int64_t rows = expert_rows(a, e);
      bad |= rows < 0;
      const int n = rows < 0 ? 0 : static_cast<int>((rows + kMvChunk - 1) / kMvChunk);
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
    if (__syncthreads_or(bad)) return;
  }

  const int n_out = kSilu ? a.n / 2 : a.n;
  const int blocks = (n_out + kCols - 1) / kCols;
  // shares of the units, and of their steps, as equal as can be; in 32 bits,
  // since 64-bit divisions took 1.5 of one token's 10 us
  auto split = [](uint32_t n, uint32_t parts, uint32_t i) {
    const uint32_t each = n / parts;
    return static_cast<int>(each * i + min(i, n - each * parts));
  };
  const int total = s_first[a.n_expert] * blocks;
  const int u0 = split(total, gridDim.x, blockIdx.x), u1 = split(total, gridDim.x, blockIdx.x + 1);
  if (u0 == u1) return;
  const int steps = (a.k + kMvStep - 1) / kMvStep;
  const int row_bytes = a.k / 2;
  // this warp's steps of the CTA's
  const int all = (u1 - u0) * steps;
  auto share = [&](int w) { return split(all, kMvWarps, w); };
  const int i0 = share(warp), i1 = share(warp + 1);

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
    n.row0 = __ldg(a.eo + lo) + static_cast<int64_t>(n.chunk - s_first[lo]) * kMvChunk;
    n.rows = static_cast<int>(min(static_cast<int64_t>(kMvChunk), __ldg(a.eo + lo + 1) - n.row0));
  };
  auto advance = [&](Unit& n) {
    if (++n.block < blocks) return false;
    n.block = 0;
    ++n.chunk;
    find_chunk(n);
    return true;
  };

  // Weights: the lane copies piece q of every eighth row of both sets.
  const uint32_t slots =
      smem_u32(s_slots) + static_cast<uint32_t>(warp) * (kMvSlots * kSlotBytes);
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
    w_set[1] = w_set[0] + static_cast<int64_t>(kSilu ? n_out : kSetRows) * row_bytes;
    w_left = static_cast<int64_t>(a.n_expert) * a.n - (row + (kSilu ? n_out : kSetRows));
  };
  // Rows past an expert's last are the next expert's, and not stored; only the
  // tensor's end is checked.
  auto copy_weights = [&](int step, int slot) {
    const uint32_t dst = copy_at + slot * kSlotBytes;
    const int byte = step * (kMvStep / 2);
    if (byte + kMvStep / 2 <= row_bytes && w_left >= kSetRows) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < 2 * kSetTiles; ++m)
          copy16(dst + (h * 2 * kSetTiles + m) * 512,
                 w_set[h] + byte + static_cast<uint64_t>(w_stride) * m, 16);
    } else {
      const bool in = byte + q * 16 < row_bytes;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 0; m < 2 * kSetTiles; ++m) {
          const bool on = in && 8 * m < w_left + (h ? 0 : kSilu ? n_out : kSetRows);
          copy16(dst + (h * 2 * kSetTiles + m) * 512,
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
      const int c = (kSilu ? first : first + kSetRows * h) + lane % kSetRows;
      s_set[h] = static_cast<const T*>(a.scale) +
                 (base + (kSilu ? h * n_out : 0) + min(c, n_out - 1)) * a.groups;
    }
  };
  T s_next[2][kGroups];
  auto load_scales = [&](int step) {
    // A step's scales of a row at once, where they are four: 83 instead of 124
    // us for the decode case in groups of 32 (a load of every lane's own row is
    // 32 lines to look up); two, in groups of 64, gain nothing (72 against 69).
    if (kGroups == 4 && a.scale_packs) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const ScalePack<T, kGroups> p =
            *reinterpret_cast<const ScalePack<T, kGroups>*>(s_set[h] + step * kGroups);
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) s_next[h][gi] = p.v[gi];
      }
      return;
    }
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
  uint4 xr[4];
  auto clear_x = [&] {
#pragma unroll
    for (int i = 0; i < 4; ++i) xr[i] = make_uint4(0, 0, 0, 0);
  };
  const T* x_row = nullptr;
  bool x_on = false;
  auto find_row = [&](const Unit& n) {
    const int64_t src = g < n.rows ? source_row(a, n.row0 + g) : -1;
    x_on = src >= 0;
    x_row = static_cast<const T*>(a.x) + (src < 0 ? 0 : src) * a.x_stride + q * kWords * 8;
    if (!x_on) clear_x();
  };
  auto load_x = [&](int step) {
    const int k0 = step * kMvStep;
    const bool tail = k0 + kMvStep > a.k;
    if (!x_on) return;
    const uint4* p = reinterpret_cast<const uint4*>(x_row + k0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = (i / kWords) * (G / 8) + i % kWords;
      if (!tail || k0 + (at + q * kWords) * 8 < a.k) xr[i] = __ldg(p + at);
      else xr[i] = make_uint4(0, 0, 0, 0);
    }
  };

  float acc[kTiles][4];
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][c] = 0.f;
  };
  // acc[i] holds rows 2 q and 2 q + 1, columns g and g + 8 of tile i; a
  // transpose gives each lane one row and two neighbouring columns
  auto store = [&](const Unit& n) {
    constexpr int kOut = kSilu ? kSetTiles : kTiles;
    uint32_t pair[kOut][2];
#pragma unroll
    for (int i = 0; i < kOut; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        __align__(4) T v[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float y = acc[i][half * 2 + j];
          v[j] = Num<T>::from_f(
              kSilu ? silu_mul(y, acc[kSilu ? i + kSetTiles : i][half * 2 + j]) : y);
        }
        // volatile: all lanes have to take part, also those that store nothing
        asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;"
                     : "=r"(pair[i][half]) : "r"(*reinterpret_cast<const uint32_t*>(v)));
      }
    if (g >= n.rows) return;
    T* out = static_cast<T*>(a.out) + (n.row0 + g) * n_out;
#pragma unroll
    for (int i = 0; i < kOut; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int col = n.block * kCols + i * 16 + half * 8 + 2 * q;
        const T* p = reinterpret_cast<const T*>(&pair[i][half]);
        if (n_out % 2 == 0) {
          if (col < n_out) *reinterpret_cast<uint32_t*>(out + col) = pair[i][half];
        } else {
          if (col < n_out) out[col] = p[0];
          if (col + 1 < n_out) out[col + 1] = p[1];
        }
      }
  };
  auto leave_sum = [&] {  // for the warp that has the unit's first steps
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
      s_sum[((warp - 1) * kTiles + i) * 32 + lane] =
          make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  };

  // `cur` is the unit that is computed, `ahead` the one whose weights are
  // copied next
  Unit cur, done;
  int step = 0, from = 0;  // the step at hand, the unit's first one of this warp
  bool open = false;       // acc holds a unit's first steps, not its last
  clear();
  clear_x();
  if (i0 < i1) {
    const int u = u0 + i0 / steps;
    step = from = i0 % steps;
    cur.chunk = u / blocks;
    cur.block = u - cur.chunk * blocks;
    find_chunk(cur);
    Unit ahead = cur;
    find_weights(ahead);
    int st_ahead = step;
    int i_ahead = i0;
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
    find_scales(cur);
    load_scales(step);
    find_row(cur);
    load_x(step);

    int slot = 0;
    for (int left = i1 - i0; left > 0; --left) {
      // x in the weights' pairing: b[word][j] = (x[j], x[j + 4])
      uint32_t b[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b[i][0] = __byte_perm(xr[i].x, xr[i].z, 0x5410);
        b[i][1] = __byte_perm(xr[i].x, xr[i].z, 0x7632);
        b[i][2] = __byte_perm(xr[i].y, xr[i].w, 0x5410);
        b[i][3] = __byte_perm(xr[i].y, xr[i].w, 0x7632);
      }
      float s_row[2][kGroups];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) s_row[h][gi] = Num<T>::to_f(s_next[h][gi]);
      const bool last = step + 1 == steps;
      if (last) done = cur;
      if (left > 1) {
        if (last) {
          if (advance(cur)) find_row(cur);
          find_scales(cur);
        }
        load_x(last ? 0 : step + 1);
        load_scales(last ? 0 : step + 1);
      }
      copies_wait<kMvSlots - 1>();
      __syncwarp();
      const uint32_t base = slot * kSlotBytes;
      constexpr float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {  // tile i: rows 16 (i % kSetTiles) of set i / kSetTiles
        uint32_t w[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int gi = 0; gi < kGroups; ++gi)
            load_shared<kWords>(read_at[gi] + base + (i * 2 + half) * 512, &w[half][gi * kWords]);
#pragma unroll
        for (int gi = 0; gi < kGroups; ++gi) {
          float part[4];
#pragma unroll
          for (int j = 0; j < kWords; ++j) {
            const int wi = gi * kWords + j;
            uint32_t f[2][4];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int p = 0; p < 4; ++p) f[half][p] = Mma<T>::weights(w[half][wi], p);
            Mma<T>::mma(part, f[0][0], f[1][0], f[0][1], f[1][1], b[wi][0], b[wi][1],
                        j == 0 ? zero : part);
            Mma<T>::mma(part, f[0][2], f[1][2], f[0][3], f[1][3], b[wi][2], b[wi][3], part);
          }
          const int row = i % kSetTiles * 16 + g;
          const float s0 = __shfl_sync(0xffffffffu, s_row[i / kSetTiles][gi], row);
          const float s1 = __shfl_sync(0xffffffffu, s_row[i / kSetTiles][gi], row + 8);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][c] = fmaf(part[c], c < 2 ? s0 : s1, acc[i][c]);
        }
      }
      __syncwarp();
      copy_next(slot);
      slot = slot + 1 == kMvSlots ? 0 : slot + 1;

      if (last) {
        if (from == 0) store(done);
        else leave_sum();
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
      leave_sum();
      open = false;
    }
  }
  __syncthreads();
  if (!open) return;
  // the warps after this one that have steps of its last unit
  const int end = i1 + (steps - step);
  for (int v = warp + 1; v < kMvWarps && share(v) < end; ++v) {
    if (share(v) == share(v + 1)) continue;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const float4 p = s_sum[((v - 1) * kTiles + i) * 32 + lane];
      acc[i][0] += p.x;
      acc[i][1] += p.y;
      acc[i][2] += p.z;
      acc[i][3] += p.w;
    }
  }
  store(cur);
}

template <typename T, int G, int kTiles, bool kSilu>
int launch_mv_kernel(const MvArgs& a, int64_t units, cudaStream_t st) {
  const int smem = kMvWarps * kMvSlots * kTiles * kMvTileBytes +
                   (kMvWarps - 1) * kTiles * 32 * static_cast<int>(sizeof(float4)) +
                   (a.n_expert + 1) * static_cast<int>(sizeof(int));
  const int64_t sms = num_sms(current_device()), steps = (a.k + kMvStep - 1) / kMvStep;
  I8_REQUIRE(units < (int64_t(1) << 31) && (units / sms + 1) * steps < (int64_t(1) << 31),
             "int4_grouped_mv: too many rows for one call");
  auto kernel = mv_mma_kernel<T, G, kTiles, kSilu>;
  constexpr int kMost = kMvWarps * kMvSlots * kTiles * kMvTileBytes +
                        (kMvWarps - 1) * kTiles * 32 * 16 + 4 * (kMvMaxExperts + 1);
  static std::atomic<uint64_t> allowed{0};  // a bit per device
  const uint64_t bit = uint64_t(1) << (current_device() % 64);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    I8_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(units, sms));
  kernel<<<grid, kMvThreads, smem, st>>>(a);
  return check_launch("int4_grouped_mv");
}

template <typename T, int kTiles, bool kSilu>
int launch_mv_group(const MvArgs& a, int64_t units, cudaStream_t st) {
  if (a.group == 128) return launch_mv_kernel<T, 128, kTiles, kSilu>(a, units, st);
  if (a.group == 64) return launch_mv_kernel<T, 64, kTiles, kSilu>(a, units, st);
  return launch_mv_kernel<T, 32, kTiles, kSilu>(a, units, st);
}

// Units of four tiles, or of two where the former leave SMs without work (one
// row of 4096 x 4096: 8.3 us instead of 10.4; with work for all SMs twice the
// loads of x cost more, 16.4 instead of 14.5 us for 4 tokens of the decode
// case).
template <typename T, bool kSilu>
int launch_mv(const MvArgs& a, cudaStream_t st) {
  const int64_t chunks = std::min<int64_t>(a.rows, (a.rows + kMvChunk - 1) / kMvChunk + a.n_expert);
  const int cols = kSilu ? 32 : 64, n_out = kSilu ? a.n / 2 : a.n;
  const int64_t units = (n_out + cols - 1) / cols * chunks;
  if (units >= num_sms(current_device())) return launch_mv_group<T, 4, kSilu>(a, units, st);
  return launch_mv_group<T, 2, kSilu>(a, (n_out + cols / 2 - 1) / (cols / 2) * chunks, st);
}

// One warp per group: scale = max|w| / 7 rounded to the scale's type, and
// u = clamp(rint(w / scale), -8, 7) + 8 by that rounded scale, so that its
// rounding shifts no weight twice.  A group of zeros (or one whose scale
// rounds to zero) gets scale 0 and u = 8; one with a NaN scale NaN, one with an
// infinity (or whose scale leaves its type) scale inf, and u = 8 both, so that
// what is wrong with a weight reaches the products as NaN.
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
    for (int c = k0 + lane; c < k1; c += 32) m = max_nan(m, fabsf(Num<T>::to_f(src[c])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
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
  I8_REQUIRE(w && packed && scale, "quantize_weights_int4: every tensor must be given");
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
  I8_REQUIRE(n_expert >= 0 && n_expert <= kMvMaxExperts, "int4_grouped_mv: n_expert must be in [0, 2048]");
  I8_REQUIRE(n_rows >= 0 && n_rows < (int64_t(1) << 31) && x_rows >= 0,
             "int4_grouped_mv: bad n_rows");
  I8_REQUIRE(topk >= 1 && topk < (int64_t(1) << 31), "int4_grouped_mv: topk must be positive");
  I8_REQUIRE(permuted_idx != nullptr || x_rows >= n_rows,
             "int4_grouped_mv: x has fewer rows than the output");
  if (n_rows == 0 || n == 0 || n_expert == 0) return I8MOE_OK;
  I8_REQUIRE(x && w_packed && w_scale && expert_offsets && out,
             "int4_grouped_mv: every tensor must be given");
  I8_REQUIRE(x_stride >= k && x_stride % 8 == 0 && bits(x) % 16 == 0 && bits(w_packed) % 16 == 0 &&
                 bits(out) % 16 == 0,
             "int4_grouped_mv: x rows, w_packed and out must be 16-byte aligned");
  MvArgs a{x, x_stride, x_rows, permuted_idx, static_cast<int>(topk), w_packed, w_scale,
           static_cast<int>(group_size),
           static_cast<int>((k + group_size - 1) / group_size),
           k % kMvStep == 0 && bits(w_scale) % 8 == 0, expert_offsets,
           static_cast<int>(n_expert), n_rows, static_cast<int>(n), static_cast<int>(k), out};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == I8MOE_BF16)
    return silu ? launch_mv<__nv_bfloat16, true>(a, st) : launch_mv<__nv_bfloat16, false>(a, st);
  return silu ? launch_mv<__half, true>(a, st) : launch_mv<__half, false>(a, st);
}

}  // extern "C"
