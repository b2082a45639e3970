// Matrix product of 8-bit (e4m3) operands with block scales, on the matrix cores.
//
//   C[m][t] = sum_b ws[m / 128][b] xs[b][t] sum_{k in block b} w[m][k] x[t][k]
//
// over blocks of 128 features, C in bf16 or float32, features-major [M][T] or token-major
// [T][M]. A block's sum is scaled and added to the output's float32 accumulator, which is
// rounded once at the end.
//
// The 8-bit matrix instructions (v_mfma_f32_16x16x128_f8f6f4 and the shorter ones alike) add each
// 8 neighbouring products of a row before they reach the float32 accumulator, and in that sum
// drop what lies below 2^-13 of the largest of the 8 (measured on MI355X: a product 2^-13 of its
// neighbour counts, one of 2^-14 does not; 8 features further on products count down to 2^-23).
// Against float64 that is 1.5e-5 of the result for normally distributed operands and 6e-5 for
// features of very different sizes, where float32 sums are off by 1e-8: less than a hundredth of
// a bf16 output's own rounding, but far more than a float32 output's, and more than either where a
// large product that others of its 8 cancel hides the rest. So a float32 output takes
// its operands to bf16 (exact, v_cvt_scalef32_pk_bf16_fp8) and multiplies with the bf16
// instructions, at half the rate; a bf16 output does so in the kernel for few tokens, where it costs
// nothing. In tiles it would (us, 8-bit and bf16 instructions): 1280 x 2560 x 333 6.7, 8.3; 2560 x 1280
// x 512 7.1, 9.8; 5120 x 1280 x 1024 13.0, 20; x 16384 130, 196; 50280 x 768 x 8 8.6, 9.0. A caller who
// needs float32 sums there asks for a float32 output.
#include <hip/hip_runtime.h>

#include <cmath>

#include "mss_serve.h"

namespace mss {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 8 e4m3 values as bf16.
__device__ __forceinline__ bf16x8 to_bf16x8(int lo, int hi) {
  const bf16x2_t v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
  const bf16x2_t v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
  const bf16x2_t v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
  const bf16x2_t v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
  return bf16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}

__device__ __forceinline__ i32x8 join(const u32x4& lo, const u32x4& hi) {
  return i32x8{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(lo[2]), static_cast<int>(lo[3]),
               static_cast<int>(hi[0]), static_cast<int>(hi[1]), static_cast<int>(hi[2]), static_cast<int>(hi[3])};
}

// A lane's 32 values of an operand's block, ready for the matrix instructions.
template <bool kF8>
struct MmFrag;
template <>
struct MmFrag<true> {
  i32x8 v;
  __device__ __forceinline__ void set(const u32x4& lo, const u32x4& hi) { v = join(lo, hi); }
};
template <>
struct MmFrag<false> {
  bf16x8 v[4];
  __device__ __forceinline__ void set(const u32x4& lo, const u32x4& hi) {
    v[0] = to_bf16x8(lo[0], lo[1]);
    v[1] = to_bf16x8(lo[2], lo[3]);
    v[2] = to_bf16x8(hi[0], hi[1]);
    v[3] = to_bf16x8(hi[2], hi[3]);
  }
};
// The sum over one block: rows of `a` (16) by rows of `b` (16). Lane l holds a's row l % 16 (the
// result's rows) and b's row l % 16 (its columns), features 16 (l / 16) .. + 16 of the block's
// first half and the same of the second; the result's lane l has column l % 16, rows
// 4 (l / 16) .. + 4. The order of the features inside a block is the same in both operands, and
// that is all their sum needs.
__device__ __forceinline__ f32x4 mfma_block(const MmFrag<true>& a, const MmFrag<true>& b) {
  const f32x4 z = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, z, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_block(const MmFrag<false>& a, const MmFrag<false>& b) {
  f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], d, 0, 0, 0);
  return d;
}

// The 16 bytes of a row from k on, zero past K (k a multiple of 16, below the row's stride). The
// bytes between K and the stride may hold anything, and the last row may end at K.
__device__ __forceinline__ u32x4 load_chunk(const unsigned char* __restrict__ base, long long ld, int row, int rows, int k,
                                         int K) {
  const unsigned char* r = base + row * ld + k;
  const int n = K - k;
  u32x4 v = {};
  if (n >= 16 || (n > 0 && row < rows - 1)) {
    v = *reinterpret_cast<const u32x4*>(r);
  } else {
#pragma unroll 1
    for (int i = n - 1; i >= 0; --i)
      v = u32x4{(v[0] << 8) | r[i], (v[1] << 8) | (v[0] >> 24), (v[2] << 8) | (v[1] >> 24), (v[3] << 8) | (v[2] >> 24)};
  }
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int left = n - 4 * d;
    v[d] &= left <= 0 ? 0u : left >= 4 ? 0xffffffffu : (1u << (8 * left)) - 1;
  }
  return v;
}

// ------------------------------------------------------------------------- few tokens, few tiles
// No LDS on the way in: a wave reads its operands' rows straight from memory and the caches, a
// block ahead of the products. The 8 waves of a workgroup share one tile of 16 x 16, every eighth
// block each, and their sums meet in LDS in a fixed order.
struct RowBlock {
  u32x4 v[2];  // 16 bytes at 16 g and 16 at 16 g + 64 of the block
  __device__ __forceinline__ void load(const unsigned char* __restrict__ base, long long ld, int row, int rows, int k,
                                       int K) {
    v[0] = v[1] = u32x4{0, 0, 0, 0};
    if (row < rows) {
      const unsigned char* r = base + row * ld + k;
      if (k + 80 <= K) {
        v[0] = *reinterpret_cast<const u32x4*>(r);
        v[1] = *reinterpret_cast<const u32x4*>(r + 64);
      } else {
        v[0] = load_chunk(base, ld, row, rows, k, K);
        v[1] = load_chunk(base, ld, row, rows, k + 64, K);
      }
    }
  }
};

constexpr int kRowsWaves = 8;
template <typename out_t>
__global__ __launch_bounds__(64 * kRowsWaves) void fp8mm_rows_kernel(Fp8MmParams p) {
  __shared__ f32x4 s_part[kRowsWaves - 1][64];
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m0 = blockIdx.x * 16, t = blockIdx.y * 16 + j;
  const int nkb = (p.K + kFp8Block - 1) / kFp8Block;
  const float* __restrict__ ws = p.ws + static_cast<long long>(m0 / kFp8Block) * nkb;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  RowBlock w, x;
  float s;
  const auto fetch = [&](int b) {
    const int k = b * kFp8Block + 16 * g;
    w.load(p.w, p.ldw, m0 + j, p.M, k, p.K);
    x.load(p.x, p.ldx, t, p.T, k, p.K);
    s = t < p.T ? p.xs[static_cast<long long>(b) * p.T + t] * ws[b] : 0.f;
  };
  int b = wave;
  if (b < nkb) fetch(b);
  for (; b < nkb; b += kRowsWaves) {
    MmFrag<false> wf, xf;
    wf.set(w.v[0], w.v[1]);
    xf.set(x.v[0], x.v[1]);
    const float sc = s;
    if (b + kRowsWaves < nkb) fetch(b + kRowsWaves);
    const f32x4 d = mfma_block(wf, xf);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(d[e], sc, acc[e]);
  }
  if (wave > 0) s_part[wave - 1][lane] = acc;
  __syncthreads();
  if (wave > 0 || t >= p.T) return;
#pragma unroll
  for (int q = 0; q < kRowsWaves - 1; ++q) acc += s_part[q][lane];
  // Lane: column t of the tile, 4 rows of W.
  out_t* __restrict__ C = static_cast<out_t*>(p.c);
  const int m = m0 + 4 * g;
  out_t v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) store_as(&v[e], acc[e]);
  if (p.token_major && m + 4 <= p.M) {
    __builtin_memcpy(C + t * p.ldc + m, v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (m + e < p.M) C[p.token_major ? t * p.ldc + m + e : (m + e) * p.ldc + t] = v[e];
  }
}

static void launch_rows(const Fp8MmParams& p, hipStream_t stream) {
  const dim3 grid((p.M + 15) / 16, (p.T + 15) / 16), block(64 * kRowsWaves);
  if (p.out_bf16) hipLaunchKernelGGL(fp8mm_rows_kernel<bf16_t>, grid, block, 0, stream, p);
  else hipLaunchKernelGGL(fp8mm_rows_kernel<float>, grid, block, 0, stream, p);
}

// ------------------------------------------------------------------------------ large products
// Both operands are "rows of K bytes", so the kernel is written for a row operand R, whose index
// runs along C's rows in memory, and a column operand Q: C[q * ldc + r]. R is X for a
// features-major C and W for a token-major one.
//
// A workgroup computes a kBR x kBQ tile. The operands' blocks of 128 features travel global ->
// LDS in two stages by direct copies (16 bytes a lane), one in flight while the other is
// multiplied. A row's 8 chunks of 16 bytes are stored at chunk ^ key(row), with keys that let the
// 16 rows of an operand read cover all banks. The wave's tiles of 16 R rows take every fourth
// group of 4 out of 64 rows, so that a lane ends up with 16 consecutive rows of a column and C
// leaves in 16-byte stores, whole 128-byte lines for a bf16 wave; they are not kept in the L2, which
// the operands need (130 us against 149 for 5120 x 1280 x 16384).
//
// What bounds that size: its parts alone take 80 us (the copies), 97 (LDS reads, products and sums
// of one block's data over and over) and about 35 (the stores, 168 MB), and the two workgroups of a
// CU overlap them in part.
__device__ __forceinline__ int r_key(int row) { return ((row >> 3) & 6) | ((row >> 1) & 1); }
__device__ __forceinline__ int q_key(int row) { return (row >> 1) & 7; }

template <int kBR_, int kBQ_, int kWR_, int kWQ_, int kParts_ = 1>
struct MmShape {
  // kParts: teams of kWaves waves that share a tile, each taking every kParts-th block of K.
  static constexpr int kBR = kBR_, kBQ = kBQ_, kWR = kWR_, kWQ = kWQ_, kWaves = kWR * kWQ, kThreads = 64 * kWaves;
  static constexpr int kParts = kParts_;
  static constexpr int kRT = kBR / kWR / 16, kQT = kBQ / kWQ / 16;  // 16 x 16 tiles of a wave
  static constexpr int kRCopies = kBR * 8 / kThreads, kQCopies = kBQ * 8 / kThreads;
  static_assert(kRT % 4 == 0 &&  kBR * 8 % kThreads == 0 &&
                kBQ * 8 % kThreads == 0, "");
};

typedef const __attribute__((address_space(4))) float* const_f32_t;

struct MmOperand {
  const unsigned char* base;
  long long ld;
  int rows;
};

template <typename S, bool kF8, typename out_t, bool kTokenRows>
__global__ __launch_bounds__(S::kThreads * S::kParts, 2) void fp8mm_tile_kernel(Fp8MmParams p, int tiles_r, int tiles_q) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host's pass knows no buffer resources
  constexpr int kToks = kTokenRows ? S::kBR : S::kBQ;
  // A stage: R's rows, Q's rows, the tokens' scales (copied 64 at a time).
  constexpr int kSlots = 8 * (S::kBR + S::kBQ) + (kToks < 64 ? 64 : kToks) / 4;
  __shared__ u32x4 s_even[S::kParts * kSlots], s_odd[S::kParts * kSlots];
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int part = S::kParts > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / S::kThreads) : 0;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) - part * S::kWaves;
  u32x4 *const s0 = s_even + part * kSlots, *const s1 = s_odd + part * kSlots;
  const int wr = wave % S::kWR, wq = wave / S::kWR;
  const MmOperand R = kTokenRows ? MmOperand{p.x, p.ldx, p.T} : MmOperand{p.w, p.ldw, p.M};
  const MmOperand Q = kTokenRows ? MmOperand{p.w, p.ldw, p.M} : MmOperand{p.x, p.ldx, p.T};
  const int nkb = (p.K + kFp8Block - 1) / kFp8Block;

  // Neighbouring tiles on one XCD: 8 of R by 4 of Q share their operands in its L2.
  int tr, tq;
  {
    const unsigned n = gridDim.x, per = n / 8, rem = n % 8, x = blockIdx.x % 8;
    const unsigned id = x * per + min(x, rem) + blockIdx.x / 8;
    const unsigned group = id / (8 * tiles_q), first = group * 8, wide = min(8u, tiles_r - first);
    const unsigned in = id - group * 8 * tiles_q;
    tr = first + in % wide;
    tq = in / wide;
  }
  const int r0 = tr * S::kBR, q0 = tq * S::kBQ;

  // Copy i of a stage: slots 64 i + lane, row slot / 8, stored chunk slot % 8. Rows past the
  // operand's end read its last row; their products are not stored.
  uint32_t off_r[S::kRCopies], off_q[S::kQCopies];
#pragma unroll
  for (int t = 0; t < S::kRCopies; ++t) {
    const int row = 8 * (wave + S::kWaves * t) + (lane >> 3);
    off_r[t] = static_cast<uint32_t>(min(row, R.rows - 1 - r0)) * static_cast<uint32_t>(R.ld) + 16 * ((lane & 7) ^ r_key(row));
  }
#pragma unroll
  for (int t = 0; t < S::kQCopies; ++t) {
    const int row = 8 * (wave + S::kWaves * t) + (lane >> 3);
    off_q[t] = static_cast<uint32_t>(min(row, Q.rows - 1 - q0)) * static_cast<uint32_t>(Q.ld) + 16 * ((lane & 7) ^ q_key(row));
  }
  const auto rsrc = [](const MmOperand& o, int first, int K) {
    const long long n = (o.rows - 1 - first) * o.ld + K;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(o.base + first * o.ld), 0,
                                             static_cast<uint32_t>(n < 0xffffffffll ? n : 0xffffffffll), 0x00027000);
  };
  const auto bufR = rsrc(R, r0, p.K), bufQ = rsrc(Q, q0, p.K);
  const int t0 = kTokenRows ? r0 : q0;
  const auto issue_scales = [&](int b, u32x4* d) {  // by every wave, some of them the same ones
    const int i = wave % ((kToks + 63) / 64);
    __builtin_amdgcn_global_load_lds((gbl_void_t)(p.xs + static_cast<long long>(b) * p.T + min(t0 + 64 * i + lane, p.T - 1)),
                                     (lds_void_t)(d + 8 * (S::kBR + S::kBQ) + 16 * i), 4, 0, 0);
  };
  const auto issue = [&](int b, u32x4* d) {
    issue_scales(b, d);
#pragma unroll
    for (int t = 0; t < S::kRCopies; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(bufR, (lds_void_t)(d + 64 * (wave + S::kWaves * t)), 16, off_r[t],
                                               b * kFp8Block, 0, 0);
#pragma unroll
    for (int t = 0; t < S::kQCopies; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(bufQ, (lds_void_t)(d + 8 * S::kBR + 64 * (wave + S::kWaves * t)), 16,
                                               off_q[t], b * kFp8Block, 0, 0);
  };

  // The wave's rows of W lie in one block.
  const int wrow = (kTokenRows ? q0 + wq * (16 * S::kQT) : r0 + wr * (16 * S::kRT)) / kFp8Block;
  static_assert(kFp8Block % (16 * (kTokenRows ? S::kQT : S::kRT)) == 0, "a wave's part of W lies in one block");
  // (constant address space: a scalar load, where a vector load would be waited for together with
  // the copies issued before it)
  const auto ws = reinterpret_cast<const_f32_t>(
      reinterpret_cast<uintptr_t>(p.ws + static_cast<long long>(min(wrow, (p.M - 1) / kFp8Block)) * nkb));

  f32x4 acc[S::kRT][S::kQT];
#pragma unroll
  for (int a = 0; a < S::kRT; ++a)
#pragma unroll
    for (int b = 0; b < S::kQT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

  // This lane's rows in the stages: of R, tile a at + 4 (a % 4) + 64 (a / 4) rows; of Q, tile c at
  // + 16 c rows. The keys are the same for all tiles.
  const int row_r = wr * (16 * S::kRT) + 16 * (j >> 2) + (j & 3), key_r = r_key(16 * (j >> 2) + (j & 3));
  const int row_q = wq * (16 * S::kQT) + j, key_q = q_key(j);
  const int r_lo = row_r * 8 + (g ^ key_r), r_hi = row_r * 8 + ((g + 4) ^ key_r);
  const int q_lo = row_q * 8 + (g ^ key_q), q_hi = row_q * 8 + ((g + 4) ^ key_q);
  const auto compute = [&](const u32x4* bR, float w) {
    const u32x4* bQ = bR + 8 * S::kBR;
    const float* bS = reinterpret_cast<const float*>(bQ + 8 * S::kBQ);
    MmFrag<kF8> r[S::kRT];
    f32x4 sr[kTokenRows ? S::kRT : 1];
#pragma unroll
    for (int a = 0; a < S::kRT; ++a) {
      const int at = 4 * (a & 3) + 64 * (a / 4);
      r[a].set(bR[r_lo + 8 * at], bR[r_hi + 8 * at]);
      if constexpr (kTokenRows) sr[a] = *reinterpret_cast<const f32x4*>(bS + wr * (16 * S::kRT) + 16 * g + at) * w;
    }
    // Products two by two; each pair is scaled and added while the next one is under way. The
    // empty asm statements and scheduler barriers keep it so: left alone, the sums move behind all
    // of the block's products, whose results then spill.
    constexpr int kPairs = S::kRT / 2;
    f32x4 d[2][2];
    float sq[2];
    MmFrag<kF8> q[2];
    const auto load_q = [&](int c) {
      q[c & 1].set(bQ[q_lo + 128 * c], bQ[q_hi + 128 * c]);
      if constexpr (!kTokenRows) sq[c & 1] = bS[row_q + 16 * c] * w;
    };
    const auto add = [&](int i) {
      const int c = i / kPairs;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int a = 2 * (i % kPairs) + h;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[a][c][e] = __builtin_fmaf(d[i & 1][h][e], kTokenRows ? sr[a][e] : sq[c & 1], acc[a][c][e]);
        asm volatile("" : "+v"(acc[a][c]));
      }
    };
    load_q(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < kPairs * S::kQT; ++i) {
      const int c = i / kPairs;
      if (i % kPairs == 1 && c + 1 < S::kQT) load_q(c + 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) d[i & 1][h] = mfma_block(r[2 * (i % kPairs) + h], q[c & 1]);
      __builtin_amdgcn_sched_barrier(0);
      if (i > 0) add(i - 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    add(kPairs * S::kQT - 1);
    __builtin_amdgcn_s_setprio(0);
  };

  const auto meet = [] {  // all waves' copies have landed and their reads are done
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0), the builtin so that the compiler knows too
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  const int full = p.K / kFp8Block;
  if (part < full) issue(part, s0);
  for (int first = 0; first < full; first += 2 * S::kParts) {  // (the teams meet equally often)
    const int b = first + part;
    meet();
    if (b + S::kParts < full) issue(b + S::kParts, s1);
    if (b < full) compute(s0, ws[b]);
    if (first + S::kParts >= full) break;
    meet();
    if (b + 2 * S::kParts < full) issue(b + 2 * S::kParts, s0);
    if (b + S::kParts < full) compute(s1, ws[b + S::kParts]);
  }
  if (full < nkb) {  // the features past K are zeros, whatever lies in the rows' padding
    const int k0 = full * kFp8Block;
    meet();
    if (part == 0) issue_scales(full, s0);
#pragma unroll 1
    for (int i = wave + S::kWaves * part; i < S::kBR / 8; i += S::kWaves * S::kParts) {  // all teams for the first one
      const int row = 8 * i + (lane >> 3);
      s_even[64 * i + lane] = load_chunk(R.base, R.ld, min(r0 + row, R.rows - 1), R.rows, k0 + 16 * ((lane & 7) ^ r_key(row)), p.K);
    }
#pragma unroll 1
    for (int i = wave + S::kWaves * part; i < S::kBQ / 8; i += S::kWaves * S::kParts) {
      const int row = 8 * i + (lane >> 3);
      s_even[8 * S::kBR + 64 * i + lane] =
          load_chunk(Q.base, Q.ld, min(q0 + row, Q.rows - 1), Q.rows, k0 + 16 * ((lane & 7) ^ q_key(row)), p.K);
    }
    meet();
    if (part == 0) compute(s0, ws[full]);
  }
  if constexpr (S::kParts > 1) {  // the teams' sums, in a fixed order
    constexpr int kSums = S::kRT * S::kQT * S::kThreads;
    static_assert(sizeof(s_even) >= (S::kParts - 1) * kSums * sizeof(f32x4), "");
    f32x4* const sums = reinterpret_cast<f32x4*>(s_even);
    meet();
    if (part > 0) {
#pragma unroll
      for (int i = 0; i < S::kRT * S::kQT; ++i)
        sums[(part - 1) * kSums + i * S::kThreads + 64 * wave + lane] = acc[i / S::kQT][i % S::kQT];
    }
    meet();
    if (part > 0) return;
#pragma unroll
    for (int q = 0; q + 1 < S::kParts; ++q)
#pragma unroll
      for (int i = 0; i < S::kRT * S::kQT; ++i)
        acc[i / S::kQT][i % S::kQT] += sums[q * kSums + i * S::kThreads + 64 * wave + lane];
  }

  // A lane's 16 rows of a column.
  out_t* __restrict__ C = static_cast<out_t*>(p.c);
#pragma unroll
  for (int c = 0; c < S::kQT; ++c) {
    const int q = q0 + wq * (16 * S::kQT) + 16 * c + j;
    if (q >= Q.rows) continue;
#pragma unroll
    for (int h = 0; h < S::kRT / 4; ++h) {
      const int r = r0 + wr * (16 * S::kRT) + 64 * h + 16 * g;
      out_t* __restrict__ dst = C + q * p.ldc + r;
      alignas(16) out_t v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) store_as(&v[e], acc[4 * h + e / 4][c][e % 4]);
      if (r + 16 <= R.rows) {
#pragma unroll
        for (int e = 0; e < static_cast<int>(sizeof(v) / 16); ++e)
          __builtin_nontemporal_store(reinterpret_cast<const u32x4*>(v)[e], reinterpret_cast<u32x4_any*>(dst) + e);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (r + e < R.rows) dst[e] = v[e];
      }
    }
  }
#endif
}

template <typename S, bool kF8, typename out_t, bool kBothLayouts = true>
static void launch_tiles(const Fp8MmParams& p, hipStream_t stream) {
  const int nr = p.token_major ? p.M : p.T, nq = p.token_major ? p.T : p.M;
  const int tr = (nr + S::kBR - 1) / S::kBR, tq = (nq + S::kBQ - 1) / S::kBQ;
  const dim3 grid(tr * tq), threads(S::kThreads * S::kParts);
  if constexpr (kBothLayouts) {
    if (!p.token_major) {
      hipLaunchKernelGGL((fp8mm_tile_kernel<S, kF8, out_t, true>), grid, threads, 0, stream, p, tr, tq);
      return;
    }
  }
  hipLaunchKernelGGL((fp8mm_tile_kernel<S, kF8, out_t, false>), grid, threads, 0, stream, p, tr, tq);
}

// 128 x 128 tiles, four waves of 64 x 64, two workgroups a CU, whose copies, products and stores
// fall at different times. (256 x 256 tiles of eight waves, one workgroup a CU: 139 us against 130
// for 5120 x 1280 x 16384, 139 against 115 for 5120 x 5120 x 4096.) 64 x 64 tiles, four waves of
// 64 x 16, four workgroups a CU, where there are fewer than 256 of the large ones, and for all float32
// outputs. Where they are few: four teams of two waves, each with a quarter of the blocks of K and its
// own copies in flight, on tiles of 64 x 32 if that makes no more than one a CU, else on 64 x 64.
// (us, one team of four waves, two, four of two, the same on 64 x 32: 1280 x 2560 x 333 10.4, 8.9, 8.2,
// 6.7; x 128 9.6, 8.1, 7.1, 5.9; 768 x 1536 x 512 6.9, 6.2, 5.8, 5.0; 2560 x 1280 x 256 6.3, 5.8, 5.6,
// and 7.9 with 320 tiles; x 512, 320 tiles of 64, 7.2, 7.5, 9.4. One team with a ring of three or four
// stages: 11.8, 11.2 for the first.) Up to 32 tokens in rows of their own: one team of two waves on
// 64 x 32, where fewer rows of tokens that are not there are copied (50280 x 768 x 8 in float32 11.1 us on 64 x 64,
// 9.0; x 32 12.6, 12.0; 32000 x 2048 x 8 13.7, 12.3).
typedef MmShape<128, 128, 2, 2> MmLarge;
typedef MmShape<64, 64, 1, 4> MmSmall;
typedef MmShape<64, 64, 1, 2, 4> MmTeams;
typedef MmShape<64, 32, 1, 2, 4> MmFew;
typedef MmShape<64, 32, 1, 2> MmThin;

// Which kernel: the one whose time, by the sums below, is less. Rows: what the workgroups read, or
// their number where they have little to read, and a wave's blocks one after the other. Tiles: the
// blocks of K one after the other, a block's time by how many tiles share a CU; a block that is
// not whole comes last and unstaged. (Teams split a block's time.) Measured (us, M x K x T: rows, tiles of 64, tiles of 128):
//   5120 x 1280 x 1         3.8     -     -      1280 x 2560 x 333    19.0   6.7  17.5
//   5120 x 1280 x 8         4.1   4.8     -      5120 x 1280 x 1024    108  15.1  12.4
//   50280 x 768 x 8 (f32)  12.8   9.0     -      1280 x 2560 x 2048   94.3  14.2  17.5
//   1280 x 2560 x 64        7.0   5.9  17.0      5120 x 1280 x 16384     -   182   130
//   64 x 64 x 16384        13.4   4.1     -      the same (f32)          -   307   356
// 130 us are 1.65 PFLOP/s; the library's product with one scale an operand reaches 3.0 at 8192^3.
// (A launch has fewer than 2^32 threads along x: M beyond 2^26 takes another one, a whole number of W's
// blocks further on.)
constexpr int kMmLaunchRows = 1 << 26;

hipError_t launch_fp8mm(const Fp8MmParams& p, hipStream_t stream) {
  if (p.M > kMmLaunchRows) {
    Fp8MmParams part = p;
    for (long long m = 0; m < p.M; m += kMmLaunchRows) {
      part.M = static_cast<int>(p.M - m < kMmLaunchRows ? p.M - m : kMmLaunchRows);
      part.w = p.w + m * p.ldw;
      part.ws = p.ws + m / kFp8Block * ((p.K + kFp8Block - 1) / kFp8Block);
      part.c = static_cast<char*>(p.c) + (p.token_major ? m : m * p.ldc) * (p.out_bf16 ? 2 : 4);
      const hipError_t e = launch_fp8mm(part, stream);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }
  const double nkb = (p.K + kFp8Block - 1) / kFp8Block;
  const auto tiles = [&](double n) { return __builtin_ceil(p.M / n) * __builtin_ceil(p.T / n); };
  const double rows = 2.5 + fmax(0.00044 * tiles(16) * nkb, 0.0026 * tiles(16)) + 0.09 * nkb;
  const double few_tiles = p.token_major ? __builtin_ceil(p.M / 64.) * __builtin_ceil(p.T / 32.)
                                         : __builtin_ceil(p.T / 64.) * __builtin_ceil(p.M / 32.);
  const bool few = few_tiles <= 256, thin = p.token_major && p.T <= 32;
  const bool teams = tiles(64) <= 256 && nkb >= 8;
  double block, start = 2;  // of the tiles
  if (few) {
    start = 3.5;
    block = p.out_bf16 ? 0.12 + 0.0002 * few_tiles : 0.16 + 0.0004 * few_tiles;
  } else {
    block = p.out_bf16 ? fmax(0.38, 0.0009 * tiles(64)) : fmax(0.55, 0.0015 * tiles(64));
  }
  const double staged = start + block * nkb + (p.K % kFp8Block ? (few ? 1.2 : 3) : 0);
  // the tiles' offsets and their number have 32 bits
  const bool far = p.ldw >= 1 << 24 || p.ldx >= 1 << 24 || tiles(64) > 2e9;
  if (far || rows < staged) launch_rows(p, stream);
  else if (few && p.out_bf16) launch_tiles<MmFew, true, bf16_t>(p, stream);
  else if (few) launch_tiles<MmFew, false, float>(p, stream);
  else if (thin && p.out_bf16) launch_tiles<MmThin, true, bf16_t, false>(p, stream);
  else if (thin) launch_tiles<MmThin, false, float, false>(p, stream);
  else if (teams && p.out_bf16) launch_tiles<MmTeams, true, bf16_t>(p, stream);
  else if (teams) launch_tiles<MmTeams, false, float>(p, stream);
  else if (!p.out_bf16) launch_tiles<MmSmall, false, float>(p, stream);
  else if (tiles(128) < 256) launch_tiles<MmSmall, true, bf16_t>(p, stream);
  else launch_tiles<MmLarge, true, bf16_t>(p, stream);
  return hipGetLastError();
}

}  // namespace mss
