// Activations and weights in 8 bits (e4m3) with block scales, and the residual add + RMSNorm
// that writes its output that way.
//
//   y[f][t]  = x[f][t], or with the norm in front: hn = h + delta, r_t = 1 / sqrt(mean_f hn^2 +
//              eps), y = hn r_t w[f]   (reference mamba/mamba1.py:300-337: nnx.RMSNorm before
//              the in-projections, the block's output added back)
//   s[b][t]  = max(max_{f in block b} |y[f][t]| / 448, 2^-126)
//   q[t][f]  = e4m3(448 y[f][t] / max_{f in block b} |y[f][t]|), or of y 2^126 at the least scale, rounded
//              to nearest even
//
// The stream is channel-major (features, tokens) and a matrix-core product wants 8-bit operands
// with the features contiguous, so these kernels also transpose: a workgroup owns a tile of
// tokens, a thread 4 to 8 neighbouring tokens of 4 features, whose bytes it packs into a dword of
// each token's row in LDS; the rows leave as 16-byte stores. y and the norm's sums are float32;
// q is the only rounding to fewer bits.
#include <hip/hip_runtime.h>

#include "mss_serve.h"

namespace mss {

// Values over a block's scale. The scale itself is rounded; q is not taken from it but from the
// block's largest magnitude, y * (448 / m) with the factor in two parts: bf16 values meet e4m3's borders
// exactly (y / m = 3 / 64, for one, is 21, between 20 and 22), and a quotient that is off by one
// float32 step there rounds the wrong way.
struct Ratio448 {  // y -> 448 y / amax
  float hi, lo;
  __device__ __forceinline__ explicit Ratio448(float amax) {
    hi = kFp8Max / amax;
    lo = __builtin_fmaf(-hi, amax, kFp8Max) * (hi * (1.f / kFp8Max));
  }
  __device__ __forceinline__ float operator()(float y) const { return __builtin_fmaf(y, hi, y * lo); }
};
struct ToFp8 {
  float scale;
  Ratio448 by;
  __device__ __forceinline__ explicit ToFp8(uint32_t m) : scale(fp8_scale(__uint_as_float(m))), by(__uint_as_float(m)) {
    if (__uint_as_float(m) < kFp8Max * 1.1754943508222875e-38f) {  // the least scale, 2^-126
      by.hi = 8.507059173023462e37f;
      by.lo = 0.f;
    }
  }
  __device__ __forceinline__ float operator()(float y) const { return by(y); }
};

// v and the values kLanes away (32, 16, 2, 1: the lane whose index differs there; 8, 4: the lane that
// far round in a row of 16, so that after both a value has met its three fellows), for all lanes, by
// `op`: register moves, where a shuffle goes through LDS.
template <int kLanes, typename op_t>
__device__ __forceinline__ uint32_t across(uint32_t v, const op_t& op) {
  if constexpr (kLanes == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return op(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
  } else if constexpr (kLanes == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return op(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
  } else {
    constexpr int kCtrl = kLanes == 8 ? 0x128 : kLanes == 4 ? 0x124 : kLanes == 2 ? 0x4E : 0xB1;  // row_ror, quad_perm
    return op(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xF, 0xF, true)));
  }
}
// The same over every lane whose index differs above kFrom - 1 and below kTo (all of 4 and 8, or neither).
template <int kFrom, int kTo = 64, typename op_t>
__device__ __forceinline__ uint32_t across_all(uint32_t v, const op_t& op) {
  if constexpr (kFrom < kTo) return across_all<2 * kFrom, kTo>(across<kFrom>(v, op), op);
  return v;
}
template <int kFrom, int kTo = 64>
__device__ __forceinline__ uint32_t max_above(uint32_t v) {
  return across_all<kFrom, kTo>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int kFrom>
__device__ __forceinline__ float sum_above(float v) {
  return __uint_as_float(across_all<kFrom>(
      __float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

// 16 bytes of a token's row from LDS (8-byte aligned there) to the features f .. f + 16 of q.
__device__ __forceinline__ void store_row16(unsigned char* __restrict__ q, const uint32_t* __restrict__ src, int f, int F) {
  if (f >= F) return;
  const uint2 a = reinterpret_cast<const uint2*>(src)[0], b = reinterpret_cast<const uint2*>(src)[1];
  if (f + 16 <= F) {
    *reinterpret_cast<u32x4*>(q) = u32x4{a.x, a.y, b.x, b.y};
  } else {
    const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (f + i < F) q[i] = static_cast<unsigned char>(w[i / 4] >> (8 * (i & 3)));
  }
}

// --------------------------------------------------------------- quantisation, token-contiguous
// A workgroup: one block of features, 64 tokens (of 64 or more). A thread holds 16 bytes (kTV tokens) of 4
// features; a feature's 64 tokens are one 128- or 256-byte read.
template <typename io_t>
__global__ __launch_bounds__(128 * sizeof(io_t)) void quant_tile_kernel(QuantParams p) {
  constexpr int kTV = 16 / sizeof(io_t), kLanes = 64 / kTV, kWaves = 2 * sizeof(io_t);
  constexpr int kPitch = kFp8Block / 4 + 2;  // dwords of a row in LDS: 8-byte aligned, and rows shift banks
  __shared__ uint32_t s_m[kWaves][64];
  __shared__ alignas(8) uint32_t s_q[64 * kPitch];
  const int l = threadIdx.x % kLanes, g = threadIdx.x / kLanes, wave = threadIdx.x / 64;
  long long t0 = blockIdx.x * 64ll;
  if (t0 + 64 > p.tokens) t0 = p.tokens - 64;  // the last tile, whole: some tokens come out twice
  const int b = blockIdx.y, f0 = b * kFp8Block + 4 * g;
  const long long t = t0 + l * kTV;
  const io_t* __restrict__ x = static_cast<const io_t*>(p.x) + t;
  float v[4][kTV];
  {
    io_t raw[4][kTV];
#pragma unroll
    for (int i = 0; i < 4; ++i) __builtin_memcpy(raw[i], x + min(f0 + i, p.features - 1) * p.sf, sizeof(raw[i]));
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kTV; ++j) v[i][j] = f0 + i < p.features ? to_f32(raw[i][j]) : 0.f;
  }
#pragma unroll
  for (int j = 0; j < kTV; ++j) {
    uint32_t m = max(max(magnitude_bits(v[0][j]), magnitude_bits(v[1][j])),
                     max(magnitude_bits(v[2][j]), magnitude_bits(v[3][j])));
    m = max_above<kLanes>(m);
    if ((threadIdx.x & 63) < kLanes) s_m[wave][l * kTV + j] = m;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kTV; ++j) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) m = max(m, s_m[i][l * kTV + j]);
    const ToFp8 to(m);
    if (g == 0) p.scales[static_cast<long long>(b) * p.tokens + t + j] = to.scale;
    s_q[(l * kTV + j) * kPitch + g] = pack_fp8x4(to(v[0][j]), to(v[1][j]), to(v[2][j]), to(v[3][j]));
  }
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < 64 * (kFp8Block / 16); i += 64 * kWaves) {
    const int row = i / (kFp8Block / 16), c = i % (kFp8Block / 16);
    store_row16(p.q + (t0 + row) * p.ldq + b * kFp8Block + 16 * c, s_q + row * kPitch + 4 * c, b * kFp8Block + 16 * c,
                p.features);
  }
}

// ------------------------------------------------------------------ any strides, or few tokens
// 16 lanes hold one token's block, 8 features each; a wave covers 4 tokens.
template <typename io_t, bool kVec>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantParams p) {
  const int lane = threadIdx.x & 15;
  const long long t = blockIdx.x * 16ll + (threadIdx.x >> 4);
  const int b = blockIdx.y;
  const int f0 = b * kFp8Block + lane * 8;
  const bool ok = t < p.tokens;
  const io_t* __restrict__ x = static_cast<const io_t*>(p.x) + (ok ? t : 0) * p.st;
  float v[8];
  if (kVec && f0 + 8 <= p.features) {
    union {
      u32x4 w[sizeof(io_t) / 2];
      io_t e[8];
    } u;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(io_t) / 2); ++i)
      u.w[i] = reinterpret_cast<const u32x4*>(x + f0)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(u.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f0 + i < p.features ? to_f32(x[(f0 + i) * p.sf]) : 0.f;
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, magnitude_bits(v[i]));
#pragma unroll
  for (int s = 1; s < 16; s *= 2) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), s)));
  const ToFp8 to(m);
  if (!ok) return;
  if (lane == 0) p.scales[static_cast<long long>(b) * p.tokens + t] = to.scale;
  // A row of q is 16-byte aligned and holds at least ceil16(features) bytes up to the next row;
  // the last row's end is the tensor's, so the bytes past the features are not touched.
  unsigned char* q = p.q + t * p.ldq + f0;
  const uint32_t lo = pack_fp8x4(to(v[0]), to(v[1]), to(v[2]), to(v[3]));
  const uint32_t hi = pack_fp8x4(to(v[4]), to(v[5]), to(v[6]), to(v[7]));
  if (f0 + 8 <= p.features) {
    *reinterpret_cast<uint2*>(q) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (f0 + i < p.features) q[i] = static_cast<unsigned char>((i < 4 ? lo : hi) >> (8 * (i & 3)));
  }
}

// --------------------------------------------------------------------------------- weights
// A workgroup owns one 128 x 128 block; a wave reads 256 or 512 contiguous bytes of a row.
template <typename io_t>
__global__ __launch_bounds__(256) void quant_weight_kernel(QuantWeightParams p) {
  __shared__ uint32_t s_m[4];
  const int c = (threadIdx.x & 63) * 2;
  const int k = blockIdx.x * kFp8Block + c;
  const int row0 = blockIdx.y * kFp8Block + (threadIdx.x >> 6);
  const io_t* __restrict__ w = static_cast<const io_t*>(p.w);
  float v[32][2];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int r = row0 + 4 * i;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      v[i][j] = r < p.M && k + j < p.K ? to_f32(w[r * p.ldw + k + j]) : 0.f;
      m = max(m, magnitude_bits(v[i][j]));
    }
  }
#pragma unroll
  for (int s = 1; s < 64; s *= 2) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), s)));
  if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(s_m[0], s_m[1]), max(s_m[2], s_m[3]));
  const ToFp8 to(m);
  if (threadIdx.x == 0) p.scales[static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x] = to.scale;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int r = row0 + 4 * i;
    if (r >= p.M || k >= p.K) continue;
    const uint32_t two = pack_fp8x4(to(v[i][0]), to(v[i][1]), 0.f, 0.f);
    unsigned char* q = p.q + r * p.ldq + k;  // k even, rows 16-byte aligned
    if (k + 1 < p.K) *reinterpret_cast<uint16_t*>(q) = static_cast<uint16_t>(two);
    else *q = static_cast<unsigned char>(two);
  }
}

// ------------------------------------------------------------------ residual add + norm
// The norm's factor r_t is the same for a token's whole block, so it drops out of q = y / s:
// with y' = hn w and m' = max |y'| over the block, q = e4m3(448 y' / m') and s = r m' / 448. So
// q needs no second pass over the features: each block leaves as it is read, and the scales,
// kept in LDS until the sum of squares is whole, are the only thing that waits for r. That is
// also one rounding less than hn r w. Where it does not hold (m' far below 1, m' or m' r not finite,
// or a scale at its lower bound) the block is done again from the formula.
__device__ __forceinline__ bool scale_is_plain(float m, float r) {
  return m == 0.f || (m > 7.9e-31f && m * r < __builtin_inff() && !(m * r < kFp8Max * 1.1754943508222875e-38f));
}

// One block of one token from the formula, by one thread: its scale.
__device__ __noinline__ float norm_block_again(const float* __restrict__ hn, const float* __restrict__ w, long long T,
                                               float r, int n, unsigned char* __restrict__ q) {
  uint32_t m = 0;
  for (int i = 0; i < n; ++i) m = max(m, magnitude_bits(hn[i * T] * r * w[i]));
  const ToFp8 to(m);
  for (int i = 0; i < n; ++i) q[i] = static_cast<unsigned char>(pack_fp8x4(to(hn[i * T] * r * w[i]), 0.f, 0.f, 0.f));
  return to.scale;
}

// Four neighbouring values as they lie in memory, of any alignment.
template <typename T>
struct Run4;
template <>
struct Run4<float> {
  f32x4 v;
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const f32x4_any*>(p); }
  __device__ __forceinline__ void set(int j, float x) { v[j] = x; }
  __device__ __forceinline__ float get(int j) const { return v[j]; }
};
template <>
struct Run4<bf16_t> {
  uint32_t v[2];
  __device__ __forceinline__ void load(const bf16_t* p) {
    const u32x2_any x = *reinterpret_cast<const u32x2_any*>(p);
    v[0] = x[0];
    v[1] = x[1];
  }
  __device__ __forceinline__ void set(int j, bf16_t x) {
    v[j / 2] = j % 2 ? (v[j / 2] & 0xffffu) | static_cast<uint32_t>(x.bits) << 16 : x.bits;
  }
  __device__ __forceinline__ float get(int j) const {
    return __uint_as_float(j % 2 ? v[j / 2] & 0xffff0000u : v[j / 2] << 16);
  }
};

// A workgroup owns 4 kL tokens and walks the features, kRound of them at a time: kL lanes hold a
// row of 4 tokens each, a thread 4 consecutive features. The next round's rows are on their way
// while a round is worked on (bare barriers: __syncthreads would wait for them).
constexpr int kNormMaxBlocks = 64;  // of a token, whose maxima wait in LDS

__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Workgroups go to the 8 XCDs in turn, and each has an L2 of its own: neighbouring tiles, which
// share cache lines, are given to one XCD.
__device__ __forceinline__ unsigned tile_of_xcd(unsigned id, unsigned n) {
  const unsigned per = n / 8, rem = n % 8, x = id % 8;
  return x * per + min(x, rem) + id / 8;
}

template <typename delta_t, bool kDelta, int kL, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void norm_fp8_tile_kernel(QuantParams p) {
  constexpr int kTok = 4 * kL, kGroups = 64 * kWaves / kL, kRound = 4 * kGroups;
  constexpr int kBlockWaves = kL / 2;  // waves that hold one block: 32 groups of kL lanes
  constexpr int kPitch = kRound / 4 + 2;
  static_assert(kRound % kFp8Block == 0 && kBlockWaves >= 1, "whole blocks and waves");
  __shared__ uint32_t s_m[kWaves][kTok];
  __shared__ alignas(8) uint32_t s_q[kTok * kPitch];
  __shared__ float s_block[kNormMaxBlocks][kTok];
  __shared__ float s_ss[kWaves][kTok];
  __shared__ int s_again;
  const int l = threadIdx.x % kL, g = threadIdx.x / kL;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const long long T = p.tokens;
  // The last tile begins earlier rather than be cut: its first tokens come out the same twice. (Not
  // in place, where they would be added to twice.)
  long long t0 = static_cast<long long>(tile_of_xcd(blockIdx.x, gridDim.x)) * kTok;
  if (t0 + kTok > T && T >= kTok && (!kDelta || p.hn != p.x)) t0 = T - kTok;
  const long long t = t0 + 4 * l;
  const int F = p.features;
  const bool whole = t + 4 <= T;
  const float* __restrict__ h = static_cast<const float*>(p.x) + t;
  const delta_t* __restrict__ delta = static_cast<const delta_t*>(p.delta) + t;

  // (raw vectors, the deltas converted where they are used, and one branch around all loads: they
  // are in flight together)
  f32x4 hv[4];
  float wv[4];
  Run4<delta_t> dv[4];
  const bool whole_tile = t0 + kTok <= T;
  const auto fetch = [&](int f0) {
    if (whole_tile) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = min(f0 + i, F - 1);
        wv[i] = p.w[f];
        hv[i] = *reinterpret_cast<const f32x4_any*>(h + f * T);
        if constexpr (kDelta) dv[i].load(delta + f * T);
      }
    } else {
      asm volatile("");  // else the compiler takes the single loads for both
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int f = min(f0 + i, F - 1);
        wv[i] = p.w[f];
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // (tokens past the end: the last one again, its results unused)
          const long long o = f * T + min(static_cast<long long>(j), T - 1 - t);
          hv[i][j] = h[o];
          if constexpr (kDelta) dv[i].set(j, delta[o]);
        }
      }
    }
  };
  float ss[4] = {0.f, 0.f, 0.f, 0.f};
  fetch(4 * g);
  for (int f0 = 4 * g; f0 - 4 * g < F; f0 += kRound) {
    float y[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = f0 + i < F;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = kDelta ? hv[i][j] + dv[i].get(j) : hv[i][j];
        y[i][j] = in ? x : 0.f;
        ss[j] = __builtin_fmaf(y[i][j], y[i][j], ss[j]);
      }
      if constexpr (kDelta) {
        if (in) {
          float* o = p.hn + (f0 + i) * T + t;
          if (whole) {
            __builtin_memcpy(o, y[i], 16);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (t + j < T) o[j] = y[i][j];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) y[i][j] *= wv[i];
    }
    if (f0 - 4 * g + kRound < F) fetch(f0 + kRound);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t m = max(max(magnitude_bits(y[0][j]), magnitude_bits(y[1][j])),
                       max(magnitude_bits(y[2][j]), magnitude_bits(y[3][j])));
      m = max_above<kL>(m);
      if ((threadIdx.x & 63) < kL) s_m[wave][4 * l + j] = m;
    }
    meet();
    const int b = f0 / kFp8Block;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < kBlockWaves; ++i) m = max(m, s_m[wave / kBlockWaves * kBlockWaves + i][4 * l + j]);
      const float mf = __uint_as_float(m);
      if (g % 32 == 0 && b < kNormMaxBlocks) s_block[b][4 * l + j] = mf;
      const Ratio448 to(m ? mf : 1.f);
      s_q[(4 * l + j) * kPitch + g] = pack_fp8x4(to(y[0][j]), to(y[1][j]), to(y[2][j]), to(y[3][j]));
    }
    meet();
    // 16 bytes of the tile each
    const int row = threadIdx.x / (kRound / 16), c = threadIdx.x % (kRound / 16), f = f0 - 4 * g + 16 * c;
    if (t0 + row < T) store_row16(p.q + (t0 + row) * p.ldq + f, s_q + row * kPitch + 4 * c, f, F);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float s = sum_above<kL>(ss[j]);
    if ((threadIdx.x & 63) < kL) s_ss[wave][4 * l + j] = s;
  }
  if (threadIdx.x == 0) s_again = 0;
  meet();
  const int nb = (F + kFp8Block - 1) / kFp8Block;
  for (int i = threadIdx.x; i < nb * kTok; i += 64 * kWaves) {
    const int b = i / kTok, j = i % kTok;
    if (t0 + j >= T) continue;
    float tot = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) tot += s_ss[k][j];
    const float r = 1.f / __builtin_sqrtf(tot / F + p.eps);
    const float m = s_block[b][j];
    if (scale_is_plain(m, r)) p.scales[b * T + t0 + j] = fp8_scale(m * r);
    else s_again = 1;
  }
  meet();
  if (s_again == 0) return;
  __syncthreads();  // hn and q of this tile are written
  for (int i = threadIdx.x; i < nb * kTok; i += 64 * kWaves) {
    const int b = i / kTok, j = i % kTok, f = b * kFp8Block;
    if (t0 + j >= T) continue;
    float tot = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) tot += s_ss[k][j];
    const float r = 1.f / __builtin_sqrtf(tot / F + p.eps);
    if (!scale_is_plain(s_block[b][j], r))
      p.scales[b * T + t0 + j] =
          norm_block_again((kDelta ? p.hn : static_cast<const float*>(p.x)) + f * T + t0 + j, p.w + f, T, r,
                           min(kFp8Block, F - f), p.q + (t0 + j) * p.ldq + f);
  }
}

// Few tokens: one a workgroup, a feature a lane (neighbouring features of a few tokens share cache
// lines), kRounds x 512 of them in registers; q by the blocks' maxima before the norm, as above.
// (1280 x 8: 5.7 us with the features read twice, 4.6 with four neighbours a lane.)
template <typename delta_t, bool kDelta, int kRounds>
__global__ __launch_bounds__(512) void norm_fp8_rows_kernel(QuantParams p) {
  __shared__ float s_ss[8];
  __shared__ uint32_t s_m[kRounds][8];
  const long long T = p.tokens, t = blockIdx.x;
  const int F = p.features, wave = threadIdx.x >> 6;
  const float* __restrict__ h = static_cast<const float*>(p.x) + t;
  const delta_t* __restrict__ delta = static_cast<const delta_t*>(p.delta) + t;
  float x[kRounds], d[kRounds], w[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int f = min(512 * k + static_cast<int>(threadIdx.x), F - 1);
    x[k] = h[f * T];
    if constexpr (kDelta) d[k] = to_f32(delta[f * T]);
    w[k] = p.w[f];
  }
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const bool in = 512 * k + static_cast<int>(threadIdx.x) < F;
    if constexpr (kDelta) x[k] += d[k];
    const float sq = in ? x[k] : 0.f;  // (both factors: the last feature again may be infinite)
    ss = __builtin_fmaf(sq, sq, ss);
    w[k] *= x[k];  // y' = hn w
    const uint32_t m = max_above<1>(in ? magnitude_bits(w[k]) : 0u);
    if ((threadIdx.x & 63) == 0) s_m[k][wave] = m;
  }
  ss = wave_sum(ss);
  if ((threadIdx.x & 63) == 0) s_ss[wave] = ss;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int f = 512 * k + threadIdx.x;
    if (f < F) {
      const uint32_t m = max(s_m[k][wave], s_m[k][wave ^ 1]);
      const Ratio448 to(m ? __uint_as_float(m) : 1.f);
      p.q[t * p.ldq + f] = static_cast<unsigned char>(pack_fp8x4(to(w[k]), 0.f, 0.f, 0.f));
      if constexpr (kDelta) p.hn[f * T + t] = x[k];
    }
  }
  const int nb = (F + kFp8Block - 1) / kFp8Block;
  float tot = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) tot += s_ss[i];
  const float r = 1.f / __builtin_sqrtf(tot / F + p.eps);
  float m = 0.f;
  bool plain = true;
  if (static_cast<int>(threadIdx.x) < nb) {  // a block a lane
    const int b = threadIdx.x;
    m = __uint_as_float(max(s_m[b / 4][2 * (b % 4)], s_m[b / 4][2 * (b % 4) + 1]));
    plain = scale_is_plain(m, r);
    if (plain) p.scales[b * T + t] = fp8_scale(m * r);
  }
  if (__syncthreads_or(plain ? 0 : 1)) {
    __syncthreads();  // hn and q of this token are written
    if (!plain) {
      const int b = threadIdx.x, f = b * kFp8Block;
      p.scales[b * T + t] =
          norm_block_again((kDelta ? p.hn : static_cast<const float*>(p.x)) + f * T + t, p.w + f, T, r,
                           min(kFp8Block, F - f), p.q + t * p.ldq + f);
    }
  }
}

// More features than registers hold or the tiles take: two passes over a token's column, 32 lanes to
// a block, 4 consecutive features each.
template <typename delta_t, bool kDelta>
__global__ __launch_bounds__(512) void norm_fp8_wide_kernel(QuantParams p) {
  __shared__ float s_part[8];
  const long long T = p.tokens, t = blockIdx.x;
  const float* __restrict__ h = static_cast<const float*>(p.x) + t;
  const delta_t* __restrict__ delta = static_cast<const delta_t*>(p.delta) + t;
  float ss = 0.f;
  for (int f = threadIdx.x; f < p.features; f += 512) {
    float v = h[f * T];
    if constexpr (kDelta) v += to_f32(delta[f * T]);
    ss = __builtin_fmaf(v, v, ss);
  }
  ss = wave_sum(ss);
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = ss;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) tot += s_part[i];
  const float r = 1.f / __builtin_sqrtf(tot / p.features + p.eps);
  const int padded = (p.features + kFp8Block - 1) / kFp8Block * kFp8Block;
  for (int f0 = threadIdx.x * 4; f0 < padded; f0 += 2048) {
    float v[4], y[4];  // y' = hn w, and hn r w
    uint32_t m = 0, my = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int f = f0 + i;
      v[i] = y[i] = 0.f;
      if (f < p.features) {
        float x = h[f * T];
        if constexpr (kDelta) {
          x += to_f32(delta[f * T]);
          p.hn[f * T + t] = x;
        }
        v[i] = x * p.w[f];
        y[i] = x * r * p.w[f];
      }
      m = max(m, magnitude_bits(v[i]));
      my = max(my, magnitude_bits(y[i]));
    }
    m = max_above<1, 32>(m);
    my = max_above<1, 32>(my);
    const float mf = __uint_as_float(m);
    const bool plain = scale_is_plain(mf, r);
    const ToFp8 to(my);
    const Ratio448 by(m ? mf : 1.f);
    if ((threadIdx.x & 31) == 0) p.scales[(f0 / kFp8Block) * T + t] = plain ? fp8_scale(mf * r) : to.scale;
    const uint32_t q4 = plain ? pack_fp8x4(by(v[0]), by(v[1]), by(v[2]), by(v[3]))
                              : pack_fp8x4(to(y[0]), to(y[1]), to(y[2]), to(y[3]));
    unsigned char* q = p.q + t * p.ldq + f0;
    if (f0 + 4 <= p.features) {
      *reinterpret_cast<uint32_t*>(q) = q4;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (f0 + i < p.features) q[i] = static_cast<unsigned char>(q4 >> (8 * i));
    }
  }
}

// --------------------------------------------------------------------------------- launches
// Where each kernel starts to win (MI355X, us for features x tokens).
// quant: rows while a workgroup of them for each CU (float32) or two (bf16) hold all tokens, and for fewer
// than 64; rows/tile, bf16: 768 x 400 3.5/4.3, 2560 x 64 3.4/4.3, x 400 4.3/4.5, 5120 x 128 4.0/4.3, x 200
// 5.0/4.4, x 400 6.4/5.3; float32: 768 x 400 3.2/3.5, 2560 x 128 3.2/3.4, x 200 4.0/3.5, 5120 x 128 4.0/3.5.
// 2560 x 16384 bf16: rows 81, tiles 24.2, at the rate of a copy (5.2 TB/s).
constexpr int kQuantTileTokens = 64;
// norm, bf16 delta: a token a workgroup 1280 x 128 6.0, x 256 9.0, x 512 13.8; tiles of 8 tokens x 256
// 8.9, x 512 9.5, x 2048 12.6, x 4096 20; of 16 tokens x 2048 13.3, x 4096 15.4, x 8192 23.5, x 16384 58;
// of 32 tokens x 4096 17, x 8192 22, x 16384 45: 5.1 TB/s.
constexpr int kNormTileTokens = 256;
constexpr int kNormNarrowTokens = 2048;
constexpr int kNormMiddleTokens = 6144;

template <typename io_t>
static void launch_quant(const QuantParams& p, hipStream_t stream) {
  const unsigned blocks = (p.features + kFp8Block - 1) / kFp8Block;
  const long long rows = (p.tokens + 15ll) / 16 * blocks;  // workgroups
  if (p.st == 1 && p.tokens >= kQuantTileTokens && rows > (sizeof(io_t) == 2 ? 512 : 256)) {
    hipLaunchKernelGGL((quant_tile_kernel<io_t>), dim3((p.tokens + 63) / 64, blocks), dim3(128 * sizeof(io_t)), 0, stream, p);
    return;
  }
  const dim3 grid((p.tokens + 15) / 16, blocks);
  // 16-byte loads where a token's features are contiguous and its row starts on 16 bytes.
  const bool vec = p.sf == 1 && (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 &&
                   (p.st * static_cast<long long>(sizeof(io_t))) % 16 == 0;
  if (vec) hipLaunchKernelGGL((quant_rows_kernel<io_t, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((quant_rows_kernel<io_t, false>), grid, dim3(256), 0, stream, p);
}

hipError_t launch_quant_fp8(const QuantParams& p, bool io_bf16, hipStream_t stream) {
  if (io_bf16) launch_quant<bf16_t>(p, stream);
  else launch_quant<float>(p, stream);
  return hipGetLastError();
}

hipError_t launch_quant_fp8_weight(const QuantWeightParams& p, bool io_bf16, hipStream_t stream) {
  const dim3 grid((p.K + kFp8Block - 1) / kFp8Block, (p.M + kFp8Block - 1) / kFp8Block);
  if (io_bf16) hipLaunchKernelGGL(quant_weight_kernel<bf16_t>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(quant_weight_kernel<float>, grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <typename delta_t, bool kDelta>
static void launch_norm_rows(const QuantParams& p, hipStream_t stream) {
  const dim3 grid(p.tokens), block(512);
  if (p.features <= 1024) hipLaunchKernelGGL((norm_fp8_rows_kernel<delta_t, kDelta, 2>), grid, block, 0, stream, p);
  else if (p.features <= 2048) hipLaunchKernelGGL((norm_fp8_rows_kernel<delta_t, kDelta, 4>), grid, block, 0, stream, p);
  else if (p.features <= 8192) hipLaunchKernelGGL((norm_fp8_rows_kernel<delta_t, kDelta, 16>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((norm_fp8_wide_kernel<delta_t, kDelta>), grid, block, 0, stream, p);
}

template <typename delta_t, bool kDelta>
static void launch_norm(const QuantParams& p, hipStream_t stream) {
  const auto tiles = [&](int n) { return dim3((p.tokens + n - 1) / n); };
  if (p.tokens < kNormTileTokens || p.features > kNormMaxBlocks * kFp8Block)
    launch_norm_rows<delta_t, kDelta>(p, stream);
  else if (p.tokens <= kNormNarrowTokens)
    hipLaunchKernelGGL((norm_fp8_tile_kernel<delta_t, kDelta, 2, 8>), tiles(8), dim3(512), 0, stream, p);
  else if (p.tokens <= kNormMiddleTokens)
    hipLaunchKernelGGL((norm_fp8_tile_kernel<delta_t, kDelta, 4, 8>), tiles(16), dim3(512), 0, stream, p);
  else
    hipLaunchKernelGGL((norm_fp8_tile_kernel<delta_t, kDelta, 8, 8>), tiles(32), dim3(512), 0, stream, p);
}

hipError_t launch_norm_fp8(const QuantParams& p, bool delta_bf16, hipStream_t stream) {
  if (!p.delta) launch_norm<float, false>(p, stream);
  else if (delta_bf16) launch_norm<bf16_t, true>(p, stream);
  else launch_norm<float, true>(p, stream);
  return hipGetLastError();
}

}  // namespace mss
