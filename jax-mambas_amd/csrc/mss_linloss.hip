// A language model's loss from its head's operands, the logits not kept, with its gradients:
// logit[t][v] = sum_d x[d][t] w[v][d] for tokens t and a vocabulary of words v, the losses of
// mss_loss.h over it, dx[d][t] = sum_v w[v][d] g[t][v], dw[v][d] = sum_t g[t][v] x[d][t] with
// g[t][v] = d loss / d logit[t][v].
//
// Forward: one product whose tiles leave, for each token and tile, only the largest s and the sum of
// 2^(s - largest); they are merged a token at a time. The wanted words' logits are formed apart, one
// dot product each. Backward: in pieces of the vocabulary the product is formed again, its tiles
// turned into g (bf16) in a workspace, from which the two gradients' products read. Both at once (bf16 operands,
// wide heads): one product leaves s in 16 bits in the workspace, beside the sums, and g takes its place.
//
// All products run on the matrix cores with float32 sums. bf16 operands are taken as they are
// (v_mfma_f32_32x32x16_bf16); g is rounded to bf16 once, as its factors x and w are. A float32 matrix is taken to
// a power of two's multiple whose largest element lies below 2^15, and split into two planes of half precision: the
// rounding to 11 bits, and that of what it leaves times 2^11. Together they hold an element to 2^-23 of itself down to
// 2^-27 of the largest, and to 2^-50 of the largest below. A product is the sum of three products of planes
// (v_mfma_f32_32x32x16_f16), the two with a lower plane first: what is dropped, the lower ones' own, is at most 2^-22
// of a term, 2^-24.6 in the mean square. g, taken times 2^15, is held to 2^-23 of itself down to 2^-28, and to 2^-51
// below (2^-27 and 2^-50 of the largest upstream gradient where each row has its own). Three times the work of a bf16
// product, at 16 times the rate of the float32 matrix instructions.
//
// 32x32x16 operand layout (lane l, its 8 bf16): A[i][k] at l = i + 32 (k / 8), element k % 8;
// B[k][j] at l = j + 32 (k / 8), element k % 8; D[i][j] at l = j + 32 ((i / 4) % 2),
// register 4 (i / 8) + i % 4.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "mss_loss.h"

namespace mss {

namespace {

typedef __bf16 lbf16x8 __attribute__((ext_vector_type(8)));
typedef float lf32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 lf16x8 __attribute__((ext_vector_type(8)));
typedef short ls16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ls16x4* lds_s16x4_t;

#define LL_INLINE __attribute__((always_inline))  // of lambdas that are called from several places

constexpr int kLlK = 128;  // the gradients' products' k, and those of split matrices, are whole multiples of it

// Tiles of (32 kMT kWM) x (32 kNT kWN) by kWM x kWN waves of kMT x kNT matrix tiles each, kRing stages of kBK k in
// LDS.
template <int kWM_, int kWN_, int kMT_, int kNT_, int kRing_, int kBK_ = 64>
struct LlShape {
  static constexpr int kWM = kWM_, kWN = kWN_, kMT = kMT_, kNT = kNT_, kRing = kRing_, kBK = kBK_;
  static constexpr int kM = 32 * kMT * kWM, kN = 32 * kNT * kWN;
  static constexpr int kWaves = kWM * kWN, kThreads = 64 * kWaves;
  static constexpr int kASlots = kM * kBK / 8, kBSlots = kN * kBK / 8, kSlots = kASlots + kBSlots;  // of 16 bytes
  static constexpr int kACopies = kASlots / kThreads, kBCopies = kBSlots / kThreads;
  static constexpr int kCopies = kACopies + kBCopies;
  // (By the ring alone: with the rows' scales beside it one workgroup of LlThinM fits, which only means that its second
  // half of the tiles is begun when the first is done.)
  static constexpr int kPerCU = kRing * kSlots * 16 > 81920 ? 1 : 2;
  static constexpr int kSums = 16 * kMT * kNT;  // of a lane
  static_assert(kASlots % kThreads == 0 && kBSlots % kThreads == 0, "whole copies");
  static_assert((kRing == 2 || kRing == 4) && (kRing - 1) * kCopies < 64, "");
};

typedef uint32_t lu32x4 __attribute__((ext_vector_type(4)));

// 16 bytes a lane from a buffer to LDS, from `lds` (the same in all lanes) on; zeros past the buffer's end. In
// assembly (there is no register that it writes), since of the builtin's copies the compiler keeps account, and
// waits for all that are in flight before the next transposing read, whose place it does not know. The
// account is this file's: ll_meet. (m0 is nobody's across statements: the compiler sets it where it reads it.)
__device__ __forceinline__ void ll_copy(lu32x4 rsrc, uint32_t offset, const void* lds) {
  const uint32_t to = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_t)lds));
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(to), "v"(offset), "s"(rsrc)
      : "memory");
}

// All waves' copies but the newest kN have landed, and their reads are done.
template <int kN>
__device__ __forceinline__ void ll_meet() {
  static_assert(kN >= 0 && kN < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kN) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// An operand's part of a stage in LDS. Along: rows of kBK k, 16-byte chunks at chunk ^ ((row >> 1) & 7), so
// that the 16 lanes of a read phase (16 rows, one chunk) cover all banks; LDS row r holds matrix row
// perm(r) when kPerm > 1: perm interleaves the kPerm tiles of a wave, lane j's rows then are kPerm
// neighbours. Across: kBK rows of kTile elements, read with the transposing LDS read (a group of 16
// lanes takes 4 rows of 16 elements, lane i gets column i); 64-byte units at unit ^ key(row), the
// four rows of a phase on different banks.
template <int kTile, int kBK, bool kAcross, int kPerm>
struct LlPanel {
  static constexpr int kUnits = kTile / 32, kChunks = kBK / 8;
  static_assert(kBK == 64, "the chunks of a row are eight");
  static __device__ __forceinline__ int chunk(int row, int c) { return c ^ ((row >> 1) & 7); }
  static __device__ __forceinline__ int key(int k) { return kUnits >= 4 ? k & 3 : kUnits == 2 ? (k >> 1) & 1 : 0; }
  // Bytes from the stage's first element to what slot `s` holds.
  static __device__ __forceinline__ uint32_t source(int s, uint32_t ld) {
    if constexpr (kAcross) {
      const int k = s / (kTile / 8), c = s % (kTile / 8);
      return k * ld * 2 + ((((c >> 2) ^ key(k)) << 2) | (c & 3)) * 16;
    } else {
      int row = s / kChunks;
      const int c = chunk(row, s % kChunks);
      if constexpr (kPerm > 1) row = row / (32 * kPerm) * (32 * kPerm) + kPerm * (row & 31) + (row >> 5) % kPerm;
      return row * ld * 2 + c * 16;
    }
  }
  // The operand of matrix tile `tile` (32 rows), step ks of 16 k.
  static __device__ __forceinline__ lbf16x8 fragment(const u32x4* buf, int tile, int ks, int lane) {
    if constexpr (kAcross) {
      const int i = lane & 15, sub = (lane >> 4) & 1, g = lane >> 5, kr = i >> 2;
      const char* at = reinterpret_cast<const char*>(buf) + (ks * 16 + 8 * g + kr) * (kTile * 2) +
                       ((tile ^ key(kr)) << 6) + 32 * sub + 8 * (i & 3);
      union {
        ls16x4 h[2];
        lbf16x8 v;
      } u;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(at));
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(at + 4 * kTile * 2));
      return u.v;
    } else {
      const int row = 32 * tile + (lane & 31), c = 2 * ks + (lane >> 5);
      return __builtin_bit_cast(lbf16x8, buf[row * kChunks + chunk(row, c)]);
    }
  }
};

// The planes of a product of two split matrices (a bit each): of A and of B in pair 0, 1, 2. The sums of the first
// two are taken times 2^-11 before the third's.
constexpr int kPairs = 3;
[[maybe_unused]] constexpr int kLowPairs = 2;
[[maybe_unused]] constexpr unsigned kPairsA = 0b010, kPairsB = 0b001;
constexpr float kLowScale = 0x1p-11f;
constexpr int kGradExponent = 15;  // of the power of two that g is taken times into its planes
constexpr float kGradScale = 1 << kGradExponent;

struct LlArgs {
  LossMatrix a, b;       // from the piece's first row and k on
  int k;                 // of the product, a whole number of stages
  int pairs;             // 1 or kPairs
  int tiles_m, tiles_n;
  int units;             // of a tile: kRing stages each
  int teams;             // of the gradients' products
  int whole, rest;       // whole ranges of a team; the first range of those whose units the teams share evenly
  float* partial;        // their tiles' parts
  long long room;        // floats that these have
};

// kModeExp leaves s - ref, both to base 2, in steps of 2^-9 from -48 on: 0 to 65535 as a part of 65535, and 0 also below.
constexpr float kFixedStep = 0x1p-9f, kFixedLow = -48.f, kFixedUnit = 1.f / (65535.f * kFixedStep);
typedef unsigned short ll_u16x2 __attribute__((ext_vector_type(2)));

enum { kModeLse, kModeGrad, kModeExp, kModeDx, kModeDw };

// What all tokens' gradients are scaled by.
struct LlScale {
  const float* grad;  // NULL: 1, and so the next
  const float* by;
  float temperature;
  const int* power;    // of the split matrix that g is multiplied with; NULL: of bf16 operands
  const int* power_g;  // of the rows' upstream gradients, or NULL
};
// As a factor and a power of two, which go on one after the other: their product may lie outside float32 where what
// they make of a sum does not.
template <bool kF32>
struct LlFactor {
  float f = 1.f;
  int k = 0;
  __device__ __forceinline__ explicit LlFactor(const LlScale& s) {
    f = s.temperature;
    if (s.grad != nullptr) f *= *s.grad;
    if (s.by != nullptr) f *= *s.by;
    if constexpr (kF32) {
      k = __builtin_amdgcn_frexp_expf(f) - *s.power - kGradExponent;
      f = __builtin_amdgcn_frexp_mantf(f);
      if (s.power_g != nullptr) k -= *s.power_g;
    }
  }
  __device__ __forceinline__ float operator()(float v) const { return kF32 ? ldexpf(v * f, k) : v * f; }
};

struct LlOut {
  int rows, cols;        // of the output that exist, from the piece's first on
  float c;
  const int* powers;     // of two, of x and of w where they are split
  float2* part;          // kModeLse: [part][cols]
  const float2* scale;   // kModeGrad, kModeExp: [rows], and a tile's rows more
  bf16_t* g;
  long long ld, plane;   // row stride of g, dx, dw; from one plane of g to the next
  float* f;              // kModeDx, kModeDw with float32 output
  bf16_t* h;             // kModeDw with bf16 output
  int add;               // kModeDx, kModeDw: to what is there
  LlScale by;            // kModeDx with the last piece, kModeDw
  void* dx;              // kModeDx with the last piece: [rows][ld_dx]
  long long ld_dx;
  int dx_bf16;
  const float* live;
  float* row_sums;       // kModeExp: [part][rows]
  float* sum;            // kModeDw in blocks of the tokens: [rows][ld], added to where `add`; the last one writes dw
  int last;
  const int* only_if;    // NULL, or nothing is done where this is 0
};

// What a tile's sums become.
template <int kMode>
constexpr bool kLlTeams = kMode == kModeDx || kMode == kModeDw;
template <int kMode>
constexpr bool kLlGrad = kMode == kModeGrad || kMode == kModeExp;
template <class S, int kMode>
constexpr int ll_perm = kLlGrad<kMode> || kMode == kModeDx ? S::kNT : 1;
template <bool kValue>
struct LlBool {
  static constexpr bool value = kValue;
};
template <int kValue>
struct LlInt {
  static constexpr int value = kValue;
};

// A value's planes of half precision. (An upper one that is not finite has a lower one of zero.)
// v is the rounded float32 number for both: the compiler would round the operation that it comes from straight to the
// upper plane, but take the lower one from v, so that they disagreed where the two roundings do.
__device__ __forceinline__ void split_half(float v, uint16_t& hi, uint16_t& lo) {
  asm volatile("" : "+v"(v));
  const _Float16 h = static_cast<_Float16>(v);
  const float left = (v - static_cast<float>(h)) * (1.f / kLowScale);
  hi = __builtin_bit_cast(uint16_t, h);
  lo = fabsf(left) < INFINITY ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(left)) : 0;
}

// A value of another lane (kCtrl: 0xb1 of lane ^ 1, 0x4e of lane ^ 2, 0x124 and 0x128 of 4 and 8 places back, around
// sixteen lanes).
template <int kCtrl>
__device__ __forceinline__ float quad_mov(float v) {
  return dpp_mov<kCtrl, 0xF>(0.f, v);
}

// A wave's kMT x kNT matrix tiles: from row wm0 and column wn0 on, in part `part` of the words. table: the scales of
// its rows (kModeGrad: a subtrahend and a factor; kModeExp: a subtrahend, and what the 16 bits' fraction adds).
template <int kMode, bool kF32, int kMT, int kNT>
__device__ __forceinline__ void ll_end(const LlOut& o, lf32x16 (&acc)[kMT][kNT], int wm0, int wn0, int part, int lane,
                                       const float2* table) {
  // (What is made of the lane's number is made anew for each tile; kept from one to the next it costs the
  // registers of a copy's offset, whose reload waits for the stores.)
  asm volatile("" : "+v"(lane));
  const int j = lane & 31, g = lane >> 5;
  // (from a split product's sums to a logit to base 2)
  [[maybe_unused]] const float c = kF32 && !kLlTeams<kMode> ? ldexpf(o.c, -(o.powers[0] + o.powers[1])) : o.c;
  const auto row_of = [&](int mt, int r) LL_INLINE { return wm0 + 32 * mt + 8 * (r >> 2) + 4 * g + (r & 3); };
  if constexpr (kMode == kModeLse) {
    // Rows are words, columns tokens: a lane has the words of one token.
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      if (wm0 + 32 * kMT > o.rows) {
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (row_of(mt, r) >= o.rows) acc[mt][nt][r] = -INFINITY;
      }
      float m = acc[0][nt][0];
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[mt][nt][r]);
      m = fmaxf(m, __shfl_xor(m, 32));
      const float mc = m == -INFINITY ? 0.f : m * c;
      float s = 0.f;
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r) s += fast_exp2(__builtin_fmaf(acc[mt][nt][r], c, -mc));
      s += __shfl_xor(s, 32);
      const int t = wn0 + 32 * nt + j;
      if (g == 0 && t < o.cols)
        o.part[static_cast<long long>(part) * o.cols + t] = make_float2(m == -INFINITY ? m : mc, s);
    }
  } else if constexpr (kLlGrad<kMode>) {
    // Rows are tokens, columns words, kNT neighbours a lane. The words past the vocabulary are zeros.
    const int v = wn0 + kNT * j;
    const uint32_t at = static_cast<uint32_t>(4 * g * o.ld + v) * 2;
    const float2* scale = table + 4 * g;
    // kModeExp: of the rows' sums over the wave's words, lane r of sixteen has that of register r. Four rows at a time:
    // lanes exchange the sums of two rows for one's, then of two for one, lane % 4 of four; the other quads' are added.
    float mine[kMT], four[4];
    const bool odd = j & 1, high = j & 2;
    const auto rows = [&](auto edge) LL_INLINE {
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int up = 32 * mt + 8 * (r >> 2) + (r & 3), t = wm0 + up;  // and 4 g more
          const float2 sc = scale[up];
          const float by = kF32 ? sc.y * kGradScale : sc.y;
          float d[kNT];
          [[maybe_unused]] float fixed[kNT];
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            d[nt] = fast_exp2(__builtin_fmaf(acc[mt][nt][r], c, -sc.x));
            if constexpr (kMode == kModeGrad) d[nt] *= by;  // (kModeExp: sc.x is inf in a row that does not count)
            if (edge.value && v + nt >= o.cols) d[nt] = 0.f;
            if constexpr (kMode == kModeExp) {
              fixed[nt] = __builtin_fmaf(acc[mt][nt][r], c * kFixedUnit, sc.y);
              if (edge.value && v + nt >= o.cols) fixed[nt] = 0.f;
            }
          }
          if constexpr (kMode == kModeExp) {
            float s = d[0];
#pragma unroll
            for (int nt = 1; nt < kNT; ++nt) s += d[nt];
            four[r & 3] = s;
            if (r % 4 == 3) {
              const float a = (odd ? four[1] : four[0]) + quad_mov<0xb1>(odd ? four[0] : four[1]);
              const float b = (odd ? four[3] : four[2]) + quad_mov<0xb1>(odd ? four[2] : four[3]);
              s = (high ? b : a) + quad_mov<0x4e>(high ? a : b);
              s += quad_mov<0x124>(s);
              s += quad_mov<0x128>(s);
              mine[mt] = r == 3 || (lane & 12) == r - 3 ? s : mine[mt];
            }
          }
          if (edge.value && t + 4 * g >= o.rows) continue;
          char* dst = reinterpret_cast<char*>(o.g + t * o.ld) + at;
          if constexpr (kMode == kModeExp) {
            ll_u16x2 w[kNT / 2];
#pragma unroll
            for (int h = 0; h < kNT / 2; ++h) w[h] = __builtin_amdgcn_cvt_pknorm_u16(fixed[2 * h], fixed[2 * h + 1]);
            __builtin_memcpy(dst, w, 2 * kNT);
          } else if constexpr (kF32) {
            uint16_t hi[kNT], lo[kNT];
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) split_half(d[nt], hi[nt], lo[nt]);
            __builtin_memcpy(dst, hi, sizeof(hi));
            __builtin_memcpy(dst + o.plane * 2, lo, sizeof(lo));
          } else {
            uint32_t w[(kNT + 1) / 2];
#pragma unroll
            for (int h = 0; h < (kNT + 1) / 2; ++h) w[h] = pack_bf16x2(d[2 * h], d[2 * h + 1 < kNT ? 2 * h + 1 : 2 * h]);
            __builtin_memcpy(dst, w, 2 * kNT);
          }
        }
    };
    const bool whole = wm0 + 32 * kMT <= o.rows && wn0 + 32 * kNT <= o.cols;
    if (whole) rows(LlBool<false>{});
    else rows(LlBool<true>{});
    if constexpr (kMode == kModeExp) {
      const int i = j & 15;
#pragma unroll
      for (int mt = 0; mt < kMT; ++mt) {
        const int t = wm0 + 32 * mt + 8 * (i >> 2) + 4 * g + (i & 3);
        mine[mt] += __shfl_xor(mine[mt], 16);
        if (j < 16 && t < o.rows) o.row_sums[static_cast<long long>(part) * o.rows + t] = mine[mt];
      }
    }
    if (!whole) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the next tile counts a whole tile's stores)
  } else if constexpr (kMode == kModeDx) {
    // Rows are features, columns tokens, kNT neighbours a lane: to the sums over the pieces, or, with the last piece,
    // to dx.
    const int t = wn0 + kNT * j;
    if (t >= o.cols) return;  // (a row of sums is long enough for the last lane's kNT)
    const uint32_t at = static_cast<uint32_t>(4 * g * o.ld + t) * 4;
    const bool last = o.dx != nullptr;
    const long long at_dx = 4LL * g * o.ld_dx + t;
    static_assert(kNT <= 2, "the last lane has one token or all");
    const bool all = t + kNT <= o.cols;
    bool counts[kNT];
    const LlFactor<kF32> by(last ? o.by : LlScale{nullptr, nullptr, 1.f, o.powers, nullptr});
    if (last) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) counts[nt] = t + nt < o.cols && o.live[t + nt] != 0.f;
    }
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d = wm0 + 32 * mt + 8 * q;  // and 4 g more
        float v[4][kNT];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (o.add && d + 4 * g + r < o.rows)
            __builtin_memcpy(v[r], reinterpret_cast<const char*>(o.f + (d + r) * o.ld) + at, sizeof(v[r]));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) v[r][nt] = o.add ? v[r][nt] + acc[mt][nt][4 * q + r] : acc[mt][nt][4 * q + r];
          if (d + 4 * g + r >= o.rows) continue;
          if (!last) {
            __builtin_memcpy(reinterpret_cast<char*>(o.f + (d + r) * o.ld) + at, v[r], sizeof(v[r]));
            continue;
          }
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) v[r][nt] = counts[nt] ? by(v[r][nt]) : 0.f;
          const long long to = (d + r) * o.ld_dx + at_dx;
          if (o.dx_bf16) {
            uint32_t u[(kNT + 1) / 2];
#pragma unroll
            for (int h = 0; h < (kNT + 1) / 2; ++h) u[h] = pack_bf16x2(v[r][2 * h], v[r][2 * h + 1 < kNT ? 2 * h + 1 : 2 * h]);
            bf16_t* dst = static_cast<bf16_t*>(o.dx) + to;
            if (all) __builtin_memcpy(dst, u, 2 * kNT);
            else dst[0].bits = static_cast<uint16_t>(u[0]);
          } else {
            float* dst = static_cast<float*>(o.dx) + to;
            if (all) __builtin_memcpy(dst, v[r], sizeof(v[r]));
            else dst[0] = v[r][0];
          }
        }
        asm volatile("" ::: "memory");  // (a few rows at a time: all of what is there would not fit the registers)
      }
  } else {
    // Rows are words, columns features. Four rows and four lanes change places, so that a lane has four neighbouring
    // columns of one row: a store instruction then writes 8 rows of 64 bytes (or 128) instead of two, and it is
    // their number that short sums wait for.
    const LlFactor<kF32> by(o.by);
    const bool odd = j & 1, high = j & 2;
    const auto rows = [&](auto edge) LL_INLINE {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        const int d = wn0 + 32 * nt + (j & ~3);
        const uint32_t at = static_cast<uint32_t>((4 * g + (j & 3)) * o.ld + d);
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int v = wm0 + 32 * mt + 8 * q;  // and 4 g + j % 4 more
            float x[4], y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = acc[mt][nt][4 * q + r];
#pragma unroll
            for (int h = 0; h < 4; h += 2) {  // rows h, h + 1 between neighbours
              const float z = quad_mov<0xb1>(odd ? x[h] : x[h + 1]);
              y[h] = odd ? z : x[h];
              y[h + 1] = odd ? x[h + 1] : z;
            }
            const float z0 = quad_mov<0x4e>(high ? y[0] : y[2]), z1 = quad_mov<0x4e>(high ? y[1] : y[3]);
            float w[4] = {high ? z0 : y[0], high ? z1 : y[1], high ? y[2] : z0, high ? y[3] : z1};
            if (edge.value && v + 4 * g + (j & 3) >= o.rows) continue;
            const bool all = !edge.value || d + 4 <= o.cols;
            if (o.sum != nullptr) {
              float* sum = o.sum + v * o.ld + at;
              if (o.add) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (all || d + e < o.cols) w[e] += sum[e];
              }
              if (!o.last) {
                if (all) {
                  __builtin_memcpy(sum, w, 16);
                } else {
#pragma unroll
                  for (int e = 0; e < 3; ++e)
                    if (d + e < o.cols) sum[e] = w[e];
                }
                continue;
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = by(w[e]);
            if (o.h != nullptr) {
              char* dst = reinterpret_cast<char*>(o.h + v * o.ld) + 2 * at;
              const uint32_t u[2] = {pack_bf16x2(w[0], w[1]), pack_bf16x2(w[2], w[3])};
              if (all) {
                __builtin_memcpy(dst, u, 8);
              } else {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                  if (d + e < o.cols) reinterpret_cast<uint16_t*>(dst)[e] = static_cast<uint16_t>(u[e / 2] >> (16 * (e & 1)));
              }
            } else {
              char* dst = reinterpret_cast<char*>(o.f + v * o.ld) + 4 * at;
              if (all) {
                __builtin_memcpy(dst, w, 16);
              } else {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                  if (d + e < o.cols) reinterpret_cast<float*>(dst)[e] = w[e];
              }
            }
          }
      }
    };
    if (wm0 + 32 * kMT <= o.rows && wn0 + 32 * kNT <= o.cols) {
      rows(LlBool<false>{});
    } else {
      rows(LlBool<true>{});
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the next tile counts a whole tile's stores)
    }
  }
}

// A workgroup's work is a row of segments: units of one tile each, whose copies follow one another through the
// ring without a gap, so that a tile's first stages arrive under the one before's last products and its end.
//
// kModeLse, kModeGrad, kModeExp: whole tiles. The tiles are dealt out so that those at hand on one XCD are neighbours (8 of
// A by all of B share their operands in its L2), and a workgroup's next one is as many further on as the
// XCD has workgroups.
//
// kModeDx, kModeDw: the tiles of one range of tokens (words) are taken by a team of as many workgroups as there
// are tiles of features, side by side, so that g is read once. A team has a number of whole ranges, and the teams
// share evenly the units of the fewer than a range for each that are left, in order: a part of one range, or the end of
// one and the beginning of the next, whose sums go to `partial` and are added in order by ll_join_kernel.
struct LlSegment {
  int tm, tn, unit, n;  // the tile, its first unit, units: none at the end
};

struct LlDeal {
  int first, step, end;       // whole tiles
  int team, member;           // teams
  long long from, to;         // units of the shared ranges
};

// Where a team's share of the `units` of the shared ranges begins.
__device__ __forceinline__ long long share_start(const LlArgs& p, long long units, int team) { return units * team / p.teams; }

template <int kMode>
__device__ __forceinline__ LlDeal ll_deal(const LlArgs& p) {
  const unsigned n = gridDim.x, per = n / 8, rem = n % 8, x = blockIdx.x % 8, on = x < rem ? per + 1 : per;
  LlDeal d{};
  if constexpr (kLlTeams<kMode>) {
    const int size = kMode == kModeDx ? p.tiles_m : p.tiles_n;
    const unsigned id = x * per + min(x, rem) + blockIdx.x / 8;
    const int team = id / size;
    const long long units = static_cast<long long>((kMode == kModeDx ? p.tiles_n : p.tiles_m) - p.rest) * p.units;
    d.team = team;
    d.member = id % size;
    d.from = share_start(p, units, team);
    d.to = share_start(p, units, team + 1);
  } else {
    const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n;
    const long long before = x * per + min(x, rem);  // workgroups of the XCDs before this one
    d.first = static_cast<int>(tiles * before / n + blockIdx.x / 8);
    d.end = static_cast<int>(tiles * (before + on) / n);
    d.step = on;
  }
  return d;
}

template <int kMode>
__device__ __forceinline__ LlSegment ll_segment(const LlArgs& p, const LlDeal& d, int i) {
  LlSegment s{};
  if constexpr (kLlTeams<kMode>) {
    int range = d.team * p.whole + i;
    if (i < p.whole) {
      s.n = range < p.rest ? p.units : 0;
    } else {
      const int shared = static_cast<int>(d.from / p.units) + i - p.whole;
      const long long begin = static_cast<long long>(shared) * p.units;
      const long long a = d.from > begin ? d.from : begin, b = d.to < begin + p.units ? d.to : begin + p.units;
      range = p.rest + shared;
      s.unit = static_cast<int>(a - begin);
      s.n = a < b ? static_cast<int>(b - a) : 0;
    }
    s.tm = kMode == kModeDx ? d.member : range;
    s.tn = kMode == kModeDx ? range : d.member;
  } else {
    const int id = d.first + i * d.step;
    if (id >= d.end) return s;
    const unsigned group = id / (8u * p.tiles_n), first = group * 8, wide = min(8u, p.tiles_m - first);
    const unsigned in = id - group * 8 * p.tiles_n;
    s.tm = first + in % wide;
    s.tn = in / wide;
    s.n = p.units;
  }
  return s;
}

// The sums of a part: of a team's first shared range (which = 0) or its second.
template <class S, int kMode>
__device__ __forceinline__ f32x4* ll_part(const LlArgs& p, int team, int which, int member) {
  const int size = kMode == kModeDx ? p.tiles_m : p.tiles_n;
  return reinterpret_cast<f32x4*>(p.partial) + ((2LL * team + which) * size + member) * (S::kM * S::kN / 4);
}

template <class S, int kMode, bool kF32>
__global__ __launch_bounds__(S::kThreads) void ll_kernel(LlArgs p, LlOut o) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host's pass knows no buffer resources
  constexpr bool kAAcross = kLlTeams<kMode>, kBAcross = kMode == kModeDw;
  constexpr int kBK = S::kBK;
  using PA = LlPanel<S::kM, kBK, kAAcross, 1>;
  using PB = LlPanel<S::kN, kBK, kBAcross, ll_perm<S, kMode>>;
  __shared__ u32x4 s0[S::kSlots], s1[S::kSlots], s2[S::kRing == 4 ? S::kSlots : 1], s3[S::kRing == 4 ? S::kSlots : 1];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % S::kWM, wn = wave / S::kWM;
  __shared__ float2 s_scale[kLlGrad<kMode> ? S::kM : 1];
  if constexpr (!kLlTeams<kMode>) {
    if (o.only_if != nullptr && *o.only_if == 0) return;
  }
  const LlDeal deal = ll_deal<kMode>(p);
  const int nk = p.k / kBK;

  uint32_t off_a[S::kACopies], off_b[S::kBCopies];
#pragma unroll
  for (int t = 0; t < S::kACopies; ++t)
    off_a[t] = PA::source((wave + S::kWaves * t) * 64 + lane, static_cast<uint32_t>(p.a.ld));
#pragma unroll
  for (int t = 0; t < S::kBCopies; ++t)
    off_b[t] = PB::source((wave + S::kWaves * t) * 64 + lane, static_cast<uint32_t>(p.b.ld));

  // The stage that is copied next. What lies past a matrix's end, in a tile's stages past its last k, or past the
  // last segment is zeros.
  LlSegment next = ll_segment<kMode>(p, deal, 0);
  int next_i = 0, next_left = next.n * S::kRing, next_pair = next.unit * S::kRing / nk, next_k = next.unit * S::kRing % nk;
  const auto rsrc = [&](const LossMatrix& m, int pl, long long at) LL_INLINE {
    const long long left = next_left > 0 && next_pair < p.pairs ? (m.end - at) * 2 : 0;
    const uint64_t base = reinterpret_cast<uint64_t>(m.base + pl * m.plane + at);
    return lu32x4{static_cast<uint32_t>(base), static_cast<uint32_t>(base >> 32) & 0xffff,
                  static_cast<uint32_t>(left < 0 ? 0 : left > 0xfffffff0ll ? 0xfffffff0ll : left), 0x00027000};
  };
  const auto issue = [&](u32x4* d) LL_INLINE {
    const int pa = kF32 ? (kPairsA >> next_pair) & 1 : 0, pb = kF32 ? (kPairsB >> next_pair) & 1 : 0;
    const long long k0 = static_cast<long long>(next_k) * kBK, m0 = static_cast<long long>(next.tm) * S::kM,
                    n0 = static_cast<long long>(next.tn) * S::kN;
    const auto ra = rsrc(p.a, pa, kAAcross ? k0 * p.a.ld + m0 : m0 * p.a.ld + k0);
    const auto rb = rsrc(p.b, pb, kBAcross ? k0 * p.b.ld + n0 : n0 * p.b.ld + k0);
#pragma unroll
    for (int t = 0; t < S::kACopies; ++t)
      ll_copy(ra, off_a[t], d + 64 * (wave + S::kWaves * t));
#pragma unroll
    for (int t = 0; t < S::kBCopies; ++t)
      ll_copy(rb, off_b[t], d + S::kASlots + 64 * (wave + S::kWaves * t));
    if (++next_k == nk) {
      next_k = 0;
      ++next_pair;
    }
    if (--next_left == 0) {
      next = ll_segment<kMode>(p, deal, ++next_i);
      next_left = next.n * S::kRing;
      next_pair = next.unit * S::kRing / nk;
      next_k = next.unit * S::kRing % nk;
    }
  };

  // The scales of a tile's rows, by every wave, some of them the same ones.
  const auto scales = [&](int tm) LL_INLINE {
    constexpr int kSlices = (S::kM + 127) / 128;  // of 1 KB
    const uint64_t base = reinterpret_cast<uint64_t>(o.scale + tm * S::kM);
    // (readfirstlane: it is the same in all lanes, which the compiler does not see)
    const lu32x4 r{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(base))),
                   static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(base >> 32) & 0xffff)),
                   S::kM * 8, 0x00027000};
    const int slice = wave % kSlices;
    if (S::kM % 128 == 0 || 1024 * slice + 16 * lane < S::kM * 8)
      ll_copy(r, 1024 * slice + 16 * lane, reinterpret_cast<const char*>(s_scale) + 1024 * slice);
  };

  lf32x16 acc[S::kMT][S::kNT];
  // Operands of the step at hand and of the one after it.
  lbf16x8 fa[2][S::kMT], fb[2][S::kNT];
  const auto load = [&](const u32x4* buf, int ks) LL_INLINE {
#pragma unroll
    for (int t = 0; t < S::kMT; ++t) fa[ks & 1][t] = PA::fragment(buf, wm * S::kMT + t, ks, lane);
#pragma unroll
    for (int t = 0; t < S::kNT; ++t) fb[ks & 1][t] = PB::fragment(buf + S::kASlots, wn * S::kNT + t, ks, lane);
  };
  const auto multiply = [&](int ks) LL_INLINE {
#pragma unroll
    for (int mt = 0; mt < S::kMT; ++mt)
#pragma unroll
      for (int nt = 0; nt < S::kNT; ++nt)
        if constexpr (kF32)
          acc[mt][nt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lf16x8, fa[ks & 1][mt]),
                                                               __builtin_bit_cast(lf16x8, fb[ks & 1][nt]), acc[mt][nt], 0, 0, 0);
        else
          acc[mt][nt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[ks & 1][mt], fb[ks & 1][nt], acc[mt][nt], 0, 0, 0);
  };
  const auto lower = [&]() LL_INLINE {  // the sums with a lower plane
#pragma unroll
    for (int mt = 0; mt < S::kMT; ++mt)
#pragma unroll
      for (int nt = 0; nt < S::kNT; ++nt) acc[mt][nt] *= kLowScale;
  };
  constexpr int kSteps = kBK / 16;
  constexpr int kReads = S::kMT * (kAAcross ? 2 : 1) + S::kNT * (kBAcross ? 2 : 1), kProducts = S::kMT * S::kNT;
  constexpr int kEach = (kReads + kProducts - 1) / kProducts;
  const auto weave = [&]() LL_INLINE {  // a read behind each product
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
    }
  };
  // A ring of kRing stages. Before the last step of a stage all waves meet: they have read all of it, so its place
  // takes the copies of the stage kRing further on, and the stage behind it has landed, so that its first
  // operands are read under that last step's products.
  const auto step = [&](u32x4* cur, const u32x4* next, auto newer) LL_INLINE {
#pragma unroll
    for (int ks = 0; ks + 1 < kSteps; ++ks) {
      load(cur, ks + 1);
      multiply(ks);
      weave();
    }
    ll_meet<(S::kRing - 2) * S::kCopies + newer.value>();
    issue(cur);
    load(next, 0);
    multiply(kSteps - 1);
    weave();
  };
  issue(s0);
  issue(s1);
  if constexpr (S::kRing == 4) {
    issue(s2);
    issue(s3);
  }
  ll_meet<(S::kRing - 1) * S::kCopies>();
  load(s0, 0);
  for (int i = 0;; ++i) {
    const LlSegment seg = ll_segment<kMode>(p, deal, i);
    if (seg.n == 0) break;
#pragma unroll
    for (int a = 0; a < S::kMT; ++a)
#pragma unroll
      for (int b = 0; b < S::kNT; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;
    const auto unit = [&](auto newer, bool first) LL_INLINE {
      step(s0, s1, newer);
      // The scales of the tile's rows, once all waves are through with the ones before.
      if constexpr (kLlGrad<kMode>) {
        if (first) scales(seg.tm);
      }
      if constexpr (S::kRing == 2) {
        step(s1, s0, LlInt<0>{});
      } else {
        step(s1, s2, LlInt<0>{});
        step(s2, s3, LlInt<0>{});
        step(s3, s0, LlInt<0>{});
      }
    };
    // (The first unit of a later tile meets while the stores of the one before, newer than its copies, go on.)
    // (dw: a part's stores are as many.)
    constexpr int kOut = kLlGrad<kMode> ? (kF32 ? 2 : 1) * 16 * S::kMT : kMode == kModeDw ? S::kSums / 4 : 0;
    constexpr int kStores = S::kRing == 2 && kOut <= 55 ? kOut : 0;
    const int low = kLowPairs * nk / S::kRing - seg.unit;  // units with a lower plane (a product's k is whole units)
    int u = 0;
    if constexpr (kLlGrad<kMode> || kStores > 0) {
      if (i > 0) unit(LlInt<kStores>{}, true);
      else unit(LlInt<0>{}, true);
      u = 1;
    }
    for (; u < seg.n; ++u) {
      if constexpr (kF32) {
        if (u == low) lower();
      }
      unit(LlInt<0>{}, false);
    }
    if constexpr (kF32) {
      if (seg.n <= low) lower();
    }
    if constexpr (kLlTeams<kMode>) {
      if (seg.n < p.units) {
        // A part: its sums, in the order in which the lanes hold them.
        f32x4* dst = ll_part<S, kMode>(p, deal.team, i > p.whole, deal.member) + wave * (S::kSums / 4 * 64) + lane;
#pragma unroll
        for (int e = 0; e < S::kSums / 4; ++e)
          dst[64 * e] = f32x4{acc[e / 4 / S::kNT][e / 4 % S::kNT][4 * (e % 4)], acc[e / 4 / S::kNT][e / 4 % S::kNT][4 * (e % 4) + 1],
                              acc[e / 4 / S::kNT][e / 4 % S::kNT][4 * (e % 4) + 2], acc[e / 4 / S::kNT][e / 4 % S::kNT][4 * (e % 4) + 3]};
        continue;
      }
    }
    ll_end<kMode, kF32>(o, acc, seg.tm * S::kM + wm * 32 * S::kMT, seg.tn * S::kN + wn * 32 * S::kNT,
                      kMode == kModeExp ? seg.tn * S::kWN + wn : seg.tm * S::kWM + wm, lane,
                  s_scale + wm * 32 * S::kMT);
    // (None of the loads that the compiler knows of is outstanding: else it would wait in the loop, with the copies.)
    if constexpr (kMode == kModeDx) __builtin_amdgcn_s_waitcnt(0x0f70);
    if constexpr (kMode == kModeDw) {
      if (o.add) __builtin_amdgcn_s_waitcnt(0x0f70);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the workgroup's LDS
#endif
}

// The tiles of the shared ranges: the parts' sums, in a fixed order. A workgroup for each row of matrix tiles of a
// wave, whose four waves take every fourth part.
constexpr int kJoinWaves = 4;

template <class S, int kMode, bool kF32>
__global__ __launch_bounds__(64 * kJoinWaves) void ll_join_kernel(LlArgs p, LlOut o) {
  __shared__ f32x4 s_sum[kJoinWaves - 1][4 * S::kNT][64];
  const int lane = threadIdx.x & 63, mine = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int size = kMode == kModeDx ? p.tiles_m : p.tiles_n, ranges = kMode == kModeDx ? p.tiles_n : p.tiles_m;
  const int mt = blockIdx.x % S::kMT, wave = blockIdx.x / S::kMT % S::kWaves;
  const int tile = blockIdx.x / (S::kMT * S::kWaves), shared = tile / size, member = tile % size, range = p.rest + shared;
  const long long units = static_cast<long long>(ranges - p.rest) * p.units, begin = static_cast<long long>(shared) * p.units;
  int team = static_cast<int>(begin * p.teams / units);  // the one with the range's first unit
  while (team > 0 && share_start(p, units, team) > begin) --team;
  while (share_start(p, units, team + 1) <= begin) ++team;
  lf32x16 acc[1][S::kNT];
#pragma unroll
  for (int b = 0; b < S::kNT; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[0][b][e] = 0.f;
  int end = static_cast<int>((begin + p.units) * p.teams / units);  // the first team behind the range
  while (end > 0 && share_start(p, units, end - 1) >= begin + p.units) --end;
  while (end < p.teams && share_start(p, units, end) < begin + p.units) ++end;
#pragma unroll 2
  for (team += mine; team < end; team += kJoinWaves) {
    if (share_start(p, units, team) == share_start(p, units, team + 1)) continue;  // (fewer units than teams)
    const f32x4* src = ll_part<S, kMode>(p, team, share_start(p, units, team) / p.units != shared, member) +
                       wave * (S::kSums / 4 * 64) + mt * (S::kNT * 4 * 64) + lane;
#pragma unroll
    for (int e = 0; e < 4 * S::kNT; ++e) {
      const f32x4 v = src[64 * e];
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[0][e / 4][4 * (e % 4) + q] += v[q];
    }
  }
  if (mine > 0) {
#pragma unroll
    for (int e = 0; e < 4 * S::kNT; ++e)
      s_sum[mine - 1][e][lane] = f32x4{acc[0][e / 4][4 * (e % 4)], acc[0][e / 4][4 * (e % 4) + 1], acc[0][e / 4][4 * (e % 4) + 2],
                                       acc[0][e / 4][4 * (e % 4) + 3]};
  }
  __syncthreads();
  if (mine > 0) return;
#pragma unroll
  for (int i = 0; i < kJoinWaves - 1; ++i)
#pragma unroll
    for (int e = 0; e < 4 * S::kNT; ++e) {
      const f32x4 v = s_sum[i][e][lane];
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[0][e / 4][4 * (e % 4) + q] += v[q];
    }
  const int tm = kMode == kModeDx ? member : range, tn = kMode == kModeDx ? range : member;
  ll_end<kMode, kF32>(o, acc, tm * S::kM + (wave % S::kWM * S::kMT + mt) * 32, tn * S::kN + wave / S::kWM * 32 * S::kNT, 0, lane,
                nullptr);
}

// ------------------------------------------------------------------------- operands
// The largest finite magnitudes of float32 matrices, a block's each (as bits, in the order of the values): x's of the
// tokens that count in the first kMaxX, w's behind them.
constexpr int kMaxX = 128, kMaxW = 512;
static_assert(kMaxX + kMaxW == kLinLossMaxima, "");

__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

__device__ __forceinline__ bool row_counts(const LinLossParams& p, int t) {
  return p.r.targets != nullptr ? p.r.targets[t] != p.r.ignore : p.r.live[t] != 0.f;
}

template <int kWaves>
__device__ __forceinline__ uint32_t block_max(uint32_t m, uint32_t* s) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), off)));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) m = max(m, s[i]);
  return m;
}

// 16 waves, so that enough of the matrix is on its way.
__global__ __launch_bounds__(1024) void ll_max_kernel(LinLossParams p) {
  __shared__ uint32_t s[16];
  uint32_t m = 0;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (blockIdx.x < kMaxX) {
    const float* x = static_cast<const float*>(p.x);
    const bool along_f = p.sf == 1;
    const int rows = along_f ? p.tokens : p.features, cols = along_f ? p.features : p.tokens;
    for (int r = blockIdx.x * 16 + w; r < rows; r += 16 * kMaxX)
      for (int c0 = lane; c0 < cols; c0 += 8 * 64) {
        float v[8];  // (on their way at once; a place past the row's end takes its last one)
        bool counts[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = min(c0 + 64 * e, cols - 1), f = along_f ? c : r, t = along_f ? r : c;
          v[e] = x[f * p.sf + t * p.st];
          counts[e] = row_counts(p, t);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) m = counts[e] ? max(m, finite_bits(v[e])) : m;
      }
  } else {
    const float* v = static_cast<const float*>(p.w);
    for (int r = (blockIdx.x - kMaxX) * 16 + w; r < p.vocab; r += 16 * kMaxW) {
      const float* row = v + r * p.ldw;
      for (int c0 = 4 * lane; c0 + 4 <= p.features; c0 += 4 * 256) {
        u32x4 u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = *reinterpret_cast<const u32x4_any*>(row + min(c0 + 256 * e, p.features - 4));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          m = max(max(m, max(finite_bits(__uint_as_float(u[e][0])), finite_bits(__uint_as_float(u[e][1])))),
                  max(finite_bits(__uint_as_float(u[e][2])), finite_bits(__uint_as_float(u[e][3]))));
      }
      if (lane < p.features % 4) m = max(m, finite_bits(row[p.features - 1 - lane]));
    }
  }
  m = block_max<16>(m, s);
  if (threadIdx.x == 0) p.maxima[blockIdx.x] = m;
}

// The power of two that takes the largest of kN maxima to 2^14 and more, below 2^15, to all of a block.
template <int kN>
__device__ __forceinline__ int plane_power(const uint32_t* maxima, int* power) {
  __shared__ uint32_t s[4];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kN; i += 256)
    if (i + static_cast<int>(threadIdx.x) < kN) m = max(m, maxima[i + threadIdx.x]);
  m = block_max<4>(m, s);
  const int e = m == 0 ? 0 : 15 - __builtin_amdgcn_frexp_expf(__uint_as_float(m));
  if (power != nullptr && threadIdx.x == 0) *power = e;
  return e;
}

// 8 neighbours of a row in their planes: as they are, or split after scaling.
template <bool kF32>
__device__ __forceinline__ void store_planes(const float (&v)[8], int power, bf16_t* dst, long long plane) {
  alignas(16) uint16_t hi[8], lo[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (kF32) split_half(ldexpf(v[e], power), hi[e], lo[e]);
    else hi[e] = f32_to_bf16(v[e]).bits;
  }
  *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(hi);
  if constexpr (kF32) *reinterpret_cast<u32x4*>(dst + plane) = *reinterpret_cast<const u32x4*>(lo);
}

// x (features, tokens) as token-major rows of `width` features, zeros past the last feature and in rows that
// do not count (whatever a masked token holds then reaches nothing). Tiles of 64 x 64 through LDS, read
// along whichever axis is contiguous.
// With targets the first blocks note the rows' words too.
template <typename in_t>
__global__ __launch_bounds__(256) void ll_pack_x_kernel(LinLossParams p) {
  constexpr bool kF32 = sizeof(in_t) == 4;
  int power = 0;
  if constexpr (kF32) power = plane_power<kMaxX>(p.maxima, blockIdx.x + blockIdx.y == 0 ? p.powers : nullptr);
  __shared__ float s[64][65];
  __shared__ bool s_live[64];
  const int t0 = blockIdx.x * 64, f0 = blockIdx.y * 64;
  const in_t* x = static_cast<const in_t*>(p.x);
  const bool along_f = p.sf == 1;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (w == 0) {
    const int t = t0 + lane;
    float live = 0.f;
    if (t < p.tokens) {
      if (p.r.targets != nullptr) {
        const long long v = p.r.targets[t];
        const bool inside = v >= 0 && v < p.r.vocab;
        live = v == p.r.ignore ? 0.f : inside ? 1.f : __builtin_nanf("");
        if (blockIdx.y == 0) {
          p.r.words[t] = live == 1.f ? static_cast<int>(v) : -1;
          p.r.q[t] = 1.f;
          p.r.live[t] = live;
        }
      } else {
        live = p.r.live[t];
      }
    }
    s_live[lane] = live != 0.f;
    if (p.r.targets != nullptr && blockIdx.y == 0) {
      const int n = __popcll(__ballot(live != 0.f));
      if (lane == 0) p.r.counts[blockIdx.x] = n;
    }
  }
  in_t v[16];  // (all of them on their way at once: loads under a condition would follow one another)
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int f = min(f0 + (along_f ? lane : w + 4 * i), p.features - 1);
    const int t = min(t0 + (along_f ? w + 4 * i : lane), p.tokens - 1);
    v[i] = x[f * p.sf + t * p.st];
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int a = along_f ? lane : w + 4 * i, b = along_f ? w + 4 * i : lane;  // feature, token
    s[a][b] = f0 + a < p.features && t0 + b < p.tokens ? to_f32(v[i]) : 0.f;
  }
  __syncthreads();
  const long long plane = static_cast<long long>(p.tokens) * p.width;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int slot = threadIdx.x + 256 * i, b = slot / 8, c = 8 * (slot % 8);
    const int t = t0 + b;
    if (t >= p.tokens) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = s_live[b] ? s[c + e][b] : 0.f;
    store_planes<kF32>(v, power, p.xp + static_cast<long long>(t) * p.width + f0 + c, plane);
  }
}

// The weight's rows, `width` features each.
template <typename in_t>
__global__ __launch_bounds__(256) void ll_pack_w_kernel(LinLossParams p) {
  constexpr bool kF32 = sizeof(in_t) == 4;
  int power = 0;
  if constexpr (kF32) power = plane_power<kMaxW>(p.maxima + kMaxX, blockIdx.x == 0 ? p.powers + 1 : nullptr);
  const int per = p.width / 8;
  const long long n = static_cast<long long>(p.vocab) * per, plane = static_cast<long long>(p.vocab) * p.width;
  const in_t* w = static_cast<const in_t*>(p.w);
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) {
    const long long row = i / per;
    const int c = 8 * static_cast<int>(i - row * per);
    const in_t* src = w + row * p.ldw + c;
    alignas(16) in_t raw[8];
    float v[8];
    if (c + 8 <= p.features) {
#pragma unroll
      for (int e = 0; e < static_cast<int>(sizeof(raw) / 16); ++e)
        reinterpret_cast<u32x4*>(raw)[e] = reinterpret_cast<const u32x4_any*>(src)[e];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = to_f32(raw[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < p.features ? to_f32(src[e]) : 0.f;
    }
    store_planes<kF32>(v, power, p.wp + row * p.width + c, plane);
  }
}

// ------------------------------------------------------------------------- the wanted words' logits
// A wave takes four words of a token's list at a time.
template <bool kF32>
__device__ __forceinline__ void load_planes(const bf16_t* at, long long plane, float (&v)[8]) {
  const u32x4 u = *reinterpret_cast<const u32x4*>(at);
  if constexpr (kF32) {
    const u32x4 l = *reinterpret_cast<const u32x4*>(at + plane);
    const lf16x8 hi = __builtin_bit_cast(lf16x8, u), lo = __builtin_bit_cast(lf16x8, l);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(static_cast<float>(lo[i]), kLowScale, static_cast<float>(hi[i]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
}

// The logits of kN words of token t (a negative word: 0), in all lanes.
template <bool kF32, int kN>
__device__ __forceinline__ void ll_dots(const LinLossParams& p, const LossMatrix& w, long long t, const int (&word)[kN],
                                        int lane, float (&sum)[kN]) {
  const long long xplane = static_cast<long long>(p.tokens) * p.width;
#pragma unroll
  for (int e = 0; e < kN; ++e) sum[e] = 0.f;
  for (int c = 8 * lane; c < p.width; c += 512) {
    float x[8];
    load_planes<kF32>(p.xp + t * p.width + c, xplane, x);
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      if (word[e] < 0) continue;
      float v[8];
      load_planes<kF32>(w.base + word[e] * w.ld + c, w.plane, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[e] = __builtin_fmaf(x[i], v[i], sum[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < kN; ++e) {
    sum[e] = wave_sum(sum[e]);
    if constexpr (kF32) sum[e] = ldexpf(sum[e], -(p.powers[0] + p.powers[1]));
  }
}

// table (or NULL): what a token's exponentials are taken relative to, to base 2 (kModeExp), the largest logit of its
// list's first four words; inf for one that does not count. blocks: of tokens, whose notes are cleared.
template <bool kF32>
__global__ __launch_bounds__(256) void ll_pick_kernel(LinLossParams p, LossMatrix w, float2* table, int blocks) {
  const int lane = threadIdx.x & 63;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < blocks; i += 256) p.bad[i] = 0;
  const int per = (p.r.top + 3) / 4;
  const long long id = blockIdx.x * 4LL + (threadIdx.x >> 6);
  const long long t = id / per;
  if (t >= p.tokens) return;
  const int k0 = 4 * static_cast<int>(id - t * per);
  int word[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) word[e] = k0 + e < p.r.top ? p.r.words[t * p.r.top + k0 + e] : -1;
  float sum[4];
  ll_dots<kF32>(p, w, t, word, lane, sum);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane == 0 && k0 + e < p.r.top) p.picked[t * p.r.top + k0 + e] = sum[e];
  if (table != nullptr && k0 == 0 && lane == 0) {
    float ref = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (word[e] >= 0) ref = fmaxf(ref, sum[e]);
    ref = p.r.live[t] == 0.f ? INFINITY : fabsf(ref) < INFINITY ? ref * p.c : 0.f;
    table[t] = make_float2(ref, (-kFixedLow - ref) * kFixedUnit);
  }
}

// ------------------------------------------------------------------------- a token's loss
// 16 tokens a workgroup: the parts' sums merged, 64 slices of them side by side, then a wave a token over its list.
// kPick: there is one word a token, whose logit is formed here.
constexpr int kFinishTokens = 16, kFinishSlices = 64;

// (m, s) with (m2, s2): the sums of 2^(. - m), 2^(. - m2).
__device__ __forceinline__ void sums_merge(float& m, float& s, float m2, float s2) {
  const float mx = fmaxf(m, m2);
  if (mx == -INFINITY) {
    s += s2;  // zero, or NaN
    return;
  }
  s = s * fast_exp2(m - mx) + s2 * fast_exp2(m2 - mx);
  m = mx;
}

template <bool kPick, bool kF32>
__global__ __launch_bounds__(kFinishTokens * kFinishSlices) void ll_finish_kernel(LinLossParams p, LossMatrix wm) {
  __shared__ float s_m[kFinishSlices][kFinishTokens], s_s[kFinishSlices][kFinishTokens], s_log[kFinishTokens];
  if (p.only_if != nullptr && *p.only_if == 0) return;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int t0 = blockIdx.x * kFinishTokens;
  const int mine = threadIdx.x % kFinishTokens, slice = threadIdx.x / kFinishTokens;
  const long long t = t0 + w;
  float logit[1] = {0.f};
  if constexpr (kPick) {
    if (t < p.tokens) {
      const int word[1] = {p.r.words[t]};
      ll_dots<kF32>(p, wm, t, word, lane, logit);
      if (lane == 0) p.picked[t] = logit[0];
    }
  }
  {
    float m = -INFINITY, s = 0.f;
    if (t0 + mine < p.tokens) {
      for (int i0 = slice; i0 < p.parts; i0 += 4 * kFinishSlices) {
        float2 q[4];  // (on their way at once)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          q[e] = p.part[static_cast<long long>(min(i0 + e * kFinishSlices, p.parts - 1)) * p.tokens + t0 + mine];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i0 + e * kFinishSlices < p.parts) sums_merge(m, s, q[e].x, q[e].y);
      }
    }
    s_m[slice][mine] = m;
    s_s[slice][mine] = s;
  }
  for (int h = kFinishSlices / 2; h > 0; h /= 2) {
    __syncthreads();
    if (slice < h) {
      float m = s_m[slice][mine], s = s_s[slice][mine];
      sums_merge(m, s, s_m[slice + h][mine], s_s[slice + h][mine]);
      s_m[slice][mine] = m;
      s_s[slice][mine] = s;
    }
  }
  __syncthreads();
  if (threadIdx.x < kFinishTokens) {
    if (t0 + mine < p.tokens) {
      const float live = p.r.live[t0 + mine];  // (NaN for a row that has a word outside the vocabulary)
      p.stat[t0 + mine] = make_float2(s_m[0][mine], live == 0.f ? 0.f : 1.f / s_s[0][mine] + (live - live));
    }
    s_log[mine] = fast_log2(s_s[0][mine]);
  }
  __syncthreads();
  if (t >= p.tokens) return;
  const float m = s_m[0][w], log_s = s_log[w];
  float sum = 0.f;
  for (int k = lane; k < p.r.top; k += 64) {
    const long long at = t * p.r.top + k;
    if (p.r.words[at] < 0) continue;
    const float q = p.r.q[at];
    const float z = kPick ? logit[0] : p.picked[at];
    sum = __builtin_fmaf(q, (m - z * p.c) + log_s + fast_log2(q), sum);
  }
  sum = wave_sum(sum) * (kLn2 * p.temperature * p.temperature);
  const float live = p.r.live[t];
  if (live == 0.f) sum = 0.f;
  if (lane == 0) p.loss[t] = sum + (live - live);
}

// ------------------------------------------------------------------------- both directions at once
// For a block of tokens and the whole vocabulary at a time, kModeExp leaves the words' s - ref in 16 bits, with ref a
// logit of the token's own list, and the sums S of 2^(s - ref); then g = 2^(s - ref) / S - q, rounded to bf16, takes
// their place: the logits are formed once, not twice. The 16 bits hold s to half of 2^-9, so that g is off by 2^-10.5
// of itself before it is rounded (by 2^-8 at most), and zero where s - ref is below -48, a probability below 2^-38 (S
// being more than 2^-10); a bf16 2^(s - ref), the division left to x's rows and dx's
// columns, would need no conversion, but cost dw another whole rounding. It fails where S passes 2^79, a token whose
// words lie that far below its largest logit: such a row is noted in `bad`, and the kernels of the two apart,
// launched behind, make the block's losses and g anew; else they return at once.
// (These kernels' tokens are a block's.)
__global__ __launch_bounds__(kFinishTokens * kFinishSlices) void ll_block_kernel(LinLossParams p, int parts) {
  __shared__ float s_s[kFinishSlices][kFinishTokens];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int first = blockIdx.x * kFinishTokens;
  const int mine = threadIdx.x % kFinishTokens, slice = threadIdx.x / kFinishTokens;
  {
    float s = 0.f;
    if (first + mine < p.tokens) {
#pragma unroll 4
      for (int i = slice; i < parts; i += kFinishSlices) s += p.row_sums[static_cast<long long>(i) * p.tokens + first + mine];
    }
    s_s[slice][mine] = s;
  }
  for (int h = kFinishSlices / 2; h > 0; h /= 2) {
    __syncthreads();
    if (slice < h) s_s[slice][mine] += s_s[slice + h][mine];
  }
  __syncthreads();
  const long long t = first + w;
  if (t >= p.tokens) return;
  const float live = p.r.live[t], S = s_s[0][w];
  const bool counts = live != 0.f;
  const float ref = p.scale[t].x, log_s = fast_log2(S);
  if (lane == 0) {  // (a live of NaN: a word outside the vocabulary)
    p.stat[t] = make_float2(ref, counts ? 1.f / S + (live - live) : 0.f);
    if (counts && !(S > 0x1p-10f && S < 0x1p79f)) *p.bad = 1;
  }
  float sum = 0.f;
  for (int k = lane; k < p.r.top; k += 64) {
    const long long i = t * p.r.top + k;
    if (p.r.words[i] < 0) continue;
    const float q = p.r.q[i];
    sum = __builtin_fmaf(q, (ref - p.picked[i] * p.c) + log_s + fast_log2(q), sum);
  }
  sum = wave_sum(sum) * (kLn2 * p.temperature * p.temperature);
  if (lane == 0) p.loss[t] = (counts ? sum : 0.f) + (live - live);
}

// A workgroup a token: its 16 bits to g, then its list's words anew. (8192 x 50280: 322 us, 5.1 TB/s. In parts of 1280
// tokens, which stay in the cache of 256 MB, 45 us each, but the product then has fewer tiles a launch: 1115 us for both
// instead of 1010.)
__global__ __launch_bounds__(256) void ll_convert_kernel(LinLossParams p) {
  if (*p.bad != 0) return;
  const long long t = gridDim.x - 1 - blockIdx.x;  // (the last ones are in the caches)
  bf16_t* row = p.g + t * p.ldg;
  const float2 st = p.stat[t];
  const float by = kFixedLow + fast_log2(st.y);  // (a row that does not count has zeros: -inf)
  const float zero = st.y - st.y;  // or NaN
#pragma unroll 4
  for (int c = 8 * threadIdx.x; c < p.ldg; c += 8 * 256) {
    u32x4 v = *reinterpret_cast<const u32x4*>(row + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = v[i] & 0xffffu, hi = v[i] >> 16;
      const float a = fast_exp2(__builtin_fmaf(static_cast<float>(lo), kFixedStep, by));
      const float d = fast_exp2(__builtin_fmaf(static_cast<float>(hi), kFixedStep, by));
      v[i] = pack_bf16x2(lo == 0 ? zero : a, hi == 0 ? zero : d);
    }
    *reinterpret_cast<u32x4*>(row + c) = v;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < p.r.top; k += 256) {
    const long long i = t * p.r.top + k;
    const int word = p.r.words[i];
    if (word >= 0) store_as(row + word, __builtin_fmaf(fast_exp2(__builtin_fmaf(p.picked[i], p.c, -st.x)), st.y, -p.r.q[i]));
  }
}

// Gradients of an upstream gradient of 1 to those of another one (nothing for 1).
template <typename T>
__device__ __forceinline__ void rescale(T* v, long long n, float f) {
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) store_as(v + i, to_f32(v[i]) * f);
}

__global__ __launch_bounds__(256) void ll_rescale_kernel(bf16_t* dx, long long nx, void* dw, int dw_bf16, long long nw,
                                                         const float* grad) {
  const float f = *grad;
  if (f == 1.f) return;
  rescale(dx, nx, f);
  if (dw_bf16) rescale(static_cast<bf16_t*>(dw), nw, f);
  else rescale(static_cast<float*>(dw), nw, f);
}

// ------------------------------------------------------------------------- backward, around the products
// A token's largest s, and what its 2^(s - largest) are scaled by: one over their sum, and without a reduction its own
// upstream gradient, before g is rounded. (With one, no gradient: what all tokens share is left to the products' ends,
// since 1 / tokens has an error of its own in bf16, the same for every token.)
// (Split, they are taken to a power of two's multiple below 1 first: one workgroup.)
template <bool kF32>
__global__ __launch_bounds__(1024) void ll_scale_kernel(LinLossParams p, float2* scale) {
  int power = 0;
  if constexpr (kF32) {
    __shared__ uint32_t s[16];
    uint32_t m = 0;
#pragma unroll 4
    for (int t = threadIdx.x; t < p.tokens; t += 1024) {
      const uint32_t up = finite_bits(p.grad[t] * p.temperature);
      m = p.stat[t].y == 0.f ? m : max(m, up);  // (whatever comes to a row that does not count)
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), off)));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int i = 0; i < 16; ++i) m = max(m, s[i]);
    power = m == 0 ? 0 : -__builtin_amdgcn_frexp_expf(__uint_as_float(m));
    if (threadIdx.x == 0) p.power_g[0] = power;
  }
  for (int t = blockIdx.x * 1024 + threadIdx.x; t < p.tokens; t += gridDim.x * 1024) {
    const float2 st = p.stat[t];
    scale[t] = make_float2(st.x, st.y == 0.f ? 0.f : st.y * ldexpf(p.grad[t] * p.temperature, power));
  }
}

// g at the wanted words of the piece that begins at word v0. In bf16 from their own logits, since their probabilities
// are rounded there. The planes of a float32 one hold it to 2^-23: it is the product's own then, whose exponential is
// part of the row's sum, so that what they are both off by cancels where the probability is nearly 1.
template <bool kF32>
__global__ __launch_bounds__(256) void ll_wanted_kernel(LinLossParams p, const float2* scale, int v0, int words) {
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= static_cast<long long>(p.tokens) * p.r.top || (p.only_if != nullptr && *p.only_if == 0)) return;
  const int v = p.r.words[i] - v0;
  if (p.r.words[i] < 0 || v < 0 || v >= words) return;
  const long long t = i / p.r.top;
  float up = 1.f;
  if (p.reduction == kLossNone) up = ldexpf(p.grad[t] * p.temperature, kF32 ? p.power_g[0] : 0);
  bf16_t* dst = p.g + t * p.ldg + v;
  if constexpr (kF32) {
    bf16_t* low = dst + p.tokens * p.ldg;
    const float d = __builtin_fmaf(static_cast<float>(__builtin_bit_cast(_Float16, low->bits)), kLowScale,
                                   static_cast<float>(__builtin_bit_cast(_Float16, dst->bits)));
    split_half(__builtin_fmaf(-p.r.q[i] * up, kGradScale, d), dst->bits, low->bits);
  } else {
    const float2 sc = scale[t];
    store_as(dst, __builtin_fmaf(fast_exp2(__builtin_fmaf(p.picked[i], p.c, -sc.x)), sc.y, -p.r.q[i] * up));
  }
}

unsigned blocks_for(long long n, long long most) {
  const long long b = (n + 255) / 256;
  return static_cast<unsigned>(b < most ? b : most);
}

//                WM WN MT NT ring
typedef LlShape<2, 4, 4, 2, 2> LlLargeM;   // 256 x 256, waves of 128 x 64
typedef LlShape<4, 2, 2, 4, 2> LlLargeN;   // 256 x 256, waves of 64 x 128
typedef LlShape<4, 2, 2, 3, 2> LlMidM;     // 256 x 192, waves of 64 x 96
typedef LlShape<2, 4, 3, 2, 2> LlMidN;     // 192 x 256, waves of 96 x 64
typedef LlShape<2, 2, 2, 2, 2> LlSmall;    // 128 x 128, waves of 64 x 64
typedef LlShape<4, 1, 1, 1, 4> LlThinN;    // 128 x 32, waves of 32 x 32
typedef LlShape<1, 4, 1, 1, 4> LlThinM;    // 32 x 128

// Teams of `size` workgroups for `ranges` ranges of `units`. Only whole ranges where the last team is not waited for
// longer than a part costs to write and to read again (kPart units); else what is left of them in even shares, a team
// having at least that much in all. (With all ranges shared, two parts a team instead of one, the weight's gradient of
// 8192 x 768 x 50280 took 573 us and 69 us to join, so 557 and 22.)
struct LlTeams {
  int teams, whole, rest;
};

template <class S>
LlTeams ll_teams(int size, int ranges, int units) {
  constexpr int kPart = 8;
  const long long all = static_cast<long long>(ranges) * units;
  long long n = kCUs * S::kPerCU / size;
  n = n < 1 ? 1 : n;
  const long long each = (ranges + n - 1) / n;
  long long shares = all / kPart < n ? all / kPart : n;
  shares = shares < 1 ? 1 : shares;
  if (each * units <= all / shares + kPart)
    return {static_cast<int>((ranges + each - 1) / each), static_cast<int>(each), ranges};
  const int teams = static_cast<int>(shares), whole = ranges / teams;
  return {teams, whole, whole * teams};
}

// How a gradient's product of `rows` by `cols`, its k `stages` long over all pairs of planes, is shared out.
struct LlShare {
  int tiles_m, tiles_n, units, size, ranges;
  LlTeams t;
  long long sums;  // floats of the teams' parts
};

template <class S, int kMode>
LlShare ll_share(int rows, int cols, int stages) {
  LlShare h{};
  h.tiles_m = (rows + S::kM - 1) / S::kM;
  h.tiles_n = (cols + S::kN - 1) / S::kN;
  h.units = (stages + S::kRing - 1) / S::kRing;
  h.size = kMode == kModeDx ? h.tiles_m : h.tiles_n;
  h.ranges = kMode == kModeDx ? h.tiles_n : h.tiles_m;
  h.t = ll_teams<S>(h.size, h.ranges, h.units);
  h.sums = h.t.rest == h.ranges ? 0 : 2LL * h.t.teams * h.size * S::kM * S::kN;
  return h;
}

// The gradients' k is taken up to whole steps of kLlK.
int grad_k(int n) { return (n + kLlK - 1) / kLlK * kLlK; }

// Floats of the parts of one piece's gradients: dx of `features` by `tokens` over `words`, dw of `words` by `features` over
// `tokens`, in tiles of SX and SW.
template <class SX, class SW>
long long part_sums(int features, int tokens, int words, int pairs) {
  return std::max(ll_share<SX, kModeDx>(features, tokens, grad_k(words) / SX::kBK * pairs).sums,
                  ll_share<SW, kModeDw>(words, features, grad_k(tokens) / SW::kBK * pairs).sums);
}

// (A gradient's parts have to fit the workspace that the plan asked for: refused, if they ever should not.)
template <class S, int kMode, bool kF32 = false>
hipError_t launch_product(LlArgs a, const LlOut& o, hipStream_t stream) {
  const int stages = a.k / S::kBK * a.pairs;
  if constexpr (kLlTeams<kMode>) {
    const LlShare h = ll_share<S, kMode>(o.rows, o.cols, stages);
    if (h.sums > a.room) return hipErrorInvalidValue;
    a.tiles_m = h.tiles_m;
    a.tiles_n = h.tiles_n;
    a.units = h.units;
    a.teams = h.t.teams;
    a.whole = h.t.whole;
    a.rest = h.t.rest;
    hipLaunchKernelGGL((ll_kernel<S, kMode, kF32>), dim3(a.teams * h.size), dim3(S::kThreads), 0, stream, a, o);
    const int shared = h.ranges - a.rest;
    if (shared > 0)
      hipLaunchKernelGGL((ll_join_kernel<S, kMode, kF32>), dim3(static_cast<unsigned>(shared) * h.size * S::kWaves * S::kMT),
                         dim3(64 * kJoinWaves), 0, stream, a, o);
  } else {
    a.tiles_m = (o.rows + S::kM - 1) / S::kM;
    a.tiles_n = (o.cols + S::kN - 1) / S::kN;
    a.units = (stages + S::kRing - 1) / S::kRing;
    const int room = kCUs * S::kPerCU;
    const long long tiles = static_cast<long long>(a.tiles_m) * a.tiles_n;
    hipLaunchKernelGGL((ll_kernel<S, kMode, kF32>), dim3(static_cast<unsigned>(tiles < room ? tiles : room)), dim3(S::kThreads), 0,
                       stream, a, o);
  }
  return hipSuccess;
}

// f of the tiles of dx and of dw, as launch_shaped takes them.
template <typename F>
auto with_grad_shapes(int shape_x, int shape_w, F&& f) {
  const auto both = [&](auto x) { return shape_w == 1 ? f(x, LlLargeM{}) : f(x, LlSmall{}); };
  return shape_x == 0 ? both(LlSmall{}) : shape_x == 1 ? both(LlLargeM{}) : both(LlThinN{});
}

template <int kMode, bool kF32>
hipError_t launch_shaped(const LinLossPlan& plan, const LlArgs& a, const LlOut& o, hipStream_t stream) {
  if constexpr (kMode == kModeGrad) {
    if (plan.shape == 0) return launch_product<LlSmall, kMode, kF32>(a, o, stream);
    if (plan.shape == 1) return launch_product<LlLargeN, kMode, kF32>(a, o, stream);
    if (plan.shape == 3) return launch_product<LlMidN, kMode, kF32>(a, o, stream);
    return launch_product<LlThinM, kMode, kF32>(a, o, stream);
  } else if constexpr (kMode == kModeDw) {
    if (plan.shape_w == 1) return launch_product<LlLargeM, kMode, kF32>(a, o, stream);
    return launch_product<LlSmall, kMode, kF32>(a, o, stream);
  } else {
    const int shape = kMode == kModeDx ? plan.shape_x : plan.shape;
    if constexpr (kMode == kModeLse) {
      if (shape == 3) return launch_product<LlMidM, kMode, kF32>(a, o, stream);
    }
    if (shape == 0) return launch_product<LlSmall, kMode, kF32>(a, o, stream);
    if (shape == 1) return launch_product<LlLargeM, kMode, kF32>(a, o, stream);
    return launch_product<LlThinN, kMode, kF32>(a, o, stream);
  }
}

LossMatrix weight_planes(const LinLossParams& p) {
  LossMatrix w{};
  w.base = p.pack_w ? p.wp : static_cast<const bf16_t*>(p.w);
  w.ld = p.pack_w ? p.width : p.ldw;
  w.plane = static_cast<long long>(p.vocab) * p.width;
  w.end = (p.vocab - 1LL) * w.ld + p.width;
  return w;
}

LossMatrix x_planes(const LinLossParams& p) {
  const long long n = static_cast<long long>(p.tokens) * p.width;
  return LossMatrix{p.xp, p.width, n, n};
}

}  // namespace

int loss_target_blocks(int tokens) { return (tokens + 63) / 64; }

static long long tiles_of(long long rows, long long cols, int tm, int tn) {
  return ((rows + tm - 1) / tm) * ((cols + tn - 1) / tn);
}

// Which tiles: the ones whose rounds take the least time, in quarters of a large one's (256 x 256): 3.2 for 256 words
// by 192 tokens, 2.8 for two small ones (128 x 128) on a CU, which reads each operand twice as often and has half
// the products for each of its waits. Up to 32 tokens in thin ones. (us, 333 tokens x 768 x 50280, large, 192, small:
// 46.6, 37.6, 37.0; 256 tokens 26.6, 36.7, 28.8; 128 tokens 25.4, 20.9, 18.7.)
LinLossPlan linloss_plan(int tokens, int features, int vocab, int planes) {
  LinLossPlan q{};
  const auto rounds = [](long long n, long long at_once) { return static_cast<double>((n + at_once - 1) / at_once); };
  if (tokens <= 32) {
    q.shape = 2;
  } else {
    const double large = 4 * rounds(tiles_of(vocab, tokens, 256, 256), kCUs);
    const double mid = 3.2 * rounds(tiles_of(vocab, tokens, 256, 192), kCUs);
    const double small = 2.8 * rounds(tiles_of(vocab, tokens, 128, 128), 2 * kCUs);
    q.shape = large <= small && large <= mid ? 1 : mid <= small ? 3 : 0;
  }
  const int tv = q.shape == 1 || q.shape == 3 ? 256 : 128;
  q.parts = static_cast<int>((vocab + tv - 1) / tv) * (q.shape == 2 || q.shape == 3 ? 4 : 2);
  // Pieces of at most 1 GiB.
  const long long most = (1LL << 30) / (2LL * planes * tokens) / 256 * 256;
  const long long whole = (vocab + 255LL) / 256 * 256;
  const long long pieces = (whole + (most > 256 ? most : 256) - 1) / (most > 256 ? most : 256);
  q.piece = static_cast<int>(((whole / 256 + pieces - 1) / pieces) * 256);
  q.ldg = q.piece;
  q.ldx = (tokens + 3) / 4 * 4;
  const int words = q.piece < vocab ? q.piece : vocab;
  // The gradients' products are shared evenly, so that it is their padding that counts, and for dx of few tokens the
  // parts, of which larger tiles have more (us with the join, large and small, x 768 x 50280: 128 tokens 48 and 37, 256
  // tokens 50 and 45, 384 tokens 67 and 45, 512 tokens 56 and 57, 700 tokens 67 and 92).
  const auto large = [](int rows, int cols) { return 4. * tiles_of(rows, cols, 256, 256) <= 1.4 * tiles_of(rows, cols, 128, 128); };
  q.shape_x = tokens <= 32 ? 2 : tokens > 384 && large(features, tokens) ? 1 : 0;
  q.shape_w = large(words, features) ? 1 : 0;
  // (The last piece may be shorter, and be shared out in another way.)
  const int last = vocab - (vocab - 1) / q.piece * q.piece;
  q.partial = with_grad_shapes(q.shape_x, q.shape_w, [&](auto x, auto w) {
    const auto of = [&](int n) { return part_sums<decltype(x), decltype(w)>(features, tokens, n, planes == 1 ? 1 : kPairs); };
    return std::max(of(words), of(last));
  });
  // Both directions at once, where the logits' product costs more than their 16 bits read and g written, which its
  // features decide, and launches that may not be needed (us of both, apart and at once, x 50280: 4096 x 256 612 and 690;
  // 512 x 768 276 and 276; 1024 x 768 433 and 408; 16384 x 768 4875 and 4536; 2048 x 2560 2071 and 1723; 131072 x
  // 1280 x 260 1200 and 1208).
  q.both = planes == 1 && tokens >= 512 && features >= 640 && vocab >= 1024 && static_cast<long long>(tokens) * vocab >= 1LL << 25;
  if (q.both) {
    q.lde = whole;
    const long long rows = (1LL << 30) / (2 * q.lde) / 256 * 256, blocks = (tokens + rows - 1) / rows;
    q.block = static_cast<int>(((tokens + blocks - 1) / blocks + 255) / 256 * 256);
    const int n = q.block < tokens ? q.block : tokens, last_n = tokens - (tokens - 1) / q.block * q.block;
    const auto of = [&](int t) { return part_sums<LlLargeM, LlLargeM>(features, t, vocab, 1); };
    q.partial_both = std::max(of(n), of(last_n));  // (so may the last block)
    q.parts_both = static_cast<int>(whole / 256) * LlLargeN::kWN;
  }
  return q;
}

// The rows' words, x token-major, the weight's copy where it needs one.
static hipError_t launch_operands(const LinLossParams& p, hipStream_t stream) {
  if (p.r.targets == nullptr) {
    const hipError_t e = launch_loss_rows(p.r, stream);
    if (e != hipSuccess) return e;
  }
  const bool f32 = p.planes == 2;
  const dim3 xg((p.tokens + 63) / 64, p.width / 64);
  if (f32) hipLaunchKernelGGL(ll_max_kernel, dim3(kMaxX + kMaxW), dim3(1024), 0, stream, p);
  if (f32) hipLaunchKernelGGL(ll_pack_x_kernel<float>, xg, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(ll_pack_x_kernel<bf16_t>, xg, dim3(256), 0, stream, p);
  if (p.pack_w) {
    const dim3 wg(blocks_for(static_cast<long long>(p.vocab) * (p.width / 8), 8192));
    if (f32) hipLaunchKernelGGL(ll_pack_w_kernel<float>, wg, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(ll_pack_w_kernel<bf16_t>, wg, dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

// The words' logits (unless they are there), the sums over the vocabulary, the tokens' losses.
static hipError_t launch_losses(const LinLossParams& p, const LinLossPlan& plan, bool picked, hipStream_t stream) {
  const bool f32 = p.planes == 2, lists = p.r.targets == nullptr;
  LlArgs a{};
  a.a = weight_planes(p);
  a.b = x_planes(p);
  a.k = p.width;
  a.pairs = f32 ? kPairs : 1;
  LlOut o{};
  o.rows = p.vocab;
  o.cols = p.tokens;
  o.c = p.c;
  o.part = p.part;
  o.powers = p.powers;
  o.only_if = p.only_if;
  const hipError_t e = f32 ? launch_shaped<kModeLse, true>(plan, a, o, stream) : launch_shaped<kModeLse, false>(plan, a, o, stream);
  if (e != hipSuccess) return e;
  const dim3 fg((p.tokens + kFinishTokens - 1) / kFinishTokens), fb(kFinishTokens * kFinishSlices);
  if (picked) {
    hipLaunchKernelGGL((ll_finish_kernel<false, false>), fg, fb, 0, stream, p, a.a);
  } else if (lists) {
    const long long picks = static_cast<long long>(p.tokens) * ((p.r.top + 3) / 4);
    const dim3 pg(static_cast<unsigned>((picks + 3) / 4));
    if (f32) hipLaunchKernelGGL(ll_pick_kernel<true>, pg, dim3(256), 0, stream, p, a.a, static_cast<float2*>(nullptr), 0);
    else hipLaunchKernelGGL(ll_pick_kernel<false>, pg, dim3(256), 0, stream, p, a.a, static_cast<float2*>(nullptr), 0);
    hipLaunchKernelGGL((ll_finish_kernel<false, false>), fg, fb, 0, stream, p, a.a);
  } else if (f32) {
    hipLaunchKernelGGL((ll_finish_kernel<true, true>), fg, fb, 0, stream, p, a.a);
  } else {
    hipLaunchKernelGGL((ll_finish_kernel<true, false>), fg, fb, 0, stream, p, a.a);
  }
  return hipGetLastError();
}

hipError_t launch_linloss_fwd(const LinLossParams& p, const LinLossPlan& plan, hipStream_t stream) {
  hipError_t e = launch_operands(p, stream);
  if (e == hipSuccess) e = launch_losses(p, plan, false, stream);
  if (e != hipSuccess || p.reduction == kLossNone) return e;
  return launch_loss_mean(p.loss, p.r, p.reduction, p.mean, p.by, stream);
}

hipError_t launch_linloss_bwd(const LinLossParams& p, const LinLossPlan& plan, hipStream_t stream) {
  const bool f32 = p.planes == 2;
  const float2* scale = p.stat;
  if (p.reduction == kLossNone) {
    scale = p.scale;
    if (f32) hipLaunchKernelGGL(ll_scale_kernel<true>, dim3(1), dim3(1024), 0, stream, p, p.scale);
    else hipLaunchKernelGGL(ll_scale_kernel<false>, dim3((p.tokens + 1023) / 1024), dim3(1024), 0, stream, p, p.scale);
  }
  const LossMatrix w = weight_planes(p), x = x_planes(p);
  LlScale by{p.reduction == kLossNone ? nullptr : p.grad, p.reduction == kLossMean ? p.by : nullptr,
             p.reduction == kLossNone ? 1.f : p.temperature,
             nullptr, f32 && p.reduction == kLossNone ? p.power_g : nullptr};
  hipError_t e = hipSuccess;
  for (long long v0 = 0; v0 < p.vocab; v0 += p.piece) {
    const int words = static_cast<int>(p.vocab - v0 < p.piece ? p.vocab - v0 : p.piece);
    LossMatrix wp = w;
    wp.base += v0 * w.ld;
    wp.end -= v0 * w.ld;
    LossMatrix g{};
    g.base = p.g;
    g.ld = p.ldg;
    g.plane = p.tokens * p.ldg;
    g.end = g.plane;
    LlArgs a{};
    a.pairs = f32 ? kPairs : 1;
    // g
    a.a = x;
    a.b = wp;
    a.k = p.width;
    a.partial = p.partial;
    a.room = plan.partial;
    LlOut o{};
    o.rows = p.tokens;
    o.cols = words;
    o.c = p.c;
    o.scale = scale;
    o.g = p.g;
    o.ld = p.ldg;
    o.plane = g.plane;
    o.powers = p.powers;
    e = f32 ? launch_shaped<kModeGrad, true>(plan, a, o, stream) : launch_shaped<kModeGrad, false>(plan, a, o, stream);
    if (e != hipSuccess) return e;
    const dim3 wg(static_cast<unsigned>((static_cast<long long>(p.tokens) * p.r.top + 255) / 256));
    if (f32) hipLaunchKernelGGL(ll_wanted_kernel<true>, wg, dim3(256), 0, stream, p, scale, static_cast<int>(v0), words);
    else hipLaunchKernelGGL(ll_wanted_kernel<false>, wg, dim3(256), 0, stream, p, scale, static_cast<int>(v0), words);
    if (p.dx != nullptr) {
      a.a = wp;
      a.b = g;
      a.k = grad_k(words);
      o = LlOut{};
      o.rows = p.features;
      o.cols = p.tokens;
      o.f = p.dx_sum;
      o.ld = p.ldx;
      o.add = v0 > 0;
      o.powers = p.powers;
      if (v0 + words == p.vocab) {
        o.dx = p.dx;
        o.ld_dx = p.tokens;
        o.dx_bf16 = !f32;
        o.by = by;
        o.by.power = f32 ? p.powers + 1 : nullptr;
        o.live = p.r.live;
      }
      e = f32 ? launch_shaped<kModeDx, true>(plan, a, o, stream) : launch_shaped<kModeDx, false>(plan, a, o, stream);
      if (e != hipSuccess) return e;
    }
    if (p.dw != nullptr) {
      a.a = g;
      a.b = x;
      a.k = grad_k(p.tokens);
      o = LlOut{};
      o.rows = words;
      o.cols = p.features;
      o.ld = p.features;
      o.by = by;
      o.by.power = f32 ? p.powers : nullptr;
      void* dst = static_cast<char*>(p.dw) + v0 * p.features * (p.dw_bf16 ? 2 : 4);
      if (p.dw_bf16) o.h = static_cast<bf16_t*>(dst);
      else o.f = static_cast<float*>(dst);
      e = f32 ? launch_shaped<kModeDw, true>(plan, a, o, stream) : launch_shaped<kModeDw, false>(plan, a, o, stream);
      if (e != hipSuccess) return e;
    }
  }
  return hipGetLastError();
}

hipError_t launch_linloss_both(const LinLossParams& p, const LinLossPlan& plan, hipStream_t stream) {
  hipError_t e = launch_operands(p, stream);
  if (e != hipSuccess) return e;
  e = launch_loss_mean(nullptr, p.r, p.reduction, nullptr, p.by, stream);
  if (e != hipSuccess) return e;
  const LossMatrix w = weight_planes(p);
  const long long picks = static_cast<long long>(p.tokens) * ((p.r.top + 3) / 4);
  hipLaunchKernelGGL(ll_pick_kernel<false>, dim3(static_cast<unsigned>((picks + 3) / 4)), dim3(256), 0, stream, p, w, p.scale,
                     (p.tokens + plan.block - 1) / plan.block);
  const LlScale by{nullptr, p.reduction == kLossMean ? p.by : nullptr, p.temperature, nullptr, nullptr};
  for (int t0 = 0; t0 < p.tokens; t0 += plan.block) {
    LinLossParams b = p;  // of the block's tokens
    b.tokens = b.r.rows = p.tokens - t0 < plan.block ? p.tokens - t0 : plan.block;
    b.r.words += static_cast<long long>(t0) * p.r.top;
    b.r.q += static_cast<long long>(t0) * p.r.top;
    b.picked += static_cast<long long>(t0) * p.r.top;
    b.r.live += t0;
    b.scale += t0;
    b.stat += t0;
    b.loss += t0;
    b.xp += static_cast<long long>(t0) * p.width;
    b.bad += t0 / plan.block;
    const LossMatrix x = x_planes(b), g{b.g, b.ldg, 0, b.tokens * b.ldg};
    LlArgs a{};
    a.pairs = 1;
    a.partial = p.partial;
    a.room = plan.partial_both;
    a.a = x;
    a.b = w;
    a.k = p.width;
    LlOut o{};
    o.rows = b.tokens;
    o.cols = p.vocab;
    o.c = p.c;
    o.scale = b.scale;
    o.g = b.g;
    o.ld = b.ldg;
    o.row_sums = p.row_sums;
    e = launch_product<LlLargeN, kModeExp>(a, o, stream);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(ll_block_kernel, dim3((b.tokens + kFinishTokens - 1) / kFinishTokens),
                       dim3(kFinishTokens * kFinishSlices), 0, stream, b, (p.vocab + 255) / 256 * LlLargeN::kWN);
    hipLaunchKernelGGL(ll_convert_kernel, dim3(b.tokens), dim3(256), 0, stream, b);
    b.only_if = o.only_if = b.bad;
    e = launch_losses(b, plan, true, stream);
    if (e != hipSuccess) return e;
    o.scale = b.stat;
    e = launch_product<LlLargeN, kModeGrad>(a, o, stream);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(ll_wanted_kernel<false>, dim3(static_cast<unsigned>((static_cast<long long>(b.tokens) * p.r.top + 255) / 256)),
                       dim3(256), 0, stream, b, b.stat, 0, p.vocab);
    a.a = w;
    a.b = g;
    a.k = grad_k(p.vocab);
    o = LlOut{};
    o.rows = p.features;
    o.cols = b.tokens;
    o.dx = static_cast<bf16_t*>(p.dx) + t0;
    o.ld_dx = p.tokens;
    o.dx_bf16 = 1;
    o.by = by;
    o.live = b.r.live;
    e = launch_product<LlLargeM, kModeDx>(a, o, stream);
    if (e != hipSuccess) return e;
    a.a = g;
    a.b = x;
    a.k = grad_k(b.tokens);
    o = LlOut{};
    o.rows = p.vocab;
    o.cols = p.features;
    o.ld = p.features;
    o.by = by;
    o.sum = p.tokens > plan.block ? p.dw_sum : nullptr;
    o.add = t0 > 0;
    o.last = t0 + b.tokens == p.tokens;
    if (p.dw_bf16) o.h = static_cast<bf16_t*>(p.dw);
    else o.f = static_cast<float*>(p.dw);
    e = launch_product<LlLargeM, kModeDw>(a, o, stream);
    if (e != hipSuccess) return e;
  }
  return launch_loss_mean(p.loss, p.r, p.reduction, p.mean, p.by, stream);
}

hipError_t launch_linloss_rescale(const LinLossParams& p, hipStream_t stream) {
  const long long nx = static_cast<long long>(p.features) * p.tokens, nw = static_cast<long long>(p.vocab) * p.features;
  hipLaunchKernelGGL(ll_rescale_kernel, dim3(blocks_for(nx > nw ? nx : nw, 4096)), dim3(256), 0, stream,
                     static_cast<bf16_t*>(p.dx), nx, p.dw, p.dw_bf16, nw, p.grad);
  return hipGetLastError();
}

}  // namespace mss
