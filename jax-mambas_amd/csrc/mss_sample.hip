// One token for each row of logits, from given uniform numbers: temperature, top-k, top-p, min-p.
//
// Of a row x (a word whose logit is -inf is absent), with m = max x and the order "larger logit
// first, then lower index":
//   weight    w_i = exp((x_i - m) / temperature)
//   top-k     the first k of the order (0: all)
//   top-p     of those, while the weight before a word is less than top_p of theirs together;
//             the first word always stays
//   min-p     of those, the words with w_i >= min_p; the first word always stays
//   token     the lowest index at which the running sum of the words left, in index order,
//             exceeds u times their sum
// A temperature that is not above zero takes the first word of the order. A row without a
// word, or with a NaN, gives -1.
//
// One workgroup a row. The filters keep a prefix of the order, so they come down to one cut: a
// logit, and the last index kept among the words with that logit. Nothing is sorted:
//
//   1. the largest logit, and the largest of each of three groups a thread. The k-th largest of
//      those is a bound that k words reach and few others do; min-p is a bound by itself.
//   2. the words that reach the bound go into a list in LDS, and the cuts and the draw are found in
//      the list: its weights added into 2048 bins (by logit, or by index for the draw), the bin
//      in which the sum reaches its target, and the few words of that bin one by one.
//      (A row of more words than registers hold is read once for both, its bound taken from its
//      first 16384 words.)
//   3. without such a bound, or when more words reach it than the list holds, the bins are filled
//      from the whole row, and the draw adds the words left by segments of 512.
//   4. where one bin holds too many words (ties), a radix selection on the logits' order in
//      integers takes any row, three passes of 11 bits.
//
// Weights are added as integers of 2^-43, which makes every sum exact and independent of its
// order: at most 2^20 words a row keep it below 2^63. (The one pass adds a thread's weights in
// float64, in the row's order, and makes that an integer: the same from run to run too.)
#include <hip/hip_runtime.h>

#include "mss_serve.h"

namespace mss {

typedef unsigned long long u64;

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kSampleChunk = kSampleThreads * 8;  // words a pass of the workgroup takes at a time
constexpr int kSampleMaxVocab = 1 << 20;
constexpr int kSampleMaxSeg = kSampleMaxVocab / kSampleChunk * kSampleWaves;
constexpr int kSampleBins = 2048;  // 11 bits of the key at a time
constexpr int kSampleRegVocab = 8 * kSampleChunk;  // rows that stay in registers, 64 words a thread
constexpr int kSampleList = 12288;
constexpr int kSampleSmall = 256;                  // words of one bin that are looked at one by one
// A list as short as this needs no bins (50280 words, top-k 100: 14.9 us, by bins 15.8; 200: 22.3, 16.6).
constexpr int kSampleFew = 128;
constexpr int kSampleGroups = 3 * kSampleThreads;  // a thread's chunks c, c + 3, ... have one largest logit
constexpr float kFixed = 8796093022208.f;  // 2^43

// Integers in the order of the floats; -0 and 0 are the same.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t kAbsent = 0x007fffffu;  // order_key(-inf)

// w = 2^((v - m) c), c = log2(e) / temperature in two float32 parts. The product carries its
// rounding error along (c's own would shift all weights the same way), the exponential is
// v_exp_f32's. The difference is rounded, which costs a weight 2^-y at most y ln 2 of 2^-24: words far
// below the largest are a small part of the sum, unless they are many; at worst, a million equal ones at
// y = 20 that outweigh the rest, a sum is off by 2^-20, and a running sum's share of it by half that.
// For 2^-100 < c < 2^100 and finite m only. A word that is absent or below 2^-64 (2^-depth) counts as
// that, which is no unit of the sums.
struct FastWeight {
  float m, c, c_lo, least;
  __device__ __forceinline__ FastWeight(float max, float temperature, float c_, float depth = 64.f) : m(max), c(c_) {
    // what c = log2(e) / temperature lacks (log2(e) = 1.442695022 + 1.92596e-8)
    c_lo = (__builtin_fmaf(-c, temperature, 1.442695022f) + 1.92596301e-8f) / temperature;
    least = -depth / c;
  }
  __device__ __forceinline__ float operator()(float v) const {
    const float d = fmaxf(v - m, least);
    const float y = d * c;
    const float lo = __builtin_fmaf(d, c_lo, __builtin_fmaf(d, c, -y));
    const float e = __builtin_amdgcn_exp2f(y);
    return __builtin_fmaf(e, lo * kLn2, e);
  }
};
// w (at most 1) as an integer of 2^-43, in the low bits of a double of 512 and more.
constexpr u64 kFixedBias = 0x4080000000000000ull;  // 512.0
__device__ __forceinline__ u64 biased_fixed(float w) {
  return __builtin_bit_cast(u64, static_cast<double>(w) + 512.0);
}

// The same for any row (an infinite largest logit, any temperature above zero), the difference's
// rounding error carried along too.
struct Weight {
  float m, c, c_lo;
  __device__ __forceinline__ void set(float max, float temperature) {
    const double cd = 1.4426950408889634 / static_cast<double>(temperature);
    m = max;
    c = cd < 1e30 ? static_cast<float>(cd) : 1e30f;
    c_lo = cd < 1e30 ? static_cast<float>(cd - static_cast<double>(c)) : 0.f;
  }
  __device__ __forceinline__ float operator()(float v) const {
    if (m == __builtin_inff()) return v == m ? 1.f : 0.f;
    const float d = v - m;
    const float bb = d - v;
    const float err = (v - (d - bb)) - (m + bb);
    const float y = d * c;
    if (!(y > -60.f)) return 0.f;  // below 2^-44: not a unit of the sums
    const float lo = __builtin_fmaf(d, c, -y) + __builtin_fmaf(d, c_lo, err * c);
    const float e = __builtin_amdgcn_exp2f(y);
    return __builtin_fmaf(e, lo * kLn2, e);
  }
};
__device__ __forceinline__ u64 fixed(float w) { return static_cast<u64>(__builtin_fmaf(w, kFixed, 0.5f)); }

// Cross-lane sums by DPP moves: a few clocks each, where a shuffle through LDS takes over a hundred.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ u64 dpp64(u64 v) {  // lanes without a source get 0
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, kRowMask, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), kCtrl, kRowMask, 0xF, false);
  return (static_cast<u64>(hi) << 32) | lo;
}
__device__ __forceinline__ u64 readlane64(u64 v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
  return (static_cast<u64>(hi) << 32) | lo;
}
__device__ __forceinline__ u64 wave_incl(u64 v) {
  v += dpp64<kRowShr1, 0xF>(v);
  v += dpp64<kRowShr2, 0xF>(v);
  v += dpp64<kRowShr4, 0xF>(v);
  v += dpp64<kRowShr8, 0xF>(v);
  v += dpp64<kRowBcast15, 0xA>(v);
  v += dpp64<kRowBcast31, 0xC>(v);
  return v;
}
__device__ __forceinline__ u64 wave_total(u64 v) { return readlane64(wave_incl(v), 63); }
template <int kCtrl, int kRowMask>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, kRowMask, 0xF, false)));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = dpp_max<kRowShr1, 0xF>(v);
  v = dpp_max<kRowShr2, 0xF>(v);
  v = dpp_max<kRowShr4, 0xF>(v);
  v = dpp_max<kRowShr8, 0xF>(v);
  v = dpp_max<kRowBcast15, 0xA>(v);
  v = dpp_max<kRowBcast31, 0xC>(v);
  return __builtin_amdgcn_readlane(static_cast<int>(v), 63);
}
__device__ __forceinline__ int words_segments(int vocab) {  // segments that a pass over the row writes
  return (vocab + kSampleChunk - 1) / kSampleChunk * kSampleWaves;
}

struct SampleShared {
  u64 wave[kSampleWaves];
  u64 seg[kSampleMaxSeg];
  u64 mass[kSampleBins];
  uint32_t count[kSampleBins];
  u64 found_above;
  uint32_t found_bin, found_count;
  uint32_t key;
  int index;
  // the list: logits and their words
  float list_v[kSampleList];
  int list_i[kSampleList];
  int list_n, small_n, picked;
  struct alignas(16) Entry {
    u64 w;
    float v;
    int i;
  } small[kSampleSmall];
  u64 sum[kSampleSmall];  // what the entries of `small` before each weigh, and how many they are
  uint32_t rank[kSampleSmall];
};

// Exclusive sum over the workgroup in thread order; `total` gets the whole sum.
__device__ __forceinline__ u64 block_excl(SampleShared& s, u64 v, u64& total) {
  const u64 in = wave_incl(v);
  __syncthreads();  // s.wave's earlier readers are done
  if ((threadIdx.x & 63) == 63) s.wave[threadIdx.x >> 6] = in;
  __syncthreads();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kSampleWaves; ++i) {
    if (i == static_cast<int>(threadIdx.x >> 6)) before = total;
    total += s.wave[i];
  }
  return before + in - v;
}

template <typename io_t, bool kVec>
struct Row {
  const io_t* x;
  long long sv;
  int vocab;
  // Words i .. i + 8; past the row's end they are absent.
  __device__ __forceinline__ void load8(int i, float (&v)[8]) const {
    if (kVec && i + 8 <= vocab) {
      io_t e[8];
      __builtin_memcpy(e, x + i, sizeof(e));
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = to_f32(e[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = i + k < vocab ? to_f32(x[(i + k) * sv]) : -__builtin_inff();
    }
  }
};

// A row's words, 8 at a time to a thread: f(words, index of the first, chunk, chunk % 3 as a type).
// Short rows are read once and stay in registers.
template <int kV>
struct Third {
  static constexpr int value = kV;
};
template <typename io_t, bool kVec, bool kReg>
struct Words {
  static constexpr bool kHeld = kReg;
  Row<io_t, kVec> row;
  float held[kReg ? 8 : 1][8];
  __device__ __forceinline__ void start() {
    if constexpr (kReg) {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c * kSampleChunk < row.vocab) row.load8(c * kSampleChunk + threadIdx.x * 8, held[c]);
    }
  }
  template <typename F>
  __device__ __forceinline__ void chunk(int at, const F& f) const {  // one chunk (the same for a wave)
    const int i = threadIdx.x * 8;
    if constexpr (kReg) {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c == at) f(held[c], c * kSampleChunk + i);
    } else {
      float v[8];
      row.load8(at * kSampleChunk + i, v);
      f(v, at * kSampleChunk + i);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(const F& f) const {
    const int i = threadIdx.x * 8;
    if constexpr (kReg) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if (c * kSampleChunk < row.vocab) {
          if (c % 3 == 0) f(held[c], c * kSampleChunk + i, c, Third<0>());
          else if (c % 3 == 1) f(held[c], c * kSampleChunk + i, c, Third<1>());
          else f(held[c], c * kSampleChunk + i, c, Third<2>());
        }
      }
    } else {  // two chunks ahead
      float v[3][8];
      const int n = (row.vocab + kSampleChunk - 1) / kSampleChunk;
      row.load8(i, v[0]);
      row.load8(kSampleChunk + i, v[1]);
      for (int c = 0; c < n; c += 3) {
        row.load8((c + 2) * kSampleChunk + i, v[2]);
        f(v[0], c * kSampleChunk + i, c, Third<0>());
        if (c + 1 >= n) break;
        row.load8((c + 3) * kSampleChunk + i, v[0]);
        f(v[1], (c + 1) * kSampleChunk + i, c + 1, Third<1>());
        if (c + 2 >= n) break;
        row.load8((c + 4) * kSampleChunk + i, v[1]);
        f(v[2], (c + 2) * kSampleChunk + i, c + 2, Third<2>());
      }
    }
  }
};

// The bin, from the highest on, at which the running sum reaches `target` (1 <= target <= the
// sum): s.found_bin, s.found_above (the sum of the bins above it) and s.found_count.
template <bool kMass>
__device__ __forceinline__ void find_bin(SampleShared& s, u64 target) {
  const int hi = kSampleBins - 1 - 2 * threadIdx.x;
  const u64 a = kMass ? s.mass[hi] : s.count[hi], b = kMass ? s.mass[hi - 1] : s.count[hi - 1];
  u64 total;
  const u64 above = block_excl(s, a + b, total);
  if (above < target && target <= above + a + b) {
    const bool first = target <= above + a;
    s.found_bin = first ? hi : hi - 1;
    s.found_above = first ? above : above + a;
    s.found_count = s.count[first ? hi : hi - 1];
  }
  __syncthreads();
}

// The last word of the order's shortest prefix whose count (or weight) is at least `target`:
// its key, and the last index kept among the words with that key.
template <bool kMass, typename row_t>
__device__ void select(SampleShared& s, const row_t& row, const Weight& weight, u64 target, uint32_t& key, int& index) {
  uint32_t prefix = 0, n = 0;
  u64 above = 0;
#pragma unroll
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, above_shift = level == 0 ? 32 : level == 1 ? 21 : 10;
    const uint32_t mask = level == 2 ? 1023u : 2047u;
    for (int i = threadIdx.x; i < kSampleBins; i += kSampleThreads) {
      s.count[i] = 0;
      s.mass[i] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x * 8; i < row.vocab; i += kSampleChunk) {
      float v[8];
      row.load8(i, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t key_k = order_key(v[k]);
        if (key_k != kAbsent && (level == 0 || (key_k >> (above_shift & 31)) == prefix)) {
          const uint32_t bin = (key_k >> shift) & mask;
          atomicAdd(&s.count[bin], 1u);
          if (kMass) atomicAdd(&s.mass[bin], fixed(weight(v[k])));
        }
      }
    }
    __syncthreads();
    find_bin<kMass>(s, target - above);
    prefix = (prefix << (level == 2 ? 10 : 11)) | s.found_bin;
    above += s.found_above;
    n = s.found_count;
    __syncthreads();
  }
  key = prefix;
  u64 keep = target - above;  // words with that key to keep
  if (kMass) {
    const u64 w = fixed(weight(key_value(key)));
    keep = w ? (keep + w - 1) / w : 1;
  }
  index = 0x7fffffff;
  if (keep >= n) return;
  // The index of the keep-th word with the key: counts by wave and chunk, then word by word.
  for (int i = threadIdx.x * 8, c = 0; c * kSampleChunk < row.vocab; i += kSampleChunk, ++c) {
    float v[8];
    row.load8(i, v);
    int ties = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) ties += order_key(v[k]) == key ? 1 : 0;
    const u64 in = wave_incl(static_cast<u64>(ties));
    if ((threadIdx.x & 63) == 63) s.seg[c * kSampleWaves + (threadIdx.x >> 6)] = in;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    u64 before = 0;
    int g = 0;
    while (before + s.seg[g] < keep) before += s.seg[g++];
    const int i = g * 512 + threadIdx.x * 8;
    float v[8];
    row.load8(i, v);
    int ties = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) ties += order_key(v[k]) == key ? 1 : 0;
    u64 at = before + wave_incl(static_cast<u64>(ties)) - ties;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (order_key(v[k]) == key && ++at == keep) s.index = i + k;
  }
  __syncthreads();
  index = s.index;
  __syncthreads();
}

// The draw of any row, whole passes over it each time.
template <typename row_t>
__device__ __forceinline__ void draw_by_radix(SampleShared& s, const row_t row, uint32_t top, float temperature, int top_k,
                                           float top_p, float min_p, double u, long long* token) {
  Weight weight;
  weight.set(key_value(top), temperature);

  // The cut: words above its key stay, and those with the key up to its index.
  uint32_t cut_key = kAbsent;
  int cut_index = -1;
  u64 total;
  const bool by_k = top_k > 0 && top_k < row.vocab, by_p = top_p < 1.f;
  if (by_k) {
    u64 words = 0;
    for (int i = threadIdx.x * 8; i < row.vocab; i += kSampleChunk) {
      float v[8];
      row.load8(i, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) words += order_key(v[k]) != kAbsent ? 1 : 0;
    }
    block_excl(s, words, total);
    if (total > static_cast<u64>(top_k)) select<false>(s, row, weight, top_k, cut_key, cut_index);
  }
  if (by_p) {
    u64 mine = 0;
    for (int i = threadIdx.x * 8; i < row.vocab; i += kSampleChunk) {
      float v[8];
      row.load8(i, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t key = order_key(v[k]);
        if (key > cut_key || (key == cut_key && i + k <= cut_index)) mine += fixed(weight(v[k]));
      }
    }
    block_excl(s, mine, total);
    const double want = __builtin_ceil((top_p > 0.f ? static_cast<double>(top_p) : 0.0) * static_cast<double>(total));
    u64 target = want < 1.0 ? 1 : static_cast<u64>(want);
    if (target > total) target = total;
    select<true>(s, row, weight, target, cut_key, cut_index);
  }

  // The words left, by wave and chunk in index order, and the draw among them.
  const auto left = [&](float v, int i) -> u64 {
    const uint32_t key = order_key(v);
    if (key < cut_key || (key == cut_key && i > cut_index)) return 0;
    const float w = weight(v);
    return w < min_p ? 0 : fixed(w);  // min_p NaN: no filter
  };
  u64 mine = 0;
  for (int i = threadIdx.x * 8, c = 0; c * kSampleChunk < row.vocab; i += kSampleChunk, ++c) {
    float v[8];
    row.load8(i, v);
    u64 w = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) w += left(v[k], i + k);
    mine += w;
    const u64 in = wave_incl(w);
    if ((threadIdx.x & 63) == 63) s.seg[c * kSampleWaves + (threadIdx.x >> 6)] = in;
  }
  block_excl(s, mine, total);
  if (threadIdx.x >= 64) return;
  // total is at least the first word's 2^43; a number outside [0, 1) takes the nearest end
  u64 at = u >= 1.0 ? total - 1 : u > 0.0 ? static_cast<u64>(u * static_cast<double>(total)) : 0;
  if (at >= total) at = total - 1;
  u64 before = 0;
  int g = 0;
  while (before + s.seg[g] <= at) before += s.seg[g++];
  const int i = g * 512 + threadIdx.x * 8;
  float v[8];
  row.load8(i, v);
  u64 w[8], sum = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) sum += w[k] = left(v[k], i + k);
  u64 run = before + wave_incl(sum) - sum;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (run <= at && at < run + w[k]) *token = i + k;
    run += w[k];
  }
}

// ------------------------------------------------------------------------- bins and the list
// Zeroes the bins; ends with a barrier. Between a reach_bin and the next call lies a barrier.
__device__ __forceinline__ void clear_bins(SampleShared& s) {
  for (int i = threadIdx.x; i < kSampleBins; i += kSampleThreads) s.mass[i] = 0;
  if (threadIdx.x == 0) s.found_bin = kSampleBins;
  __syncthreads();
}

// The first bin at which the running sum reaches the target, which may depend on the whole sum
// (at least 1): its number, the sum before it and the target; kSampleBins where the whole sum does
// not reach it. Begins and ends with a barrier.
template <typename target_t>
__device__ __forceinline__ void reach_bin(SampleShared& s, const target_t& target_of, uint32_t& bin, u64& before,
                                          u64& target) {
  __syncthreads();
  const int at = 2 * threadIdx.x;
  const u64 a = s.mass[at], b = s.mass[at + 1];
  u64 total;
  const u64 excl = block_excl(s, a + b, total);
  target = target_of(total);
  if (excl < target && target <= excl + a + b) {
    const bool first = target <= excl + a;
    s.found_bin = first ? at : at + 1;
    s.found_above = first ? excl : excl + a;
  }
  __syncthreads();
  bin = s.found_bin;
  before = s.found_above;
}

// Bins by logit: monotone in it, the largest in bin 0.
struct ByLogit {
  float m, scale;
  __device__ __forceinline__ ByLogit(float max, float least) : m(max), scale(0.f) {
    const float range = max - least;  // the least logit's bin is the last
    if (range > 0.f) scale = (kSampleBins - 1) / range;
    if (!(scale < 1e37f)) scale = 0.f;  // (a range too small to divide by: one bin)
  }
  __device__ __forceinline__ uint32_t bin(float v, int) const {
    return static_cast<uint32_t>(fminf((v - m) * -scale, static_cast<float>(kSampleBins - 1)));
  }
  static __device__ __forceinline__ bool before(float v, int i, float w, int j) { return v > w || (v == w && i < j); }
};
struct ByIndex {
  int shift;
  __device__ __forceinline__ explicit ByIndex(int vocab) : shift(max(0, 21 - __clz(vocab))) {}  // vocab >> shift < 2048
  __device__ __forceinline__ uint32_t bin(float, int i) const { return static_cast<uint32_t>(i) >> shift; }
  static __device__ __forceinline__ bool before(float, int i, float, int j) { return i < j; }
};

// For each of the n entries of s.small (written before the call), the sum and the number of those
// before it in `order`: s.sum, s.rank. Every wave looks at a sixteenth of them for all (a thread
// that walked through all n alone took 70 ns an entry). Begins and ends with a barrier.
template <typename order_t>
__device__ __forceinline__ void places(SampleShared& s, int n, const order_t& order) {
  if (static_cast<int>(threadIdx.x) < n) {
    s.sum[threadIdx.x] = 0;
    s.rank[threadIdx.x] = 0;
  }
  __syncthreads();
  for (int t = threadIdx.x & 63; t < n; t += 64) {
    const SampleShared::Entry mine = s.small[t];
    u64 sum = 0;
    uint32_t rank = 0;
#pragma unroll 4
    for (int k = threadIdx.x >> 6; k < n; k += kSampleWaves) {
      const SampleShared::Entry o = s.small[k];
      const bool first = order.before(o.v, o.i, mine.v, mine.i);
      sum += first ? o.w : 0;
      rank += first ? 1u : 0u;
    }
    if (rank) {
      atomicAdd(&s.sum[t], sum);
      atomicAdd(&s.rank[t], rank);
    }
  }
  __syncthreads();
}

// Of the list's words in bin `bin` of `order`, the one at which the running weight reaches
// `target`, `before` being the weight of the bins before; false where they are too many. Every
// thread gets it. (Where false is returned, s.small_n has been read behind the last barrier: the caller
// meets again before anything else is done with the list.)
template <typename order_t, typename weight_t>
__device__ __forceinline__ bool settle(SampleShared& s, int n, const order_t& order, const weight_t& weight, uint32_t bin,
                                       u64 before, u64 target, float& v, int& i) {
  if (threadIdx.x == 0) s.small_n = 0;
  __syncthreads();
  for (int e = threadIdx.x; e < n; e += kSampleThreads) {
    if (order.bin(s.list_v[e], s.list_i[e]) != bin) continue;
    const u64 w = weight(e);
    if (w) {
      const int at = atomicAdd(&s.small_n, 1);
      if (at < kSampleSmall) s.small[at] = SampleShared::Entry{w, s.list_v[e], s.list_i[e]};
    }
  }
  __syncthreads();
  const int few = s.small_n;
  if (few > kSampleSmall) return false;
  places(s, few, order);
  if (static_cast<int>(threadIdx.x) < few) {
    const u64 sum = before + s.sum[threadIdx.x];
    if (sum < target && target <= sum + s.small[threadIdx.x].w) s.picked = threadIdx.x;
  }
  __syncthreads();
  v = s.small[s.picked].v;
  i = s.small[s.picked].i;
  __syncthreads();
  return true;
}
// The same with bins filled from the list.
template <typename order_t, typename weight_t, typename target_t>
__device__ __forceinline__ bool pick(SampleShared& s, int n, const order_t& order, const weight_t& weight,
                                     const target_t& target_of, float& v, int& i) {
  clear_bins(s);
  for (int e = threadIdx.x; e < n; e += kSampleThreads) {
    const u64 w = weight(e);
    if (w) atomicAdd(&s.mass[order.bin(s.list_v[e], s.list_i[e])], w);
  }
  uint32_t bin;
  u64 before, target;
  reach_bin(s, target_of, bin, before, target);
  return settle(s, n, order, weight, bin, before, target, v, i);
}

// Puts those of a thread's 8 words into the list that `takes` says, a wave's at once: one atomic for
// its places. By whole waves.
template <typename takes_t>
__device__ __forceinline__ void append(SampleShared& s, const float (&v)[8], int i, const takes_t& takes) {
  u64 mask[8], any = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) any |= mask[k] = __ballot(takes(v[k], i + k));
  if (any == 0) return;
  int n = 0, at = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) n += __popcll(mask[k]);
  if ((threadIdx.x & 63) == 0) at = atomicAdd(&s.list_n, n);
  at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (mask[k]) {
      const int mine = at + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask[k] >> 32),
                                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask[k]), 0));
      if ((mask[k] >> (threadIdx.x & 63) & 1) && mine < kSampleList) {
        s.list_v[mine] = v[k];
        s.list_i[mine] = i + k;
      }
      at += __popcll(mask[k]);
    }
  }
}

// The prefix of the order that a filter leaves: words above v, and those with it up to index i.
struct Cut {
  float v;
  int i;
  __device__ __forceinline__ bool keeps(float x, int at) const { return x > v || (x == v && at <= i); }
};

__device__ __forceinline__ u64 block_total(SampleShared& s, u64 v) {
  v = wave_total(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int i = 0; i < kSampleWaves; ++i) t += s.wave[i];
  return t;
}

__device__ __forceinline__ u64 reach_of(float top_p, u64 total) {  // the sum at which top-p's prefix ends
  const double want = __builtin_ceil((top_p > 0.f ? static_cast<double>(top_p) : 0.0) * static_cast<double>(total));
  const u64 t = want < 1.0 ? 1 : static_cast<u64>(want);
  return t > total ? total : t;
}
// u of `total` as an integer below it; a number outside [0, 1) takes the nearest end.
__device__ __forceinline__ u64 draw_of(double u, u64 total) {
  const u64 at = u >= 1.0 ? total - 1 : u > 0.0 ? static_cast<u64>(u * static_cast<double>(total)) : 0;
  return at >= total ? total - 1 : at;
}

// A logit that all words of the bins up to `bin` reach.
__device__ __forceinline__ float low_of_bin(const ByLogit& order, uint32_t bin, float m, float least) {
  return bin < kSampleBins && order.scale > 0.f ? fmaxf(least, m - (bin + 1.01f) / order.scale) : least;
}
// The share of a row's words whose list top-p's prefix is guessed to lie in.
__device__ __forceinline__ float share_of(float top_p, int vocab) {
  return fminf(top_p <= 0.6f ? 0.005f : top_p <= 0.85f ? 0.02f : top_p <= 0.92f ? 0.05f : 0.1f,
               kSampleList * 0.85f / vocab);
}

// The list made in one pass, of a row that is not held: the bound comes from the first two chunks
// (top-p's prefix is guessed at also where min-p would bound the list: some rows' first chunks have
// no large logit), the weights of the row's sum are added before the row's largest logit is known and
// put right afterwards. 256 x 131072 float32: top-k 50 45 us with a pass for the largest logit and
// one for the list, 36 with one; top-p 0.9 64 and 48, with min-p 0.001 58 and 50.
struct OnePass {
  bool done;       // else the list does not hold the words, or the row is none to do this with
  bool nan;
  float m, low;    // the row's largest logit, and the bound
  u64 all;
};
template <typename words_t>
__device__ __forceinline__ OnePass list_in_one_pass(SampleShared& s, const words_t& words, float temperature, float c,
                                                    int top_k, float top_p, float min_p) {
  const int vocab = words.row.vocab;
  const bool by_k = top_k > 0 && top_k < vocab, by_p = top_p < 1.f, by_m = min_p > 0.f;
  OnePass out{false, false, 0.f, 0.f, 0};
  float most[2] = {-__builtin_inff(), -__builtin_inff()};
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    float v[8];
    words.row.load8(q * kSampleChunk + threadIdx.x * 8, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) most[q] = fmaxf(most[q], v[k]);
  }
  const auto top_of = [&](float v) {
    uint32_t top = wave_max(order_key(v));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSampleWaves; ++i) top = max(top, static_cast<uint32_t>(s.wave[i]));
    return key_value(top);
  };
  const float m = top_of(fmaxf(most[0], most[1])), least = m - 46.f / c;
  if (!(least > -__builtin_inff() && m < __builtin_inff())) return out;
  out.low = by_m ? fmaxf(least, m + (__builtin_amdgcn_logf(min_p) - 0.01f) / c) : least;
  {
    const ByLogit order(m, least);
    clear_bins(s);
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (most[q] >= least) atomicAdd(reinterpret_cast<uint32_t*>(&s.mass[order.bin(most[q], 0)]), 1u);
    const float guess = share_of(by_p ? top_p : 1.f, vocab) * 8;  // words a group
    const int k = by_k ? top_k : max(1, static_cast<int>(2 * kSampleThreads * (1.f - __builtin_amdgcn_exp2f(-guess / kLn2))));
    uint32_t bin;
    u64 before, target;
    reach_bin(s, [&](u64) -> u64 { return k; }, bin, before, target);
    const float reach = low_of_bin(order, bin, m, least);
    if (!by_k && !by_p && reach > out.low) return out;  // min-p alone needs all of its words
    out.low = fmaxf(reach, by_k && by_p ? least : out.low);
  }
  if (threadIdx.x == 0) s.list_n = 0;
  __syncthreads();
  // The weights are relative to 2^0 where the logits allow it, else to that largest one: no difference
  // that is rounded lies between a word that counts and the row's own largest logit. (From 0 there is none;
  // from m, at m c beyond 40, it is exact for logits between m and twice, or half, of it, and words below
  // do not count. Rows whose largest is further off are left to the exact sum.)
  const bool plain = m * c >= -40.f && m * c <= 60.f;
  const float from = plain ? 0.f : m;
  const FastWeight weight(from, temperature, c, plain ? 120.f : 64.f);
  const bool whole = by_p && !by_k;
  double all = 0;
  float mine = m;
  bool nan = false;
  words.each([&](const float (&v)[8], int i, int, auto) {
    append(s, v, i, [&](float x, int) { return x >= out.low; });
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      mine = fmaxf(fmaxf(mine, v[k]), v[k + 1]);
      nan |= __builtin_isunordered(v[k], v[k + 1]);
    }
    if (whole) {
#pragma unroll
      for (int k = 0; k < 8; ++k) all += static_cast<double>(weight(v[k]));
    }
  });
  out.m = top_of(mine);
  out.nan = __syncthreads_or(nan);
  const bool exact = plain || out.m == m || out.m <= (m > 0.f ? 2.f * m : 0.5f * m);
  out.done = s.list_n <= kSampleList && (out.m - m) * c < 60.f && (exact || !whole);
  const FastWeight shift(out.m, temperature, c, 126.f);
  if (whole) out.all = block_total(s, out.done ? static_cast<u64>(all * (static_cast<double>(shift(from)) * kFixed)) : 0);
  return out;
}

// The token, or -1 where a bin holds too many words to look at one by one.
template <typename words_t>
__device__ __forceinline__ int draw_by_bins(SampleShared& s, const words_t& words, const float (&most)[3], const OnePass& made,
                                            float m, float temperature, float c, int top_k, float top_p, float min_p, double u) {
  const int vocab = words.row.vocab;
  const FastWeight weight(m, temperature, c);
  const auto fixed = [&](float v) { return biased_fixed(weight(v)) - kFixedBias; };
  const bool by_k = top_k > 0 && top_k < vocab, by_p = top_p < 1.f, by_m = min_p > 0.f;
  // Words below `least` weigh nothing. (At a high temperature that is far below them all.)
  float least = m - 46.f / c;
  if (c < 0.25f) {
    float mine = m;
    words.each([&](const float (&v)[8], int, int, auto) {
#pragma unroll
      for (int k = 0; k < 8; ++k) mine = fminf(mine, v[k] > -__builtin_inff() ? v[k] : mine);
    });
    uint32_t last = wave_max(~order_key(mine));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave[threadIdx.x >> 6] = last;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSampleWaves; ++i) last = max(last, static_cast<uint32_t>(s.wave[i]));
    least = fmaxf(least, key_value(~last));
  }
  const float m_bound = by_m ? fmaxf(least, m + (__builtin_amdgcn_logf(min_p) - 0.01f) / c) : least;  // just below min-p's

  // The list of the words that matter, where there is a bound for them: the bin that the k-th
  // largest of the groups' largest logits lies in. (Top-p counts all of top-k's words, also those
  // below min-p.) Where top-p counts the whole row, its sum is taken in the same pass, and
  // without min-p the bound is a guess at its prefix: one that a share of the words reaches which
  // grows with top_p. (Rows in registers need no guess: their bins are filled from the whole row.)
  const ByLogit order(m, least);
  const auto low_of = [&](uint32_t bin) { return low_of_bin(order, bin, m, least); };
  const int groups = min(kSampleGroups, (vocab + 7) / 8);
  const bool listed = by_k ? top_k <= kSampleGroups * 15 / 16 : by_m || (by_p && !words_t::kHeld);
  const bool whole = listed && by_p && !by_k;
  int n = kSampleList + 1;
  float low = m_bound;
  u64 all = 0;
  Cut cut{-__builtin_inff(), 0x7fffffff};
  if (made.done) {
    n = s.list_n;
    low = made.low;
    all = made.all;
  } else if (listed) {
    if (threadIdx.x == 0) s.list_n = 0;
    if (by_k || !by_m) {
      clear_bins(s);
#pragma unroll
      for (int q = 0; q < 3; ++q)
        if (most[q] >= least) atomicAdd(reinterpret_cast<uint32_t*>(&s.mass[order.bin(most[q], 0)]), 1u);
      const float guess = share_of(top_p, vocab) * vocab / groups;  // words a group
      const int k = by_k ? top_k : max(1, static_cast<int>(groups * (1.f - __builtin_amdgcn_exp2f(-guess / kLn2))));
      uint32_t bin;
      u64 before, target;
      reach_bin(s, [&](u64) -> u64 { return k; }, bin, before, target);
      low = fmaxf(low_of(bin), by_k && by_p ? least : m_bound);
    }
    __syncthreads();
    words.each([&](const float (&v)[8], int i, int, auto) {
      append(s, v, i, [&](float x, int) { return x >= low; });
      if (whole) {
#pragma unroll
        for (int k = 0; k < 8; ++k) all += biased_fixed(weight(v[k]));
        all -= 8 * kFixedBias;
      }
    });
    __syncthreads();
    n = s.list_n;
    if (whole) all = block_total(s, all);
  }
  if (n <= kSampleFew) {  // all in one: a word a thread, its place and the weight before it by looking at every other
    const int t = threadIdx.x;
    SampleShared::Entry mine{0, 0.f, 0};
    if (t < n) s.small[t] = mine = SampleShared::Entry{fixed(s.list_v[t]), s.list_v[t], s.list_i[t]};
    places(s, n, order);
    const int rank = t < n ? s.rank[t] : 0;
    const u64 before = t < n ? s.sum[t] : 0;
    bool keep = t < n && (!by_k || rank < top_k), found = true;
    if (by_p) {
      const u64 here = block_total(s, keep ? mine.w : 0), target = reach_of(top_p, whole ? all : here);
      keep = keep && before < target;
      found = target <= here || (by_m && low <= m_bound);
    }
    if (found) {
      keep = keep && !(weight(mine.v) < min_p);
      const u64 at = draw_of(u, block_total(s, keep ? mine.w : 0));
      if (t < n) s.small[t].w = keep ? mine.w : 0;
      places(s, n, ByIndex(vocab));
      if (keep && s.sum[t] <= at && at < s.sum[t] + mine.w) s.picked = mine.i;
      __syncthreads();
      return s.picked;
    }
    __syncthreads();
  }
  const auto draw_listed = [&](int n) {  // among the list's words that the cut and min-p leave
    const auto drawn = [&](int e) -> u64 {
      const float w = weight(s.list_v[e]);
      return cut.keeps(s.list_v[e], s.list_i[e]) && !(w < min_p) ? biased_fixed(w) - kFixedBias : 0;
    };
    float v;
    int i;
    return pick(s, n, ByIndex(vocab), drawn, [&](u64 total) { return draw_of(u, total) + 1; }, v, i) ? i : -1;
  };
  if (n > kSampleFew && n <= kSampleList) {
    const ByLogit order(m, low);
    const auto kept = [&](int e) { return cut.keeps(s.list_v[e], s.list_i[e]) ? fixed(s.list_v[e]) : 0; };
    if (by_k && n > top_k) {
      if (!pick(s, n, order, [](int) -> u64 { return 1; }, [&](u64) -> u64 { return top_k; }, cut.v, cut.i)) return -1;
    }
    bool found = true;
    if (by_p) {
      u64 mine = 0;
      for (int e = threadIdx.x; e < n; e += kSampleThreads) mine += kept(e);
      const u64 here = block_total(s, mine), target = reach_of(top_p, whole ? all : here);
      if (target <= here) {
        Cut to{0.f, 0};
        if (!pick(s, n, order, kept, [&](u64) { return target; }, to.v, to.i)) return -1;
        cut = to;
      } else {
        found = by_m && low <= m_bound;  // all of min-p's words are here, and top-p leaves more
      }
    }
    if (found) return draw_listed(n);
  }

  // No list: the cuts from bins of the whole row. (gather begins and ends with a barrier: every thread
  // has read the length of the list before, which is returned behind the last one, when it is cleared.)
  const auto gather = [&](const auto& takes) {
    __syncthreads();
    if (threadIdx.x == 0) s.list_n = 0;
    __syncthreads();
    words.each([&](const float (&v)[8], int i, int, auto) { append(s, v, i, takes); });
    __syncthreads();
    return s.list_n;
  };
  uint32_t bin;
  u64 before, target;
  const auto in_bin = [&](float x, int at) { return x >= least && order.bin(x, 0) == bin && cut.keeps(x, at); };
  if (by_k) {
    clear_bins(s);
    words.each([&](const float (&v)[8], int, int, auto) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (v[k] >= least) atomicAdd(reinterpret_cast<uint32_t*>(&s.mass[order.bin(v[k], 0)]), 1u);
    });
    reach_bin(s, [&](u64) -> u64 { return top_k; }, bin, before, target);
    if (bin < kSampleBins) {  // else top-k's words include all that weigh anything
      const int g = gather(in_bin);
      if (g > kSampleList || !settle(s, g, order, [](int) -> u64 { return 1; }, bin, before, target, cut.v, cut.i)) return -1;
    }
    __syncthreads();  // found_bin has been read
  }
  if (by_p) {
    clear_bins(s);
    words.each([&](const float (&v)[8], int i, int, auto) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const u64 w = !by_k || cut.keeps(v[k], i + k) ? fixed(v[k]) : 0;
        if (w) atomicAdd(&s.mass[order.bin(v[k], 0)], w);
      }
    });
    reach_bin(s, [&](u64 total) { return reach_of(top_p, total); }, bin, before, target);
    if (bin >= kSampleBins) return -1;
    const auto weigh = [&](int e) { return cut.keeps(s.list_v[e], s.list_i[e]) ? fixed(s.list_v[e]) : 0; };
    const float reach = low_of(bin);
    const int g = gather([&](float x, int) { return x >= reach; });
    Cut to{0.f, 0};
    if (g <= kSampleList) {  // the whole prefix fits the list: the draw is made there
      if (!settle(s, g, order, weigh, bin, before, target, to.v, to.i)) return -1;
      cut = to;
      return draw_listed(g);
    }
    const int h = gather(in_bin);
    if (h > kSampleList || !settle(s, h, order, weigh, bin, before, target, to.v, to.i)) return -1;
    cut = to;
  }

  // The draw: the words left by segments of 512 in index order, and one of them.
  const auto left = [&](float v, int i) -> u64 {
    const float w = weight(v);
    return cut.keeps(v, i) && !(w < min_p) ? biased_fixed(w) - kFixedBias : 0;
  };
  const bool filtered = by_k || by_p || by_m;
  u64 mine = 0;
  words.each([&](const float (&v)[8], int i, int c, auto) {
    u64 w = 0;
    if (filtered) {
#pragma unroll
      for (int k = 0; k < 8; ++k) w += left(v[k], i + k);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w += biased_fixed(weight(v[k]));
      w -= 8 * kFixedBias;
    }
    mine += w;
    w = wave_total(w);
    if ((threadIdx.x & 63) == 0) s.seg[c * kSampleWaves + (threadIdx.x >> 6)] = w;
  });
  const u64 at = draw_of(u, block_total(s, mine));
  // Every wave finds the segment, 64 at a time, and the one that holds it the word.
  before = 0;
  int g = 0;
  while (g < words_segments(vocab)) {
    const int lane = threadIdx.x & 63;
    const u64 in = wave_incl(g + lane < words_segments(vocab) ? s.seg[g + lane] : 0);
    const u64 hit = __ballot(before + in > at);
    if (hit) {
      const int first = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<long long>(hit)) - 1);
      g += first;
      if (first) before += readlane64(in, first - 1);
      break;
    }
    before += readlane64(in, 63);
    g += 64;
  }
  if (g % kSampleWaves == __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6))) {
    words.chunk(g / kSampleWaves, [&](const float (&v)[8], int i) {
      u64 w[8], sum = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += w[k] = left(v[k], i + k);
      u64 run = before + wave_incl(sum) - sum;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (run <= at && at < run + w[k]) s.index = i + k;
        run += w[k];
      }
    });
  }
  __syncthreads();
  return s.index;
}

template <typename io_t, bool kVec, bool kReg>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleParams p) {
  __shared__ SampleShared s;
  const long long r = blockIdx.x;
  Words<io_t, kVec, kReg> words;
  words.row = Row<io_t, kVec>{static_cast<const io_t*>(p.logits) + r * p.sr, p.sv, p.vocab};
  words.start();
  const float temperature = p.temperatures ? p.temperatures[r] : p.temperature;
  const int top_k = p.top_ks ? p.top_ks[r] : p.top_k;
  const float top_p = p.top_ps ? p.top_ps[r] : p.top_p;
  const float min_p = p.min_ps ? p.min_ps[r] : p.min_p;
  const double u = static_cast<double>(p.uniform[r]);

  const float c = 1.442695022f / temperature;
  OnePass made{false, false, 0.f, 0.f, 0};
  if constexpr (!kReg) {
    // (top-k's words: eight times as many and more reach the bound that the first chunks give them)
    const bool by_k = top_k > 0 && top_k < p.vocab;
    const bool fits = by_k ? static_cast<long long>(top_k) * p.vocab <= kSampleList * 3ll / 4 * kSampleChunk && top_k <= kSampleThreads
                           : top_p < 1.f || min_p > 0.f;
    if (fits && temperature > 0.f && top_k != 1 && !(min_p > 1.f) && c >= 0.25f && c < 0x1p100f)
      made = list_in_one_pass(s, words, temperature, c, top_k, top_p, min_p);
    __syncthreads();  // s.wave has been read
  }
  if (made.done) {
    const float none[3] = {};
    const int token = made.nan ? -1 : draw_by_bins(s, words, none, made, made.m, temperature, c, top_k, top_p, min_p, u);
    if (token >= 0 || made.nan) {
      if (threadIdx.x == 0) p.tokens[r] = token;
      return;
    }
    __syncthreads();
  }

  // The largest logit of each group, and whether any is NaN.
  float most[3] = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
  bool nan = false;
  words.each([&](const float (&v)[8], int, int, auto third) {
    float& mine = most[decltype(third)::value];
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      mine = fmaxf(fmaxf(mine, v[k]), v[k + 1]);
      nan |= __builtin_isunordered(v[k], v[k + 1]);
    }
  });
  const uint32_t my_top = nan ? 0xffffffffu : order_key(fmaxf(fmaxf(most[0], most[1]), most[2]));
  uint32_t top = my_top;
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) s.wave[threadIdx.x >> 6] = top;
  if (threadIdx.x == 0) s.index = 0x7fffffff;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSampleWaves; ++i) top = max(top, static_cast<uint32_t>(s.wave[i]));
  if (top == 0xffffffffu || top <= kAbsent) {
    if (threadIdx.x == 0) p.tokens[r] = -1;
    return;
  }
  if (!(temperature > 0.f) || top_k == 1 || min_p > 1.f) {  // the first word of the order
    if (my_top == top) {
      words.each([&](const float (&v)[8], int i, int, auto) {
        int first = 0x7fffffff;
#pragma unroll
        for (int k = 7; k >= 0; --k)
          if (order_key(v[k]) == top) first = i + k;
        if (first != 0x7fffffff) atomicMin(&s.index, first);
      });
    }
    __syncthreads();
    if (threadIdx.x == 0) p.tokens[r] = s.index;
    return;
  }
  const float m = key_value(top);
  if (m < __builtin_inff() && c > 0x1p-100f && c < 0x1p100f && m - 46.f / c > -__builtin_inff()) {
    const int token = draw_by_bins(s, words, most, OnePass{}, m, temperature, c, top_k, top_p, min_p, u);
    if (token >= 0) {
      if (threadIdx.x == 0) p.tokens[r] = token;
      return;
    }
    __syncthreads();
  }
  draw_by_radix(s, words.row, top, temperature, top_k, top_p, min_p, u, p.tokens + r);
}

template <typename io_t>
static void launch_sample_as(const SampleParams& p, hipStream_t stream) {
  const dim3 grid(p.rows), block(kSampleThreads);
  if (p.sv == 1 && p.vocab <= kSampleRegVocab) hipLaunchKernelGGL((sample_kernel<io_t, true, true>), grid, block, 0, stream, p);
  else if (p.sv == 1) hipLaunchKernelGGL((sample_kernel<io_t, true, false>), grid, block, 0, stream, p);
  else if (p.vocab <= kSampleRegVocab) hipLaunchKernelGGL((sample_kernel<io_t, false, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((sample_kernel<io_t, false, false>), grid, block, 0, stream, p);
}

// A launch has fewer than 2^32 threads along x: rows beyond kSampleLaunchRows take another one.
constexpr int kSampleLaunchRows = 1 << 21;

hipError_t launch_sample(const SampleParams& p, bool io_bf16, hipStream_t stream) {
  SampleParams part = p;
  for (long long r = 0; r < p.rows; r += kSampleLaunchRows) {
    part.rows = static_cast<int>(p.rows - r < kSampleLaunchRows ? p.rows - r : kSampleLaunchRows);
    part.logits = static_cast<const char*>(p.logits) + r * p.sr * (io_bf16 ? 2 : 4);
    part.uniform = p.uniform + r;
    part.temperatures = p.temperatures ? p.temperatures + r : nullptr;
    part.top_ks = p.top_ks ? p.top_ks + r : nullptr;
    part.top_ps = p.top_ps ? p.top_ps + r : nullptr;
    part.min_ps = p.min_ps ? p.min_ps + r : nullptr;
    part.tokens = p.tokens + r;
    if (io_bf16) launch_sample_as<bf16_t>(part, stream);
    else launch_sample_as<float>(part, stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mss
