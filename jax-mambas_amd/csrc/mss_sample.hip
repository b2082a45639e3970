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
// The filters keep a prefix of the order, so they come down to one cut (a logit, and the last
// index kept among the words with that logit), found by radix selection on the logits' order
// in integers, counting words for top-k and adding weights for top-p; nothing is sorted.
// Weights are added as integers of 2^-43, which makes every sum exact and independent of its
// order: at most 2^20 words a row keep it below 2^63.
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

// w = 2^((v - m) c), c = log2(e) / temperature in two float32 parts. The difference and the
// product carry their rounding errors along (they would be the largest of the whole draw:
// 2^-24 of an exponent of 20 is 1e-6 of the weight), the exponential is v_exp_f32's.
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

__device__ __forceinline__ u64 shfl_up64(u64 v, int d) {
  const uint32_t lo = __shfl_up(static_cast<int>(v), d), hi = __shfl_up(static_cast<int>(v >> 32), d);
  return (static_cast<u64>(hi) << 32) | lo;
}
__device__ __forceinline__ u64 wave_incl(u64 v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 o = shfl_up64(v, d);
    if ((threadIdx.x & 63) >= static_cast<unsigned>(d)) v += o;
  }
  return v;
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
      union {
        u32x4 w[sizeof(io_t) / 2];
        io_t e[8];
      } u;
#pragma unroll
      for (int k = 0; k < static_cast<int>(sizeof(io_t) / 2); ++k) u.w[k] = reinterpret_cast<const u32x4*>(x + i)[k];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = to_f32(u.e[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = i + k < vocab ? to_f32(x[(i + k) * sv]) : -__builtin_inff();
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

template <typename io_t, bool kVec>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleParams p) {
  __shared__ SampleShared s;
  const long long r = blockIdx.x;
  const Row<io_t, kVec> row{static_cast<const io_t*>(p.logits) + r * p.sr, p.sv, p.vocab};
  const float temperature = p.temperatures ? p.temperatures[r] : p.temperature;
  const int top_k = p.top_ks ? p.top_ks[r] : p.top_k;
  const float top_p = p.top_ps ? p.top_ps[r] : p.top_p;
  const float min_p = p.min_ps ? p.min_ps[r] : p.min_p;
  const double u = static_cast<double>(p.uniform[r]);

  // The largest logit's key; a NaN counts as the largest of all.
  uint32_t top = 0;
  for (int i = threadIdx.x * 8; i < row.vocab; i += kSampleChunk) {
    float v[8];
    row.load8(i, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, v[k] != v[k] ? 0xffffffffu : order_key(v[k]));
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
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
    for (int i = threadIdx.x * 8; i < row.vocab; i += kSampleChunk) {
      float v[8];
      row.load8(i, v);
      int first = 0x7fffffff;
#pragma unroll
      for (int k = 7; k >= 0; --k)
        if (order_key(v[k]) == top) first = i + k;
      if (first != 0x7fffffff) atomicMin(&s.index, first);
    }
    __syncthreads();
    if (threadIdx.x == 0) p.tokens[r] = s.index;
    return;
  }
  Weight weight;
  weight.set(key_value(top), temperature);

  // The cut: words above its key stay, and those with the key up to its index.
  uint32_t cut_key = kAbsent;
  int cut_index = -1;
  u64 total;
  const bool by_k = top_k > 0 && top_k < p.vocab, by_p = top_p < 1.f;
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
    if (run <= at && at < run + w[k]) p.tokens[r] = i + k;
    run += w[k];
  }
}

template <typename io_t>
static void launch_sample_as(const SampleParams& p, hipStream_t stream) {
  // 16-byte loads where a row's words are contiguous and it starts on 16 bytes.
  const bool vec = p.sv == 1 && (reinterpret_cast<uintptr_t>(p.logits) & 15) == 0 &&
                   (p.sr * static_cast<long long>(sizeof(io_t))) % 16 == 0;
  if (vec) hipLaunchKernelGGL((sample_kernel<io_t, true>), dim3(p.rows), dim3(kSampleThreads), 0, stream, p);
  else hipLaunchKernelGGL((sample_kernel<io_t, false>), dim3(p.rows), dim3(kSampleThreads), 0, stream, p);
}

hipError_t launch_sample(const SampleParams& p, bool io_bf16, hipStream_t stream) {
  if (io_bf16) launch_sample_as<bf16_t>(p, stream);
  else launch_sample_as<float>(p, stream);
  return hipGetLastError();
}

}  // namespace mss
