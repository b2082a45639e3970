// Rows' wanted words (mss_loss.h), and the loss towards them from logits at hand, with its gradient:
// the softmax's temperature, lists of words with a teacher's logits, rows that do not count.
//
// The loss is bound by memory: a row is read once into the registers of 1, 4 or 16 waves (up to 65536
// words), and where the loss will be differentiated its gradient is written from there; longer rows are read
// twice. A row's largest logit is subtracted before anything is scaled, so that logits of the type's
// lowest value are words of no weight.
#include <hip/hip_runtime.h>

#include "mss_loss.h"

namespace mss {

namespace {

__device__ __forceinline__ float wave_max_f(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
  return v;
}

__device__ __forceinline__ float wave_sum_f(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// ------------------------------------------------------------------------- the rows' wanted words
constexpr int kListRows = 4;  // rows a workgroup

// A wave a row, kPer entries a lane (entry 64 i + lane). An entry counts where its id is not negative and its
// logit not -inf; what an entry that does not count holds is not looked at. A word that stands in a list
// more than once has the sum of its entries, in the first one's place.
// (Whether one does, a table in LDS tells: four places an entry, each word put in the first free one from its own on.)
template <int kPer>
__global__ __launch_bounds__(64 * kListRows) void loss_lists_kernel(LossRows r) {
  constexpr int kPlaces = 256 * kPer;
  __shared__ int s_n[kListRows];
  __shared__ int s_table[kListRows][kPlaces];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const long long t = static_cast<long long>(blockIdx.x) * kListRows + w;
  bool any = false;
  if (t < r.rows) {
    int word[kPer];
    float z[kPer];
    float top = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int k = 64 * i + lane;
      word[i] = -1;
      z[i] = -INFINITY;
      if (k < r.top) {
        const long long at = t * r.top + k;
        const long long id = r.ids[at];
        const float v = r.teacher_bf16 ? to_f32(static_cast<const bf16_t*>(r.teacher)[at])
                                       : static_cast<const float*>(r.teacher)[at];
        if (id >= 0 && v != -INFINITY) {
          any = true;
          bad |= id >= r.vocab || !(v < INFINITY);
          word[i] = id < r.vocab ? static_cast<int>(id) : -1;
          z[i] = v;
          top = fmaxf(top, v);
        }
      }
    }
    top = wave_max_f(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      z[i] = word[i] >= 0 ? fast_exp2((z[i] - top) * r.c) : 0.f;
      sum += z[i];
    }
    sum = wave_sum_f(sum);
    const float by = 1.f / sum;
    float q[kPer];
    bool first[kPer], again = false;
    int* table = s_table[w];
#pragma unroll
    for (int i = 0; i < kPlaces / 64; ++i) table[64 * i + lane] = -1;
    __builtin_amdgcn_wave_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      q[i] = z[i];
      first[i] = true;
      if (word[i] < 0) continue;
      uint32_t at = static_cast<uint32_t>(word[i]) * 2654435761u >> 16;
      for (int tries = 0; tries < kPlaces; ++tries, ++at) {
        const int was = atomicCAS(table + at % kPlaces, -1, word[i]);
        again |= was == word[i];
        if (was == -1 || was == word[i]) break;
      }
    }
    again = __any(again);
    if (again) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) q[i] = 0.f;
    }
#pragma unroll
    for (int a = 0; a < kPer; ++a) {
      if (!again) break;
      const int n = min(64, r.top - 64 * a);
      for (int l = 0; l < n; ++l) {
        const int other = __builtin_amdgcn_readlane(word[a], l);
        const float oz = readlane(z[a], l);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (word[i] != other) continue;
          q[i] += oz;
          if (64 * a + l < 64 * i + lane) first[i] = false;
        }
      }
    }
    any = __any(any);
    bad = __any(bad);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int k = 64 * i + lane;
      if (k >= r.top) continue;
      const float v = q[i] * by;
      // (less than the least normal float is nothing: its logarithm would not be one)
      const bool held = word[i] >= 0 && first[i] && v >= 1.1754943508222875e-38f;
      r.words[t * r.top + k] = held ? word[i] : -1;
      r.q[t * r.top + k] = held ? v : 0.f;
    }
    if (lane == 0) r.live[t] = !any ? 0.f : bad ? __builtin_nanf("") : 1.f;
  }
  if (lane == 0) s_n[w] = any;
  __syncthreads();
  if (threadIdx.x == 0) {
    int all = 0;
    for (int i = 0; i < kListRows; ++i) all += s_n[i];
    r.counts[blockIdx.x] = all;
  }
}

// The reduced loss, and what a mean divides by (that alone without losses).
__global__ __launch_bounds__(1024) void loss_mean_kernel(const float* loss, int rows, const int* counts, int blocks,
                                                         int mean, float* out, float* out_by) {
  __shared__ double s_v[16];
  __shared__ long long s_n[16];
  double v = 0.;
  long long n = 0;
  if (loss != nullptr) {
#pragma unroll 4
    for (int i = threadIdx.x; i < rows; i += 1024) v += loss[i];
  }
#pragma unroll 4
  for (int i = threadIdx.x; i < blocks; i += 1024) n += counts[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    v += __shfl_xor(v, off);
    n += __shfl_xor(n, off);
  }
  if ((threadIdx.x & 63) == 0) {
    s_v[threadIdx.x >> 6] = v;
    s_n[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) {
    v += s_v[i];
    n += s_n[i];
  }
  const double by = mean && n > 1 ? 1. / n : 1.;
  if (loss != nullptr) *out = static_cast<float>(v * by);
  *out_by = static_cast<float>(by);
}

// ------------------------------------------------------------------------- the loss from logits
// 16 bytes of a row, at any alignment its type allows.
template <typename io_t>
struct DsVec;
template <>
struct DsVec<bf16_t> {
  static constexpr int kN = 8;
  static __device__ __forceinline__ void get(const u32x4& u, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ u32x4 put(const float (&v)[8]) {
    return u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
  }
  static constexpr uint32_t kNone = 0xff80ff80u;  // -inf
};
template <>
struct DsVec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void get(const u32x4& u, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
  }
  static __device__ __forceinline__ u32x4 put(const float (&v)[4]) {
    return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  }
  static constexpr uint32_t kNone = 0xff800000u;
};

// Vector i of a row, -inf past its end.
template <typename io_t>
__device__ __forceinline__ u32x4 ds_load(const io_t* row, int i, int vocab) {
  using V = DsVec<io_t>;
  const int at = i * V::kN;
  u32x4 u = {V::kNone, V::kNone, V::kNone, V::kNone};
  if (at + V::kN <= vocab) {
    u = *reinterpret_cast<const u32x4_any*>(row + at);
  } else {
    alignas(16) io_t tail[V::kN];
    __builtin_memcpy(tail, &u, 16);
#pragma unroll
    for (int e = 0; e < V::kN; ++e)
      if (at + e < vocab) tail[e] = row[at + e];
    __builtin_memcpy(&u, tail, 16);
  }
  return u;
}

template <typename io_t>
__device__ __forceinline__ void ds_store(io_t* row, int i, int vocab, const u32x4& u) {
  using V = DsVec<io_t>;
  const int at = i * V::kN;
  if (at + V::kN <= vocab) {
    *reinterpret_cast<u32x4_any*>(row + at) = u;
  } else {
    alignas(16) io_t tail[V::kN];
    __builtin_memcpy(tail, &u, 16);
#pragma unroll
    for (int e = 0; e < V::kN; ++e)
      if (at + e < vocab) row[at + e] = tail[e];
  }
}

constexpr int kDsHeld = 4096;  // words that a wave holds

// kWaves waves a row; kHeld: the row fits their registers. kDo: the loss (kDsFwd), its gradient (kDsBwd, from the
// statistics of an earlier call unless kDsFwd is there too); kDsAgain: nothing, unless the upstream
// gradient is not the 1 that an earlier call assumed.
template <typename io_t, int kWaves, bool kHeld, int kDo>
__global__ __launch_bounds__(kWaves < 4 ? 256 : 64 * kWaves) void distill_kernel(DistillParams p) {
  using V = DsVec<io_t>;
  constexpr int kVecs = kDsHeld / 64 / V::kN, kThreads = 64 * kWaves, kTeams = kWaves < 4 ? 4 / kWaves : 1;
  __shared__ float s_a[16], s_b[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int tid = kWaves < 4 ? lane : threadIdx.x;
  const long long t = static_cast<long long>(blockIdx.x) * kTeams + (kWaves < 4 ? w : 0);
  float factor = 1.f;
  if constexpr ((kDo & kDsAgain) != 0) {
    factor = p.grad[0];
    if (factor == 1.f) return;
  }
  if (t >= p.r.rows) return;  // (a whole team)
  const io_t* row = static_cast<const io_t*>(p.logits) + t * p.ld;
  io_t* out = static_cast<io_t*>(p.dlogits) + t * p.vocab;
  const int vecs = (p.vocab + V::kN - 1) / V::kN;
  const float live = p.r.live[t];

  if (live == 0.f) {
    if constexpr ((kDo & kDsFwd) != 0) {
      if (tid == 0) {
        p.loss[t] = 0.f;
        p.stat[t] = make_float2(0.f, 0.f);
      }
    }
    if constexpr ((kDo & kDsBwd) != 0)
      for (int i = tid; i < vecs; i += kThreads) ds_store<io_t>(out, i, p.vocab, u32x4{0, 0, 0, 0});
    return;
  }

  const int* words = p.r.words + t * p.r.top;
  const float* qs = p.r.q + t * p.r.top;
  u32x4 held[kHeld ? kVecs : 1];
  if constexpr (kHeld) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int at = tid + i * kThreads;
      held[i] = u32x4{V::kNone, V::kNone, V::kNone, V::kNone};
      if (at < vecs) held[i] = ds_load<io_t>(row, at, p.vocab);
    }
  }
  const auto each = [&](auto&& f) {
    if constexpr (kHeld) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
        if (tid + i * kThreads < vecs) f(tid + i * kThreads, held[i]);
    } else {
#pragma unroll 4
      for (int i = tid; i < vecs; i += kThreads) f(i, ds_load<io_t>(row, i, p.vocab));
    }
  };

  float m, l;
  if constexpr ((kDo & kDsFwd) != 0) {
    m = -INFINITY;
    float s = 0.f;
    if constexpr (kHeld) {
      each([&](int, const u32x4& u) {
        float v[V::kN];
        V::get(u, v);
#pragma unroll
        for (int e = 0; e < V::kN; ++e) m = fmaxf(m, v[e]);
      });
    } else {  // with the sum, of what comes before
      each([&](int, const u32x4& u) {
        float v[V::kN];
        V::get(u, v);
        float mx = m;
#pragma unroll
        for (int e = 0; e < V::kN; ++e) mx = fmaxf(mx, v[e]);
        if (mx > m) {
          s *= fast_exp2((m - mx) * p.r.c);
          m = mx;
        }
        const float from = m == -INFINITY ? 0.f : m;  // (then there are words of no weight, and NaNs, which count)
#pragma unroll
        for (int e = 0; e < V::kN; ++e) s += fast_exp2((v[e] - from) * p.r.c);
      });
    }
    const float mine = m;
    m = wave_max_f(m);
    if constexpr (kWaves >= 4) {
      if (lane == 0) s_a[w] = m;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kWaves; ++i) m = fmaxf(m, s_a[i]);
      __syncthreads();
    }
    if constexpr (kHeld) {
      each([&](int, const u32x4& u) {
        float v[V::kN];
        V::get(u, v);
#pragma unroll
        for (int e = 0; e < V::kN; ++e) s += fast_exp2((v[e] - m) * p.r.c);
      });
    } else {
      s = mine == -INFINITY ? s : s * fast_exp2((mine - m) * p.r.c);
    }
    float want = 0.f;  // sum q (log q - (x - m) c)
    for (int k = tid; k < p.r.top; k += kThreads) {
      if (words[k] < 0) continue;
      const float q = qs[k];
      want = __builtin_fmaf(q, fast_log2(q) - (to_f32(row[words[k]]) - m) * p.r.c, want);
    }
    s = wave_sum_f(s);
    want = wave_sum_f(want);
    if constexpr (kWaves >= 4) {
      if (lane == 0) {
        s_a[w] = s;
        s_b[w] = want;
      }
      __syncthreads();
      s = want = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        s += s_a[i];
        want += s_b[i];
      }
    }
    if (m == -INFINITY) s = __builtin_nanf("");  // no word at all
    l = fast_log2(s) + (live - live);
    if (tid == 0) {
      p.loss[t] = (want + l) * (kLn2 * p.temperature * p.temperature);
      p.stat[t] = make_float2(m, l);
    }
  } else {
    const float2 st = p.stat[t];
    m = st.x;
    l = st.y;
  }

  if constexpr ((kDo & kDsBwd) != 0) {
    float f = p.temperature;
    if constexpr ((kDo & kDsAgain) != 0) f *= factor;
    else if constexpr ((kDo & kDsFwd) == 0) f *= p.grad[p.reduction == kLossNone ? t : 0];
    if (p.reduction == kLossMean) f *= *p.by;
    each([&](int i, const u32x4& u) {
      float v[V::kN];
      V::get(u, v);
#pragma unroll
      for (int e = 0; e < V::kN; ++e) v[e] = fast_exp2(__builtin_fmaf(v[e] - m, p.r.c, -l)) * f;
      ds_store<io_t>(out, i, p.vocab, V::put(v));
    });
    // The wanted words' own, once the row's stores are done.
    __threadfence_block();
    if constexpr (kWaves >= 4) __syncthreads();
    for (int k = tid; k < p.r.top; k += kThreads) {
      const int v = words[k];
      if (v < 0) continue;
      store_as(out + v, (fast_exp2(__builtin_fmaf(to_f32(row[v]) - m, p.r.c, -l)) - qs[k]) * f);
    }
  }
}

template <typename io_t, int kDo>
void launch_do(const DistillParams& p, hipStream_t stream) {
  const int rows = p.r.rows;
  if (p.vocab <= kDsHeld)
    hipLaunchKernelGGL((distill_kernel<io_t, 1, true, kDo>), dim3((rows + 3) / 4), dim3(256), 0, stream, p);
  else if (p.vocab <= 4 * kDsHeld)
    hipLaunchKernelGGL((distill_kernel<io_t, 4, true, kDo>), dim3(rows), dim3(256), 0, stream, p);
  else if (p.vocab <= 16 * kDsHeld)
    hipLaunchKernelGGL((distill_kernel<io_t, 16, true, kDo>), dim3(rows), dim3(1024), 0, stream, p);
  else
    hipLaunchKernelGGL((distill_kernel<io_t, 16, false, kDo>), dim3(rows), dim3(1024), 0, stream, p);
}

template <int kDo>
void launch_typed(const DistillParams& p, hipStream_t stream) {
  if (p.io_bf16) launch_do<bf16_t, kDo>(p, stream);
  else launch_do<float, kDo>(p, stream);
}

}  // namespace

int loss_list_blocks(int rows) { return (rows + kListRows - 1) / kListRows; }

hipError_t launch_loss_rows(const LossRows& r, hipStream_t stream) {
  const dim3 grid(r.blocks);
  if (r.top <= 64) hipLaunchKernelGGL(loss_lists_kernel<1>, grid, dim3(64 * kListRows), 0, stream, r);
  else if (r.top <= 128) hipLaunchKernelGGL(loss_lists_kernel<2>, grid, dim3(64 * kListRows), 0, stream, r);
  else if (r.top <= 256) hipLaunchKernelGGL(loss_lists_kernel<4>, grid, dim3(64 * kListRows), 0, stream, r);
  else hipLaunchKernelGGL(loss_lists_kernel<16>, grid, dim3(64 * kListRows), 0, stream, r);
  return hipGetLastError();
}

hipError_t launch_loss_mean(const float* loss, const LossRows& r, int reduction, float* mean, float* by, hipStream_t stream) {
  hipLaunchKernelGGL(loss_mean_kernel, dim3(1), dim3(1024), 0, stream, loss, r.rows, r.counts, r.blocks,
                     reduction == kLossMean ? 1 : 0, mean, by);
  return hipGetLastError();
}

hipError_t launch_distill(const DistillParams& p, int what, hipStream_t stream) {
  if (what & kDsFwd) {
    hipError_t e = launch_loss_rows(p.r, stream);
    if (e != hipSuccess) return e;
    if (what == (kDsFwd | kDsBwd) && p.reduction == kLossMean) {
      e = launch_loss_mean(nullptr, p.r, p.reduction, nullptr, p.by, stream);
      if (e != hipSuccess) return e;
    }
  }
  if (what == kDsFwd) launch_typed<kDsFwd>(p, stream);
  else if (what == kDsBwd) launch_typed<kDsBwd>(p, stream);
  else if (what == (kDsFwd | kDsBwd)) launch_typed<kDsFwd | kDsBwd>(p, stream);
  else launch_typed<kDsBwd | kDsAgain>(p, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if ((what & kDsFwd) && p.reduction != kLossNone) return launch_loss_mean(p.loss, p.r, p.reduction, p.mean, p.by, stream);
  return hipSuccess;
}

}  // namespace mss
