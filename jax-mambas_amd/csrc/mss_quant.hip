// Activations and weights in 8 bits (e4m3) with block scales, and the residual add + RMSNorm
// that writes its output that way.
//
//   y[f][t]  = x[f][t], or with the norm in front: hn = h + delta, r_t = 1 / sqrt(mean_f hn^2 +
//              eps), y = hn r_t w[f]   (reference mamba/mamba1.py:300-337: nnx.RMSNorm before
//              the in-projections, the block's output added back)
//   s[b][t]  = max(max_{f in block b} |y[f][t]| / 448, 2^-126)
//   q[t][f]  = e4m3(y[f][t] * (1 / s[b][t])), rounded to nearest even
//
// The stream is channel-major (features, tokens) and a matrix-core product wants 8-bit operands
// with the features contiguous, so these kernels also transpose: a workgroup owns a tile of
// tokens, one token a lane, and each thread 4 consecutive features of a block, which it packs
// into one dword of the token's row in LDS; the rows leave as whole dwords. y and the norm's
// sums are float32; q is the only rounding to fewer bits.
#include <hip/hip_runtime.h>

#include "mss_serve.h"

namespace mss {

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
  const float scale = fp8_scale(__uint_as_float(m));
  const float inv = 1.f / scale;
  if (!ok) return;
  if (lane == 0) p.scales[static_cast<long long>(b) * p.tokens + t] = scale;
  // A row of q is 16-byte aligned and holds at least ceil16(features) bytes up to the next row;
  // the last row's end is the tensor's, so the bytes past the features are not touched.
  unsigned char* q = p.q + t * p.ldq + f0;
  const uint32_t lo = pack_fp8x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  const uint32_t hi = pack_fp8x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
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
  const float scale = fp8_scale(__uint_as_float(m));
  const float inv = 1.f / scale;
  if (threadIdx.x == 0) p.scales[static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x] = scale;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int r = row0 + 4 * i;
    if (r >= p.M || k >= p.K) continue;
    const uint32_t two = pack_fp8x4(v[i][0] * inv, v[i][1] * inv, 0.f, 0.f);
    unsigned char* q = p.q + r * p.ldq + k;  // k even, rows 16-byte aligned
    if (k + 1 < p.K) *reinterpret_cast<uint16_t*>(q) = static_cast<uint16_t>(two);
    else *q = static_cast<unsigned char>(two);
  }
}

// ------------------------------------------------------------------ residual add + norm
// One token a workgroup: two passes over its column.
template <typename delta_t, bool kDelta>
__global__ __launch_bounds__(512) void norm_fp8_rows_kernel(QuantParams p) {
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
  // 32 lanes hold a block, 4 consecutive features each.
  for (int f0 = threadIdx.x * 4; f0 < padded; f0 += 2048) {
    float v[4];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int f = f0 + i;
      v[i] = 0.f;
      if (f < p.features) {
        float x = h[f * T];
        if constexpr (kDelta) {
          x += to_f32(delta[f * T]);
          p.hn[f * T + t] = x;
        }
        v[i] = x * r * p.w[f];
      }
      m = max(m, magnitude_bits(v[i]));
    }
#pragma unroll
    for (int s = 1; s < 32; s *= 2) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), s)));
    const float scale = fp8_scale(__uint_as_float(m));
    const float inv = 1.f / scale;
    if ((threadIdx.x & 31) == 0) p.scales[(f0 / kFp8Block) * T + t] = scale;
    const uint32_t q4 = pack_fp8x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
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
template <typename io_t>
static void launch_quant_rows(const QuantParams& p, hipStream_t stream) {
  const dim3 grid((p.tokens + 15) / 16, (p.features + kFp8Block - 1) / kFp8Block);
  // 16-byte loads where a token's features are contiguous and its row starts on 16 bytes.
  const bool vec = p.sf == 1 && (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 &&
                   (p.st * static_cast<long long>(sizeof(io_t))) % 16 == 0;
  if (vec) hipLaunchKernelGGL((quant_rows_kernel<io_t, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((quant_rows_kernel<io_t, false>), grid, dim3(256), 0, stream, p);
}

hipError_t launch_quant_fp8(const QuantParams& p, bool io_bf16, hipStream_t stream) {
  if (io_bf16) launch_quant_rows<bf16_t>(p, stream);
  else launch_quant_rows<float>(p, stream);
  return hipGetLastError();
}

hipError_t launch_quant_fp8_weight(const QuantWeightParams& p, bool io_bf16, hipStream_t stream) {
  const dim3 grid((p.K + kFp8Block - 1) / kFp8Block, (p.M + kFp8Block - 1) / kFp8Block);
  if (io_bf16) hipLaunchKernelGGL(quant_weight_kernel<bf16_t>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(quant_weight_kernel<float>, grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_norm_fp8(const QuantParams& p, bool delta_bf16, hipStream_t stream) {
  const dim3 grid(p.tokens), block(512);
  if (!p.delta) hipLaunchKernelGGL((norm_fp8_rows_kernel<float, false>), grid, block, 0, stream, p);
  else if (delta_bf16) hipLaunchKernelGGL((norm_fp8_rows_kernel<bf16_t, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((norm_fp8_rows_kernel<float, true>), grid, block, 0, stream, p);
  return hipGetLastError();
}

}  // namespace mss
