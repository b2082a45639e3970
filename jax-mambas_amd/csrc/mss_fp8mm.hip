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
// a bf16 output's own rounding, but far more than a float32 output's. So a float32 output takes
// its operands to bf16 (exact, v_cvt_scalef32_pk_bf16_fp8) and multiplies with the bf16
// instructions, at half the rate; a bf16 output does so where that rate is not what bounds it.
#include <hip/hip_runtime.h>

#include "mss_serve.h"

namespace mss {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// The sum over one block: rows of `a` (16) by rows of `b` (16). Lane l holds a's row l % 16 (the
// result's rows) and b's row l % 16 (its columns), features 16 (l / 16) .. + 16 of the block's
// first half and the same of the second; the result's lane l has column l % 16, rows
// 4 (l / 16) .. + 4. The order of the features inside a block is the same in both operands, and
// that is all their sum needs.
// 8 e4m3 values as bf16.
__device__ __forceinline__ bf16x8 to_bf16x8(int lo, int hi) {
  const bf16x2_t v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
  const bf16x2_t v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
  const bf16x2_t v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
  const bf16x2_t v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
  return bf16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}

__device__ __forceinline__ f32x4 mfma_block_bf16(const i32x8& a, const i32x8& b) {
  f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16x8(a[i], a[i + 1]), to_bf16x8(b[i], b[i + 1]), d, 0, 0, 0);
  return d;
}

__device__ __forceinline__ i32x8 join(const u32x4& lo, const u32x4& hi) {
  return i32x8{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(lo[2]), static_cast<int>(lo[3]),
               static_cast<int>(hi[0]), static_cast<int>(hi[1]), static_cast<int>(hi[2]), static_cast<int>(hi[3])};
}

template <typename out_t>
__device__ __forceinline__ void store_out(const Fp8MmParams& p, int m, int t, float v) {
  out_t* c = static_cast<out_t*>(p.c);
  store_as(c + (p.token_major ? t * p.ldc + m : m * p.ldc + t), v);
}

// A lane's 32 bytes of a row's block: 16 at k and 16 at k + 64. Rows start on 16 bytes; a
// 16-byte piece is read where it begins before the row's end, but for the part of the last one
// that is past the tensor's end, which is read byte by byte.
__device__ __forceinline__ i32x8 load_row(const unsigned char* __restrict__ base, long long ld, int row, int rows,
                                          int k, int K) {
  u32x4 v[2] = {};
  if (row < rows) {
    const unsigned char* r = base + row * ld;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int kk = k + 64 * h;
      if (kk + 16 <= K) {
        v[h] = *reinterpret_cast<const u32x4*>(r + kk);
      } else if (kk < K) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (kk + i < K) v[h][i / 4] |= static_cast<uint32_t>(r[kk + i]) << (8 * (i % 4));
      }
    }
  }
  return join(v[0], v[1]);
}

// One wave, one 16 x 16 tile of C.
template <typename out_t>
__global__ __launch_bounds__(64) void fp8mm_kernel(Fp8MmParams p) {
  const int lane = threadIdx.x, col = lane & 15, grp = lane >> 4;
  const int m0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
  const int nkb = (p.K + kFp8Block - 1) / kFp8Block;
  const float* __restrict__ ws = p.ws + static_cast<long long>(m0 / kFp8Block) * nkb;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int b = 0; b < nkb; ++b) {
    const int k = b * kFp8Block + grp * 16;
    const i32x8 w = load_row(p.w, p.ldw, m0 + col, p.M, k, p.K);
    const i32x8 x = load_row(p.x, p.ldx, t0 + col, p.T, k, p.K);
    const float s = t0 + col < p.T ? p.xs[static_cast<long long>(b) * p.T + t0 + col] * ws[b] : 0.f;
    const f32x4 d = mfma_block_bf16(w, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(d[i], s, acc[i]);
  }
  if (t0 + col >= p.T) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + grp * 4 + i;
    if (m < p.M) store_out<out_t>(p, m, t0 + col, acc[i]);
  }
}

hipError_t launch_fp8mm(const Fp8MmParams& p, hipStream_t stream) {
  const dim3 grid((p.M + 15) / 16, (p.T + 15) / 16);
  if (p.out_bf16) hipLaunchKernelGGL(fp8mm_kernel<bf16_t>, grid, dim3(64), 0, stream, p);
  else hipLaunchKernelGGL(fp8mm_kernel<float>, grid, dim3(64), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mss
