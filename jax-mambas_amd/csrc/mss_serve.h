// Parameter blocks and small device helpers of the 8-bit serving operators (mss_quant.hip,
// mss_fp8mm.hip) and of the token draw (mss_sample.hip). The host fills the blocks after
// validation.
//
// 8-bit form of a matrix: e4m3 values (1 sign, 4 exponent, 3 fraction bits; no infinity, largest
// finite 448) in rows along the features, which start on 16 bytes, with one float32 scale for
// each block of kFp8Block features and each token (activations), or for each kFp8Block x
// kFp8Block block (weights). A block's scale is max(largest magnitude / 448, 2^-126) and a value
// stands for q * scale. A NaN or an infinity in a block makes that block's scale NaN or
// infinite, so what it stands for is NaN.
#pragma once

#include "mss_common.h"

namespace mss {

constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.f;

struct QuantParams {
  int features, tokens;
  long long sf, st;        // element strides of x along features and tokens
  long long ldq;           // bytes from one token's row of q to the next
  const void* x;
  unsigned char* q;        // [tokens][ldq]
  float* scales;           // [feature blocks][tokens]
  // residual add + norm in front (launch_norm_fp8): x is h [features][tokens]
  float eps;
  const void* delta;       // optional [features][tokens]
  const float* w;          // [features]
  float* hn;               // [features][tokens], written when delta is given
};

struct QuantWeightParams {
  int M, K;
  long long ldw, ldq;      // row strides of w (elements) and q (bytes)
  const void* w;
  unsigned char* q;
  float* scales;           // [row blocks][feature blocks]
};

struct Fp8MmParams {
  int M, K, T;
  int token_major;         // C is [T][ldc] instead of [M][ldc]
  int out_bf16;
  long long ldw, ldx, ldc; // bytes for w and x, elements for c
  const unsigned char* w;  // [M][ldw]
  const float* ws;         // [row blocks][feature blocks]
  const unsigned char* x;  // [T][ldx]
  const float* xs;         // [feature blocks][T]
  void* c;
};

struct SampleParams {
  int rows, vocab;
  long long sr, sv;        // element strides of logits along rows and words
  const void* logits;
  const float* uniform;    // [rows]
  // one value for every row, or [rows] where the pointer is set
  float temperature, top_p, min_p;
  int top_k;
  const float* temperatures;
  const int* top_ks;
  const float* top_ps;
  const float* min_ps;
  long long* tokens;       // [rows]
};

// The scale of a block whose largest magnitude is `amax` (NaN stays NaN).
__device__ __forceinline__ float fp8_scale(float amax) {
  const float s = amax / kFp8Max;
  return s < 1.1754943508222875e-38f ? 1.1754943508222875e-38f : s;
}

// Four float32 values as e4m3, rounded to nearest even, the first in bits 0..7. The inputs
// are at most 448 in magnitude up to a rounding of the scale's reciprocal, or NaN.
__device__ __forceinline__ uint32_t pack_fp8x4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
  return static_cast<uint32_t>(v);
}

// |v| as bits: ordered as the magnitudes are, a NaN above infinity.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

}  // namespace mss
