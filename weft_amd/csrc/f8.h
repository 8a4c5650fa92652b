// 8-bit floats (e4m3: sign, 4 exponent bits of bias 7, 3 of fraction, no infinity, NaN
// 0x7f) with a 32-bit scale for each 128 values: what the quantizer and the products share.
//
//   a = max(2^-100, the largest finite |x| of the block),  scale = a / 448,
//   code = the e4m3 number nearest x (448 / a), ties to even; NaN for an x that is not finite
//
// 448 is the largest e4m3 number, so the block's largest value takes the whole range;
// 2^-100 keeps 448 / a and a / 448 finite and normal, and a block of zeros is codes of 0.
#pragma once

#include "weft_common.h"
#include "weft_hip.h"

namespace weft {

constexpr int kF8Block = 128;
constexpr float kF8Top = 448.f;

// Rows of codes and their scales: bytes between rows, floats between rows (weights: blocks
// of rows) and between blocks of scales.
struct F8Rows {
  const uint8_t* codes;
  const float* scales;
  long long row, s_row, s_block;
};

__device__ __forceinline__ float f8_finite_abs(float x) {
  const float v = fabsf(x);
  return v <= 3.402823466e38f ? v : 0.f;  // NaN compares false
}
struct F8Scale {
  float factor, scale;
};
__device__ __forceinline__ F8Scale f8_scale(float most) {
  const float a = fmaxf(most, 0x1p-100f);
  return {__fdiv_rn(kF8Top, a), __fdiv_rn(a, kF8Top)};
}
// |x factor| <= 448 (1 + 2^-23), which rounds to 448 at most
__device__ __forceinline__ float f8_scaled(float x, float factor) {
  return fabsf(x) <= 3.402823466e38f ? x * factor : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return (uint32_t)w;
}
// Eight values a lane, a block in the 16 lanes of a row: this lane's codes, the block's scale.
__device__ __forceinline__ uint2 f8_quantize_16lanes(const float (&x)[8], float& scale) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, f8_finite_abs(x[i]));
  m = fmaxf(m, dpp_row<kDppXor1>(m));
  m = fmaxf(m, dpp_row<kDppXor2>(m));
  m = fmaxf(m, dpp_row<kDppHalfMirror>(m));
  m = fmaxf(m, dpp_row<kDppMirror>(m));
  const F8Scale s = f8_scale(m);
  scale = s.scale;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = f8_scaled(x[i], s.factor);
  return make_uint2(f8_pack4(y[0], y[1], y[2], y[3]), f8_pack4(y[4], y[5], y[6], y[7]));
}

// Eight values of a row from i on, zeros from k on; the row's elements are aligned, no more.
struct __attribute__((packed, aligned(4))) F8Floats8 {
  float f[8];
};
struct __attribute__((packed, aligned(2))) F8Halves8 {
  _Float16 h[8];
};
template <bool kHalf>
__device__ __forceinline__ void f8_load8(const uint8_t* row, long long i, long long k, float (&x)[8]) {
  if constexpr (kHalf) {
    const _Float16* p = reinterpret_cast<const _Float16*>(row);
    if (i + 8 <= k) {
      const F8Halves8 v = *reinterpret_cast<const F8Halves8*>(p + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)v.h[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = i + e < k ? (float)p[i + e] : 0.f;
    }
  } else {
    const float* p = reinterpret_cast<const float*>(row);
    if (i + 8 <= k) {
      const F8Floats8 v = *reinterpret_cast<const F8Floats8*>(p + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = v.f[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = i + e < k ? p[i + e] : 0.f;
    }
  }
}

// ---------------------------------------------------------------- host side
inline int64_t f8_blocks(int64_t n) { return (n + kF8Block - 1) / kF8Block; }

// Rows of F32 or F16 (row bytes apart) as codes (y_row bytes apart, the first `wide` bytes of
// each written, zeros past k) and scales at s_row, s_block floats.
void f8_quantize_rows(const uint8_t* x, bool half, long long x_row, uint8_t* y, long long y_row, int wide,
                      float* scales, long long s_row, long long s_block, int64_t rows, int k);

// y (m tokens, n weights) of weights and activations in 8 bits.
struct F8Product {
  F8Rows w, x;
  uint8_t* y;
  long long y_row;  // bytes
  int n, m, k;
  bool half_out;
};

// Up to 16 tokens: a tile of 16 weights a workgroup, K split over its waves.  plain: rows to be
// quantized on the way (p.x is not read), where f8_few_quantizes.
constexpr int64_t kF8Few = 16;
bool f8_few_quantizes(int64_t m, int64_t k);
void f8_few(const F8Product& p, const uint8_t* plain = nullptr, bool plain_half = false, long long plain_row = 0);
// More: tiles of 32 to 256 tokens through LDS; work: f8_many_work bytes, of the shapes alone.
size_t f8_many_work(int64_t m, int64_t n, int64_t k);
void f8_many(const F8Product& p, float* work);
// Its tiles of 256 x 256, for 16-bit outputs and rows in aligned chunks of 16.
void f8_large(const F8Product& p);

}  // namespace weft
