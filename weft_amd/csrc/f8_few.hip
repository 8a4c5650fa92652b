// The product of 8-bit floats for few tokens (and for any sizes, strides and alignment):
//   y[t][n] = sum over blocks b of  sx[t][b] sw[n / 128][b]  sum over k in b of x[t][k] w[n][k]
//
// e4m3 numbers are 16-bit floats, so a block's 128 values are four
// v_mfma_f32_16x16x32_f16 of a tile of 16 weights (rows of the result) and 16 tokens
// (columns), whose products are exact and whose sums have 32 bits.  The block's sums are
// added to the tile's times the two scales, one multiply-add a value: a lane has one token,
// so one scale.
//
// Lane l of a tile holds K values 32 (l / 16) .. + 31 of row l % 16, for weights and tokens
// alike; which of them an instruction takes does not matter as both have the same.
// The blocks of a row are dealt to the workgroup's waves in turn (its 16 rows are then read
// as whole contiguous pieces) and their sums meet in LDS in the order of the waves.
#include <algorithm>

#include "f8.h"
#include "runtime.h"

namespace weft {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));

struct __attribute__((packed, aligned(1))) Bytes16 {
  int w[4];
};

// 32 codes of a row from p on, of which `left` are in the row; zeros behind.  kWide: rows in
// aligned groups of 16, so that a group is wholly in the row or behind it.
template <bool kWide>
__device__ __forceinline__ v8i load32(const uint8_t* p, int left) {
  v8i v = {0, 0, 0, 0, 0, 0, 0, 0};
  if constexpr (kWide) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (left > 16 * h) {
        const int4 q = *reinterpret_cast<const int4*>(p + 16 * h);
        v[4 * h] = q.x, v[4 * h + 1] = q.y, v[4 * h + 2] = q.z, v[4 * h + 3] = q.w;
      }
  } else if (left >= 32) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Bytes16 q = *reinterpret_cast<const Bytes16*>(p + 16 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * h + e] = q.w[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (e < left) v[e / 4] |= (int)((uint32_t)p[e] << (8 * (e & 3)));
  }
  return v;
}

// the e4m3 numbers of eight codes
__device__ __forceinline__ half8 halves(int lo, int hi) {
  const half2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  const half2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const half2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  const half2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ v4f product16(v8i a, v8i b) {
  v4f c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; i += 2)
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(a[i], a[i + 1]), halves(b[i], b[i + 1]), c, 0, 0, 0);
  return c;
}

template <int MT, bool kWide>
__global__ void __launch_bounds__(1024) f8_few_kernel(F8Product p) {
  extern __shared__ float sums[];  // [wave][token][16 weights]
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16 * MT;
  const int blocks = (p.k + kF8Block - 1) / kF8Block;
  // rows past the ends are read as the last one and not stored
  const uint8_t* w = p.w.codes + min(n0 + r, p.n - 1) * p.w.row + 32 * g;
  const float* sw = p.w.scales + (n0 / kF8Block) * p.w.s_row;
  const uint8_t* x[MT];
  const float* sx[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int token = min(m0 + 16 * t + r, p.m - 1);
    x[t] = p.x.codes + token * p.x.row + 32 * g;
    sx[t] = p.x.scales + token * p.x.s_row;
  }
  v4f acc[MT] = {};
  constexpr int U = 2;
  for (int b0 = wave; b0 < blocks; b0 += U * waves) {
    v8i wv[U], xv[U][MT];
    float swv[U], sxv[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = b0 + u * waves;
      if (b >= blocks) break;
      const int left = p.k - b * kF8Block - 32 * g;
      wv[u] = load32<kWide>(w + (long long)b * kF8Block, left);
      swv[u] = sw[b * p.w.s_block];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        xv[u][t] = load32<kWide>(x[t] + (long long)b * kF8Block, left);
        sxv[u][t] = sx[t][b * p.x.s_block];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b0 + u * waves >= blocks) break;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const v4f c = product16(wv[u], xv[u][t]);
        const float s = swv[u] * sxv[u][t];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(c[i], s, acc[t][i]);
      }
    }
  }
  // lane l has weights 4 (l / 16) .. + 3 of token l % 16
#pragma unroll
  for (int t = 0; t < MT; ++t) *reinterpret_cast<v4f*>(sums + ((wave * MT + t) * 16 + r) * 16 + 4 * g) = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 256; i += blockDim.x) {
    float v = 0.f;
    for (int s = 0; s < waves; ++s) v += sums[s * MT * 256 + i];
    const int token = m0 + i / 16, n = n0 + (i & 15);
    if (token >= p.m || n >= p.n) continue;
    uint8_t* at = p.y + token * p.y_row;
    if (p.half_out)
      reinterpret_cast<_Float16*>(at)[n] = (_Float16)v;
    else
      reinterpret_cast<float*>(at)[n] = v;
  }
}

template <int MT>
void launch(const F8Product& p, bool wide, dim3 grid, int waves) {
  const size_t lds = (size_t)waves * MT * 256 * sizeof(float);
  if (wide)
    f8_few_kernel<MT, true><<<grid, waves * kWave, lds, current_stream()>>>(p);
  else
    f8_few_kernel<MT, false><<<grid, waves * kWave, lds, current_stream()>>>(p);
  check_launch("f8_few_kernel");
}

}  // namespace

void f8_few(const F8Product& all) {
  const int blocks = (int)f8_blocks(all.k);
  int waves = 1;
  while (waves < 8 && waves < blocks) waves *= 2;
  const bool wide = all.k % 16 == 0 && all.w.row % 16 == 0 && all.x.row % 16 == 0 && aligned(all.w.codes, 16) &&
                    aligned(all.x.codes, 16);
  // a launch has fewer than 2^32 threads, and 65535 groups in y
  constexpr int kMostN = 1 << 20, kMostM = 1 << 15;
  for (int64_t m = 0; m < all.m; m += kMostM)
    for (int64_t n = 0; n < all.n; n += kMostN) {
      F8Product p = all;
      p.m = (int)std::min<int64_t>(all.m - m, kMostM);
      p.n = (int)std::min<int64_t>(all.n - n, kMostN);
      p.x.codes += m * p.x.row;
      p.x.scales += m * p.x.s_row;
      p.w.codes += n * p.w.row;
      p.w.scales += n / kF8Block * p.w.s_row;
      p.y += m * p.y_row + n * (p.half_out ? 2 : 4);
      const int tiles = (p.m + 15) / 16;
      const unsigned gx = (unsigned)((p.n + 15) / 16);
      if (tiles == 1)
        launch<1>(p, wide, dim3(gx, 1), waves);
      else
        launch<2>(p, wide, dim3(gx, (unsigned)((tiles + 1) / 2)), waves);
    }
}

}  // namespace weft
