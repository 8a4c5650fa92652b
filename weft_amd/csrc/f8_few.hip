// The product of 8-bit floats for up to 16 tokens, for any strides and alignment:
//   y[t][n] = sum over blocks b of  sx[t][b] sw[n / 128][b]  sum over k in b of x[t][k] w[n][k]
//
// e4m3 numbers are 16-bit floats, so a block's 128 values are four
// v_mfma_f32_16x16x32_f16 of a tile of 16 weights (rows of the result) and 16 tokens
// (columns), whose products are exact and whose sums have 32 bits.  The block's sums are
// added to the tile's times the two scales, one multiply-add a value: a lane has one token,
// so one factor.
//
// Lane l of a tile holds two chunks of 16 of row l % 16's values, for weights and tokens alike;
// which of them an instruction takes does not matter as both have the same.
// The blocks of a row are dealt to the workgroup's waves in turn (its 16 rows are then read
// as whole contiguous pieces) and their sums meet in LDS in the order of the waves.
//
// Bound by the reading of the weights and by latency: a launch, the tokens' codes (quantized
// by each workgroup while its first weights are on their way: a launch of its own for 4096
// values costs 3 us more), then a trip to memory for each of a wave's blocks.  One token and
// 4096 x 4096 weights take 6.8 us (2.5 TB/s), 11008 x 4096 12.4 (3.6 TB/s), 4096 x 11008 11.3 (4.0).
// Tried: two blocks a wave on their way at once (7.1, 13.8, 12.5), the next block's loads before a
// block's products (6.9, 15.5, 11.2), 32 weights a wave (6.8, 14.5 and 11.3).
#include <algorithm>

#include "f8_tile.h"
#include "runtime.h"

namespace weft {
namespace {

// A lane's 32 codes of block b of a row of k: chunks g and g + 4 of 16, so that a load's four lanes
// of a row read 64 contiguous bytes; zeros behind the row's end.  kWide: rows in aligned groups of 16,
// so that a chunk is wholly in the row or behind it.
template <bool kWide>
__device__ __forceinline__ v8i load32(const uint8_t* row, int b, int g, int k) {
  const int at = b * kF8Block + 16 * g;
  uint4 q[2];
  if constexpr (kWide) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      q[h] = at + 64 * h < k ? *reinterpret_cast<const uint4*>(row + at + 64 * h) : uint4{0, 0, 0, 0};
  } else if ((b + 1) * kF8Block <= k) {
#pragma unroll
    for (int h = 0; h < 2; ++h) q[h] = codes16(row + at + 64 * h);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) q[h] = codes16(row, at + 64 * h, k);
  }
  return v8i{(int)q[0].x, (int)q[0].y, (int)q[0].z, (int)q[0].w, (int)q[1].x, (int)q[1].y, (int)q[1].z, (int)q[1].w};
}

// Plain rows of tokens, for a workgroup that quantizes them itself.
struct PlainRows {
  const uint8_t* x;
  long long row;  // bytes
};
enum Source { kCodes = 0, kF32 = 1, kF16 = 2 };
constexpr int kFusedValues = 16384;  // of all tokens, at most

// From plain rows each workgroup quantizes all tokens into LDS, its first weights on their way
// meanwhile.
template <bool kWide, int kSource>
__global__ void __launch_bounds__(1024) f8_few_kernel(F8Product p, PlainRows plain) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * 16;
  const int blocks = (p.k + kF8Block - 1) / kF8Block;
  float* sums = lds;  // [wave][token][16 weights]
  uint8_t* codes = reinterpret_cast<uint8_t*>(lds + waves * 256);
  const int pitch = blocks * kF8Block + 16;  // rows of tokens meet in different banks
  float* scales = reinterpret_cast<float*>(codes + p.m * pitch);

  // rows past the ends are read as the last one and not stored
  const int token = min(r, p.m - 1);
  const uint8_t* w = p.w.codes + min(n0 + r, p.n - 1) * p.w.row;
  const float* sw = p.w.scales + (n0 / kF8Block) * p.w.s_row;
  const uint8_t* x = kSource ? codes + token * pitch : p.x.codes + token * p.x.row;
  const float* sx = kSource ? scales + token * blocks : p.x.scales + token * p.x.s_row;
  const long long sx_block = kSource ? 1 : p.x.s_block;

  v8i wv;
  float swv;
  auto load_weights = [&](int b) {
    if (b >= blocks) return;
    wv = load32<kWide>(w, b, g, p.k);
    swv = sw[b * p.w.s_block];
  };
  load_weights(wave);

  if constexpr (kSource != kCodes) {
    const int part = threadIdx.x & 15;
    for (int i = threadIdx.x / 16; i < p.m * blocks; i += blockDim.x / 16) {
      const int t = i / blocks, b = i - t * blocks;
      float v[8];
      f8_load8<kSource == kF16>(plain.x + t * plain.row, b * kF8Block + 8 * part, p.k, v);
      float scale;
      const uint2 c = f8_quantize_16lanes(v, scale);
      *reinterpret_cast<uint2*>(codes + t * pitch + b * kF8Block + 8 * part) = c;
      if (part == 0) scales[i] = scale;
    }
    __syncthreads();
  }

  v4f acc = {0.f, 0.f, 0.f, 0.f};
  for (int b = wave; b < blocks; b += waves) {
    if (b != wave) load_weights(b);
    // codes quantized here are whole blocks
    const v8i xv =
        load32<kWide || kSource != kCodes>(x, b, g, kSource ? blocks * kF8Block : p.k);
    const float s = swv * sx[b * sx_block];
    v4f c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(wv[i], wv[i + 1]), halves(xv[i], xv[i + 1]), c, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(c[e], s, acc[e]);
  }
  // lane l has weights 4 (l / 16) .. + 3 of token l % 16
  *reinterpret_cast<v4f*>(sums + (wave * 16 + r) * 16 + 4 * g) = acc;
  __syncthreads();
  for (int i = threadIdx.x; i < 256; i += blockDim.x) {
    float v = 0.f;
    for (int s = 0; s < waves; ++s) v += sums[s * 256 + i];
    const int t = i / 16, n = n0 + i % 16;
    if (t >= p.m || n >= p.n) continue;
    uint8_t* at = p.y + t * p.y_row;
    if (p.half_out)
      reinterpret_cast<_Float16*>(at)[n] = (_Float16)v;
    else
      reinterpret_cast<float*>(at)[n] = v;
  }
}

template <int kSource>
void launch(const F8Product& p, const PlainRows& plain, bool wide) {
  const int blocks = (int)f8_blocks(p.k), tiles = (p.n + 15) / 16;
  // 16 waves up to two workgroups a CU, 8 past that (us, 16 and 8: 4096 x 11008 11.3 and 12.4,
  // 1000 x 16384 11.5 and 13.2; 11008 x 4096 14.5 and 12.4)
  int waves = tiles <= 512 ? 16 : 8;
  while (waves > 1 && waves / 2 >= blocks) waves /= 2;
  size_t lds = (size_t)waves * 256 * sizeof(float);
  if (kSource) lds += (size_t)p.m * ((size_t)blocks * kF8Block + 16 + blocks * sizeof(float));
  if (wide)
    f8_few_kernel<true, kSource><<<dim3((unsigned)tiles), waves * kWave, lds, current_stream()>>>(p, plain);
  else
    f8_few_kernel<false, kSource><<<dim3((unsigned)tiles), waves * kWave, lds, current_stream()>>>(p, plain);
  check_launch("f8_few_kernel");
}

}  // namespace

bool f8_few_quantizes(int64_t m, int64_t k) { return m <= kF8Few && m * f8_blocks(k) * kF8Block <= kFusedValues; }

void f8_few(const F8Product& all, const uint8_t* plain, bool plain_half, long long plain_row) {
  const bool wide_w = all.k % 16 == 0 && all.w.row % 16 == 0 && aligned(all.w.codes, 16);
  const bool wide = wide_w && (plain != nullptr || (all.x.row % 16 == 0 && aligned(all.x.codes, 16)));
  // a launch has fewer than 2^32 threads
  constexpr int kMostN = 1 << 24;
  for (int64_t n = 0; n < all.n; n += kMostN) {
    F8Product p = all;
    p.n = (int)std::min<int64_t>(all.n - n, kMostN);
    p.w.codes += n * p.w.row;
    p.w.scales += n / kF8Block * p.w.s_row;
    p.y += n * (p.half_out ? 2 : 4);
    const PlainRows rows{plain, plain_row};
    if (plain == nullptr)
      launch<kCodes>(p, rows, wide);
    else if (plain_half)
      launch<kF16>(p, rows, wide);
    else
      launch<kF32>(p, rows, wide);
  }
}

}  // namespace weft
