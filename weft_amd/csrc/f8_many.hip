// The product of 8-bit floats for many tokens: tiles of TN weights x TM tokens, K a block of
// 128 values at a time.
//
// A step's rows (128 bytes each) and scales come to LDS by direct 16-byte loads some steps
// ahead; a row's eight chunks of 16 bytes lie at places XORed with the row, so that the
// rows of an operand read meet in different banks.  Waves own 32 x 32 parts of the tile:
// a block's sums start at zero on the matrix pipe, then go to the part's sums times the two
// scales, one multiply-add a value (a lane has one token, so one factor).
//
// Operands are widened to 16-bit floats on their way from LDS: e4m3 numbers are 16-bit floats, so products are
// exact, and sums have 32 bits.  The matrix instructions that take the codes as they are run at twice the
// rate, but cut each eight products of a lane below 2^-13 of the largest one's power of two (measured on
// the device), so that sums whose large products cancel, or that have one large product beside small ones, lose
// more than a 16-bit output's own rounding; they are not used.
//
// Bound by the parts of a step, which hardly overlap, and, where K is cut into ranges, by writing and
// reading their sums: 2048 tokens x 4096 x 4096 take 73 us by 128-token tiles (0.94 PF), 8192^3 to 32 bits 1013 (1.09
// PF), 24 x 11008 x 4096 10.2 (4.4 TB/s of weights) and 2.5 to 4 for the sums.  Tried with the instructions that cut, without gain: 256 x 128 tiles,
// operands read from LDS a step ahead, three and four blocks' places for 128 tokens, priority for the products,
// workgroups of a CU half a step apart.
#include <algorithm>

#include "f8_tile.h"
#include "runtime.h"

namespace weft {

__device__ uint4 g_f8_zeros;  // the chunks past a row's end

namespace {

template <int TN, int TM, int WN, int WM, int STAGES, typename Out, bool kDirect>
struct Shape {
  static constexpr int kTn = TN, kTm = TM, kWn = WN, kWm = WM;
  static constexpr int kWaves = WN * WM, kThreads = kWaves * kWave;
  static constexpr int RN = TN / WN / 32, RM = TM / WM / 32;  // 32 x 32 parts of a wave
  static constexpr int kData = (TN + TM) * kF8Block;
  static constexpr int kTokenWaves = (TM + kWave - 1) / kWave;  // which load the tokens' scales
  static constexpr int kSlot = kData + (kTokenWaves + 1) * kWave * 4;  // and the tokens' scales, the weights'
  static constexpr int kLds = STAGES * kSlot;
  static constexpr int kLoadsN = TN / 8 / kWaves, kLoadsM = TM / 8 / kWaves, kLoads = kLoadsN + kLoadsM + 1;
  static_assert(TN % (8 * kWaves) == 0 && TM % (8 * kWaves) == 0 && kTokenWaves + 1 <= kWaves, "whole loads");
  static_assert(kDirect || STAGES == 2, "loads through registers fill the other slot");
};

// K in `n` ranges of `each` blocks, whose sums go to the work buffer as the lanes have them, a
// tile after the other; n == 1: straight to the output.
struct Parts {
  float* sums;
  long long range;  // floats between ranges: whole tiles
  int n, each;
};
// of a lane's first four values of a part, in groups of four
template <class S>
__device__ __forceinline__ long long sum_place(int tile, int wave, int part, int lane) {
  return (((long long)tile * S::kWaves + wave) * (S::RN * S::RM) + part) * 4 * kWave + lane;
}

// Two waves a SIMD, so that all registers are plain ones: sums in the matrix pipe's own are
// copied out one by one (two instructions a value).  Loads through registers need more than that leaves.
template <int TN, int TM, int WN, int WM, int STAGES, typename Out, bool kDirect>
__global__ void __launch_bounds__(64 * WN * WM, kDirect ? 2 : 1) f8_many_kernel(F8Product p, Parts parts, int tiles_m,
                                                                 int tiles_n) {
  using S = Shape<TN, TM, WN, WM, STAGES, Out, kDirect>;
  constexpr int RN = S::RN, RM = S::RM, LN = S::kLoadsN, LM = S::kLoadsM;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int tm, tn;
  place((int)blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int n0 = tn * TN, m0 = tm * TM;
  const int first = (int)blockIdx.y * parts.each;
  const int blocks = min((p.k + kF8Block - 1) / kF8Block - first, parts.each);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)lds;

  // ---- loads: unit i of a wave is rows 8 (i waves + wave) .. + 7 of the weights (tokens)
  const int row8 = lane >> 3, chunk = (lane & 7) ^ (4 * (wave & 1) + (row8 >> 1));
  const uint8_t* w_base = p.w.codes + n0 * p.w.row;
  const uint8_t* x_base = p.x.codes + m0 * p.x.row;
  // rows past the ends are read as the last one and not stored
  auto w_row = [&](int i) { return min(n0 + 8 * (i * S::kWaves + wave) + row8, p.n - 1) - n0; };
  auto x_row = [&](int i) { return min(m0 + 8 * (i * S::kWaves + wave) + row8, p.m - 1) - m0; };
  uint32_t w_off[LN], x_off[LM];
  if constexpr (kDirect) {
#pragma unroll
    for (int i = 0; i < LN; ++i) w_off[i] = (uint32_t)w_row(i) * (uint32_t)p.w.row + 16 * chunk;
#pragma unroll
    for (int i = 0; i < LM; ++i) x_off[i] = (uint32_t)x_row(i) * (uint32_t)p.x.row + 16 * chunk;
  }
  // the first waves load tokens' scales, the others the weights' (the same ones)
  const bool of_tokens = wave < S::kTokenWaves;
  const int w_blocks = (p.n + kF8Block - 1) / kF8Block;
  const float* s_at = of_tokens ? p.x.scales + min(m0 + kWave * wave + lane, p.m - 1) * p.x.s_row
                                : p.w.scales + min(n0 / kF8Block + lane, w_blocks - 1) * p.w.s_row;
  const long long s_step = of_tokens ? p.x.s_block : p.w.s_block;
  const uint32_t s_lds = S::kData + (of_tokens ? wave : S::kTokenWaves) * kWave * 4;

  auto issue = [&](int step, int slot) {
    const int b = first + step;
    const uint32_t to = lds0 + slot * S::kSlot;
    const uint8_t* w = w_base + (long long)b * kF8Block;
    const uint8_t* x = x_base + (long long)b * kF8Block;
    if ((b + 1) * kF8Block <= p.k) {
#pragma unroll
      for (int i = 0; i < LN; ++i) dma16(w, w_off[i], to + (i * S::kWaves + wave) * 1024);
#pragma unroll
      for (int i = 0; i < LM; ++i) dma16(x, x_off[i], to + TN * kF8Block + (i * S::kWaves + wave) * 1024);
    } else {  // chunks past k are zeros
      const bool in = b * kF8Block + 16 * chunk < p.k;
      const uint8_t* zeros = reinterpret_cast<const uint8_t*>(&g_f8_zeros);
#pragma unroll
      for (int i = 0; i < LN; ++i) dma16(in ? w + w_off[i] : zeros, to + (i * S::kWaves + wave) * 1024);
#pragma unroll
      for (int i = 0; i < LM; ++i) dma16(in ? x + x_off[i] : zeros, to + TN * kF8Block + (i * S::kWaves + wave) * 1024);
    }
    dma4(s_at + b * s_step, to + s_lds);
  };

  // ---- the same through registers, for rows of any alignment
  uint4 held[kDirect ? 1 : LN + LM];
  float held_scale = 0.f;
  auto fetch = [&](int step) {
    const int b = first + step, at = b * kF8Block + 16 * chunk;
    if ((b + 1) * kF8Block <= p.k) {
#pragma unroll
      for (int i = 0; i < LN; ++i) held[i] = codes16(w_base + w_row(i) * p.w.row + at);
#pragma unroll
      for (int i = 0; i < LM; ++i) held[LN + i] = codes16(x_base + x_row(i) * p.x.row + at);
    } else {
#pragma unroll
      for (int i = 0; i < LN; ++i) held[i] = codes16(w_base + w_row(i) * p.w.row, at, p.k);
#pragma unroll
      for (int i = 0; i < LM; ++i) held[LN + i] = codes16(x_base + x_row(i) * p.x.row, at, p.k);
    }
    held_scale = s_at[b * s_step];
  };
  auto put = [&](int slot) {
    uint8_t* to = lds + slot * S::kSlot;
#pragma unroll
    for (int i = 0; i < LN; ++i) *reinterpret_cast<uint4*>(to + (i * S::kWaves + wave) * 1024 + 16 * lane) = held[i];
#pragma unroll
    for (int i = 0; i < LM; ++i)
      *reinterpret_cast<uint4*>(to + TN * kF8Block + (i * S::kWaves + wave) * 1024 + 16 * lane) = held[LN + i];
    *reinterpret_cast<float*>(to + s_lds + 4 * lane) = held_scale;
  };

  // ---- the wave's parts of the tile
  const int r = lane & 31, h = lane >> 5;
  const int wn = wave % WN, wm = wave / WN;
  v16f acc[RN][RM] = {};
  const v16f zero = {};
  int place16[4];  // where a lane's chunks of a row lie: 16 bytes each of K 64 (c / 2) + 32 h + 16 (c & 1)
#pragma unroll
  for (int c = 0; c < 4; ++c) place16[c] = ((4 * (c >> 1) + 2 * h + (c & 1)) ^ (r >> 1 & 7)) * 16;
  auto operand = [&](const uint8_t* rows, int half) {
    const int4 a = *reinterpret_cast<const int4*>(rows + place16[2 * half]);
    const int4 b = *reinterpret_cast<const int4*>(rows + place16[2 * half + 1]);
    return v8i{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  };
  auto compute = [&](int slot) {
    const uint8_t* w = lds + slot * S::kSlot + (wn * (TN / WN) + r) * kF8Block;
    const uint8_t* x = lds + slot * S::kSlot + TN * kF8Block + (wm * (TM / WM) + r) * kF8Block;
    const float* scales = reinterpret_cast<const float*>(lds + slot * S::kSlot + S::kData);
    const float sw = scales[S::kTokenWaves * kWave + wn * (TN / WN) / kF8Block];
    float s[RM];
#pragma unroll
    for (int j = 0; j < RM; ++j) s[j] = sw * scales[wm * (TM / WM) + 32 * j + r];
    half8 xh[RM][8];
#pragma unroll
    for (int j = 0; j < RM; ++j)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const v8i v = operand(x + 32 * j * kF8Block, half);
#pragma unroll
        for (int q = 0; q < 4; ++q) xh[j][4 * half + q] = halves(v[2 * q], v[2 * q + 1]);
      }
#pragma unroll
    for (int i = 0; i < RN; ++i) {
      half8 wh[8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const v8i v = operand(w + 32 * i * kF8Block, half);
#pragma unroll
        for (int q = 0; q < 4; ++q) wh[4 * half + q] = halves(v[2 * q], v[2 * q + 1]);
      }
#pragma unroll
      for (int j = 0; j < RM; ++j) {
        v16f c = zero;
#pragma unroll
        for (int q = 0; q < 8; ++q) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(wh[q], xh[j][q], c, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = fmaf(c[e], s[j], acc[i][j][e]);
      }
    }
  };

  if constexpr (kDirect) {
#pragma unroll
    for (int b = 0; b < STAGES - 1; ++b)
      if (b < blocks) issue(b, b);
    int slot = 0;
    for (int b = 0; b < blocks; ++b) {
      // step b has arrived when only the steps after it are on their way
      if (b + STAGES - 1 <= blocks)
        arrive<(STAGES - 2) * S::kLoads>();
      else
        arrive<0>();
      // the slot of step b - 1, which every wave has left
      if (b + STAGES - 1 < blocks) issue(b + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
      compute(slot);
      slot = slot + 1 == STAGES ? 0 : slot + 1;
    }
  } else {
    fetch(0);
    put(0);
    for (int b = 0; b < blocks; ++b) {
      __syncthreads();
      if (b + 1 < blocks) fetch(b + 1);
      compute(b & 1);
      if (b + 1 < blocks) put((b + 1) & 1);  // the slot of step b - 1, which every wave has left
    }
  }

  // ---- a lane has weights 8 g + 4 h .. + 3 (g < 4) of token r of each part
  if (parts.n > 1) {
    v4f* to = reinterpret_cast<v4f*>(parts.sums + blockIdx.y * parts.range) + sum_place<S>(tm * tiles_n + tn, wave, 0, lane);
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
      for (int j = 0; j < RM; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const v16f& a = acc[i][j];
          to[((i * RM + j) * 4 + g) * kWave] = v4f{a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]};
        }
    return;
  }
  __syncthreads();  // every wave has left its operands
  static_assert(TM * kTileRow<TN, Out> <= S::kLds, "the tile fits");
#pragma unroll
  for (int j = 0; j < RM; ++j)
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        tile_put<TN, Out>(lds, wm * (TM / WM) + 32 * j + r, wn * (TN / WN) + 32 * i + 8 * g + 4 * h, acc[i][j][4 * g],
                          acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
  __syncthreads();
  tile_store<TN, TM, S::kThreads, Out>(lds, p, n0, m0);
}

// The ranges' sums added in their order.  A workgroup has 32 tokens of a tile and kSpan times 32 of its
// weights, and stores them by way of LDS: 509 x 4101 outputs of 16 bits, three ranges, take 7.5 us,
// straight from the registers 10.7.
template <class S, int kSpan, typename Out>
__global__ void __launch_bounds__(256) f8_join_kernel(F8Product p, Parts parts, int tiles_n) {
  constexpr int kWide = 32 * kSpan, kStripsN = S::kTn / kWide, kStrips = kStripsN * (S::kTm / 32);
  __shared__ __attribute__((aligned(16))) uint8_t lds[32 * kTileRow<kWide, Out>];
  const int lane = threadIdx.x & (kWave - 1), g = threadIdx.x / kWave;
  const int tile = (int)blockIdx.x / kStrips, strip = (int)blockIdx.x % kStrips;
  const int sm = strip / kStripsN, sn = strip % kStripsN;
  v4f v[kSpan];
  const v4f* at[kSpan];
#pragma unroll
  for (int q = 0; q < kSpan; ++q) {
    const int i = sn * kSpan + q;
    const int wave = sm / S::RM * S::kWn + i / S::RN, part = i % S::RN * S::RM + sm % S::RM;
    at[q] = reinterpret_cast<const v4f*>(parts.sums) + sum_place<S>(tile, wave, part, lane) + g * kWave;
    v[q] = *at[q];
  }
#pragma unroll 4
  for (int s = 1; s < parts.n; ++s)
#pragma unroll
    for (int q = 0; q < kSpan; ++q) v[q] += at[q][s * (parts.range / 4)];
#pragma unroll
  for (int q = 0; q < kSpan; ++q)
    tile_put<kWide, Out>(lds, lane & 31, 32 * q + 8 * g + 4 * (lane >> 5), v[q][0], v[q][1], v[q][2], v[q][3]);
  __syncthreads();
  tile_store<kWide, 32, 256, Out>(lds, p, tile % tiles_n * S::kTn + sn * kWide, tile / tiles_n * S::kTm + 32 * sm);
}

template <int TN, int TM, int WN, int WM, int STAGES, typename Out, bool kDirect>
void launch(const F8Product& p, const Parts& parts) {
  using S = Shape<TN, TM, WN, WM, STAGES, Out, kDirect>;
  const int tiles_m = (p.m + TM - 1) / TM, tiles_n = (p.n + TN - 1) / TN;
  f8_many_kernel<TN, TM, WN, WM, STAGES, Out, kDirect>
      <<<dim3((unsigned)(tiles_m * tiles_n), (unsigned)parts.n), S::kThreads, S::kLds, current_stream()>>>(p, parts, tiles_m,
                                                                                                       tiles_n);
  check_launch("f8_many_kernel");
  if (parts.n > 1) {
    constexpr int kSpan = TM / 32;
    const dim3 grid((unsigned)(tiles_m * tiles_n * (TN / (32 * kSpan)) * (TM / 32)));
    f8_join_kernel<Shape<TN, TM, WN, WM, 2, Out, false>, kSpan, Out><<<grid, 256, 0, current_stream()>>>(p, parts, tiles_n);
    check_launch("f8_join_kernel");
  }
}

// What a call takes: tiles of 128 weights x 32, 64 or 128 tokens, two workgroups of them a CU, with
// K in ranges, or of 256 x 256 (16-bit outputs, whole blocks), by the least of these times.
struct Plan {
  int tokens;     // of a tile: 256, 128, 64 or 32
  bool alone;     // on its CU, a workgroup
  Parts parts;
  int64_t large;  // of the weights go by tiles of 256, the rest as it would alone
  double us;
};

// us, measured.  3 to begin; a step (a block of K) of a workgroup alone on its CU, and of each of several, and what a
// workgroup takes beside its steps are in kCost; of 256 x 256 3.4 a step and 7, in a round that does not fill
// the card 2.75 to 3.35 and 8; ranges are written and read again at about 5.5 TB/s
// and joined by a launch of their own (3).  So 509 x 4101 x 11008 takes three ranges of 128-token tiles (69 us; 64-token
// tiles 77, 32 88), 512 x 4096 x 4096 one of 64 (27.7; two of 128 29.4), 600 x 9000 x 512 the same (12.1; of 128
// 13.6, of 256 21), 2048 x 4096 x 4096 one of 128 (73; of 64 82), 24 x 11008 x 4096 five of 32 (13; 64-token
// tiles 18), 4096 x 4096 x 4096 tiles of 256 (118; 128 139), which also take the weights of whole rounds
// where others take the rest.
// Costs go by K, as rows' alignment is not the shapes' and the work buffer's size is: rows of an even K
// that direct loads do not take are cut as those that they do.
constexpr int kCus = 256;
struct Cost {
  double alone, shared, each;
};
// K in whole 16 bytes and others; 32, 64 and 128 tokens
constexpr Cost kCost[2][3] = {{{0.54, 0.37, 0.6}, {0.75, 0.57, 0.8}, {1.21, 1.0, 1.3}}, {{0.85, 0.57, 0.6}, {1.1, 0.85, 0.8}, {1.7, 1.72, 1.3}}};
double rounds_us(int64_t tiles, int64_t blocks) {
  const double part = (double)(tiles % kCus) / kCus;
  return (double)(tiles / kCus) * (3.4 * (double)blocks + 7) + (part > 0 ? (2.75 + 0.6 * part) * (double)blocks + 8 : 0);
}
Plan plan_of(int64_t m, int64_t n, int64_t k, bool half_out) {
  const int64_t blocks = f8_blocks(k);
  Plan best{};
  for (const int tokens : {32, 64, 128, 256}) {
    // (tiles of 256 load two blocks before they begin)
    if (tokens == 256 && (!half_out || k % kF8Block != 0 || blocks < 2)) continue;
    const int64_t rows = tokens == 256 ? 256 : 128;
    const int64_t tiles = ((m + tokens - 1) / tokens) * ((n + rows - 1) / rows);
    const Cost& cost = kCost[k % 16 != 0][tokens == 32 ? 0 : tokens == 64 ? 1 : 2];
    for (int64_t want = 1; want <= 16 && (want == 1 || (tokens < 256 && tiles * want <= 2 * kCus && blocks >= 4 * want)); ++want) {
      const int64_t each = (blocks + want - 1) / want, parts = (blocks + each - 1) / each;
      const int64_t load = (tiles * parts + kCus - 1) / kCus;
      double us = 3;
      if (tokens == 256)
        us += rounds_us(tiles, blocks);
      else
        us += (double)load * ((double)each * (load == 1 ? cost.alone : cost.shared) + cost.each);
      if (parts > 1) us += 3 + (double)parts * (double)m * (double)n * 4 * 2 / 5.5e6;
      if (best.us > 0 && us >= best.us) continue;
      best.us = us;
      best.tokens = tokens;
      best.alone = load == 1;
      best.parts.n = (int)parts;
      best.parts.each = (int)each;
      best.parts.range = tiles * tokens * rows;
    }
    // whole rounds of large tiles and the rest
    const int64_t rounds = tiles / kCus, large = rounds * kCus / ((m + tokens - 1) / tokens) * rows;
    if (tokens == 256 && large > 0 && large < n) {
      Plan rest = plan_of(m, n - large, k, half_out);
      rest.us += rounds_us(rounds * kCus, blocks);
      if (rest.us < best.us) {
        best = rest;
        best.large = large;
      }
    }
  }
  return best;
}

// A launch has fewer than 2^31 threads: a call in pieces of at most 65536 tokens and weights.
template <class F>
void in_launches(const F8Product& all, F launch) {
  constexpr int kMost = 1 << 16;
  for (int64_t m = 0; m < all.m; m += kMost)
    for (int64_t n = 0; n < all.n; n += kMost) {
      F8Product p = all;
      p.m = (int)std::min<int64_t>(all.m - m, kMost);
      p.n = (int)std::min<int64_t>(all.n - n, kMost);
      p.x.codes += m * p.x.row;
      p.x.scales += m * p.x.s_row;
      p.w.codes += n * p.w.row;
      p.w.scales += n / kF8Block * p.w.s_row;
      p.y += m * p.y_row + n * (p.half_out ? 2 : 4);
      launch(p);
    }
}

}  // namespace

size_t f8_many_work(int64_t m, int64_t n, int64_t k) {
  // for either output type
  size_t most = 0;
  for (const bool half_out : {false, true}) {
    const Plan plan = plan_of(m, n, k, half_out);
    if (plan.parts.n > 1) most = std::max(most, (size_t)plan.parts.n * (size_t)plan.parts.range * sizeof(float));
  }
  return most;
}

void f8_many(const F8Product& all, float* work) {
  // direct loads take rows in aligned chunks of 16 and 32-bit offsets in a tile
  const bool direct = all.k % 16 == 0 && all.w.row % 16 == 0 && all.x.row % 16 == 0 && aligned(all.w.codes, 16) &&
                      aligned(all.x.codes, 16) && all.w.row < (1 << 24) && all.x.row < (1 << 24);
  Plan plan = plan_of(all.m, all.n, all.k, all.half_out);
  if (plan.large > 0 && direct) {
    F8Product p = all;
    p.n = (int)plan.large;
    in_launches(p, [](const F8Product& q) { f8_large(q); });
    p = all;
    p.n -= (int)plan.large;
    p.w.codes += plan.large * p.w.row;
    p.w.scales += plan.large / kF8Block * p.w.s_row;
    p.y += plan.large * 2;
    f8_many(p, work);
    return;
  }
  if (plan.large > 0 || (plan.tokens == 256 && !direct)) {
    plan.tokens = 128;
    plan.parts.n = 1;
    plan.parts.each = (int)f8_blocks(all.k);
  }
  plan.parts.sums = work;
  const Parts& parts = plan.parts;
  in_launches(all, [&](const F8Product& p) {
    const auto run = [&](auto out) {
      using Out = decltype(out);
      // Steps' places in LDS, of 32 and 64 tokens: three where a workgroup is alone on its CU, so that a step has
      // two others' time to arrive; two where others run beside it, of which a CU then takes three (us, three
      // places and two: 32 x 5120 x 5120 10.9 and 11.8, 64 x 8192 x 8192 19.6 and 21.1; 24 x 11008 x 4096
      // 14.2 and 13.2, 512 x 11008 x 4096 59.5 and 54.1).
      if (plan.tokens == 32)
        !direct      ? launch<128, 32, 4, 1, 2, Out, false>(p, parts)
        : plan.alone ? launch<128, 32, 4, 1, 3, Out, true>(p, parts)
                     : launch<128, 32, 4, 1, 2, Out, true>(p, parts);
      else if (plan.tokens == 64)
        !direct      ? launch<128, 64, 4, 1, 2, Out, false>(p, parts)
        : plan.alone ? launch<128, 64, 4, 1, 3, Out, true>(p, parts)
                     : launch<128, 64, 4, 1, 2, Out, true>(p, parts);
      else
        direct ? launch<128, 128, 2, 2, 2, Out, true>(p, parts) : launch<128, 128, 2, 2, 2, Out, false>(p, parts);
    };
    if (plan.tokens == 256)
      f8_large(p);
    else if (all.half_out)
      run(_Float16{});
    else
      run(float{});
  });
}

}  // namespace weft
