// The product of 8-bit floats in tiles of 256 weights x 256 tokens, for calls that fill the card
// with them and end in 16 bits (f8_many.hip says what the matrix instruction keeps).
//
// Eight waves of 128 weights x 64 tokens, a step a block of K.  A step has four phases, one
// for each 32 of a wave's weights; a phase multiplies two parts of 32 x 32.  Its weights and, in a step's
// last phase, the next step's tokens are read from LDS into registers a phase ahead, so
// that what they leave there is free at the next barrier and is loaded again at once, for
// the step after the next: loads are on their way for one to two steps and begin a
// quarter of a step at a time, after the phase's first products are under way.
//
// Bound by the clock that its power leaves it, the matrix pipe and the output's stores, which nothing
// covers: 8192^3 of random codes takes 492 to 544 us, by the card (2.0 to 2.2 PF), at about 1.95 GHz, the pipe busy 52 %
// of the time, and of zeros, the same instructions, 405 (2.7 PF).  Of
// copies with a part left out, without the scales' multiply-adds 517 us, without loads 456,
// without products 417; the stores take 29.  Tiles of 128 x 128 take 580.
#include <type_traits>

#include "f8_tile.h"
#include "runtime.h"

namespace weft {

namespace {

constexpr int kTile = 256, kWavesN = 2, kWavesM = 4, kWaves = kWavesN * kWavesM;
constexpr int kData = kTile * kF8Block;                       // of either operand and step
constexpr int kSlot = 2 * kData + (kTile + kWave) * 4;        // and the tokens' scales, the weights'
constexpr int RN = kTile / kWavesN / 32, RM = kTile / kWavesM / 32;
static_assert(RN == 4 && RM == 2, "phases and parts");

__global__ void __launch_bounds__(kWaves * kWave, 2) f8_large_kernel(F8Product p, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int tm, tn;
  place((int)blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int n0 = tn * kTile, m0 = tm * kTile;
  const int blocks = p.k / kF8Block;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)lds;

  // ---- loads.  Of a phase's 64 weights wave w has rows 128 (w / 4) + 32 phase + 8 (w % 4) .. + 7,
  // of the tokens 8 (8 u + w) .. + 7 (u < 4).  Rows past the ends are read as the last one.
  const int row8 = lane >> 3, chunk = (lane & 7) ^ (4 * (wave & 1) + (row8 >> 1));
  const int w_first = 128 * (wave >> 2) + 8 * (wave & 3);
  const uint8_t* w_base = p.w.codes + n0 * p.w.row;
  const uint8_t* x_base = p.x.codes + m0 * p.x.row;
  const uint32_t w_step = 32 * (uint32_t)p.w.row, x_step = 64 * (uint32_t)p.x.row;
  const uint32_t w_off = (uint32_t)(w_first + row8) * (uint32_t)p.w.row + 16 * chunk;
  const uint32_t x_off = (uint32_t)(8 * wave + row8) * (uint32_t)p.x.row + 16 * chunk;
  const uint32_t w_most = (uint32_t)(min(kTile, p.n - n0) - 1) * (uint32_t)p.w.row + 16 * chunk;
  const uint32_t x_most = (uint32_t)(min(kTile, p.m - m0) - 1) * (uint32_t)p.x.row + 16 * chunk;
  const bool of_tokens = wave < kTile / kWave;
  const int w_blocks = (p.n + kF8Block - 1) / kF8Block;
  const float* s_at = of_tokens ? p.x.scales + min(m0 + kWave * wave + lane, p.m - 1) * p.x.s_row
                                : p.w.scales + min(n0 / kF8Block + lane, w_blocks - 1) * p.w.s_row;
  const long long s_step = of_tokens ? p.x.s_block : p.w.s_block;
  const uint32_t s_lds = 2 * kData + (of_tokens ? wave * kWave * 4 : kTile * 4);

  // offsets are computed anew each time: kept, they would not fit the registers
  auto load_weights = [&](int b, int phase) {
    uint32_t off = w_off;
    asm volatile("" : "+v"(off));
    dma16(w_base + (long long)b * kF8Block, min(off + phase * w_step, w_most),
          lds0 + (b & 1) * kSlot + (w_first + 32 * phase) * kF8Block);
  };
  auto load_tokens = [&](int b, int part) {
    uint32_t off = x_off;
    asm volatile("" : "+v"(off));
#pragma unroll
    for (int u = 2 * part; u < 2 * part + 2; ++u)
      dma16(x_base + (long long)b * kF8Block, min(off + u * x_step, x_most),
            lds0 + (b & 1) * kSlot + kData + (64 * u + 8 * wave) * kF8Block);
    if (part == 0) dma4(s_at + b * s_step, lds0 + (b & 1) * kSlot + s_lds);
  };
  // a phase's share of a step's loads: four, three, one and one
  auto load_share = [&](int b, int phase) {
    if (phase < 2) load_tokens(b, phase);
    load_weights(b, phase);
  };

  // ---- the wave's parts
  const int r = lane & 31, h = lane >> 5;
  const int wn = wave % kWavesN, wm = wave / kWavesN;
  int place16[4];  // where a lane's chunks of a row lie
#pragma unroll
  for (int c = 0; c < 4; ++c) place16[c] = ((4 * (c >> 1) + 2 * h + (c & 1)) ^ (r >> 1 & 7)) * 16;
  auto operand = [&](const uint8_t* rows, int half) {
    const int4 a = *reinterpret_cast<const int4*>(rows + place16[2 * half]);
    const int4 b = *reinterpret_cast<const int4*>(rows + place16[2 * half + 1]);
    return v8i{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  };
  v8i wv[2][2], xv[RM][2];
  float f[RM], next_f[RM], next_w;  // the two scales' products; the next step's scales
  auto read_weights = [&](int b, int phase, v8i (&v)[2]) {
    int slot = (b & 1) * kSlot;
    asm volatile("" : "+s"(slot));
    const uint8_t* at = lds + slot + (128 * wn + 32 * phase + r) * kF8Block;
    v[0] = operand(at, 0);
    v[1] = operand(at, 1);
  };
  auto read_tokens = [&](int b, int j) {
    int slot = (b & 1) * kSlot;
    asm volatile("" : "+s"(slot));
    const uint8_t* at = lds + slot + kData + (64 * wm + 32 * j + r) * kF8Block;
    xv[j][0] = operand(at, 0);
    xv[j][1] = operand(at, 1);
  };
  auto read_scales = [&](int b) {
    const float* at = reinterpret_cast<const float*>(lds + (b & 1) * kSlot + 2 * kData);
    next_w = at[kTile + wn];
#pragma unroll
    for (int j = 0; j < RM; ++j) next_f[j] = at[64 * wm + 32 * j + r];
  };

  v16f acc[RN][RM] = {};
  const v16f zero = {};
  v16f c[2] = {zero, zero};
  float last_f = 0.f;  // of the part whose sums are in c and not yet added

#pragma unroll
  for (int phase = 0; phase < RN; ++phase) load_share(0, phase);
  if (blocks > 1) {
#pragma unroll
    for (int phase = 0; phase < RN; ++phase) load_share(1, phase);
    arrive<12>();
  } else {
    arrive<0>();
  }
  read_tokens(0, 0);
  read_tokens(0, 1);
  read_weights(0, 0, wv[0]);
  read_scales(0);

  // kMore: there is a step after the next
  auto step = [&](int b, auto more) {
    constexpr bool kMore = decltype(more)::value;
#pragma unroll
    for (int phase = 0; phase < RN; ++phase) {
      // the next phase's weights (the next step's tokens and first weights) have arrived when
      // only later loads are on their way; every wave has this phase's operands in registers
      if constexpr (!kMore) {
        arrive<0>();
      } else if (phase == 0 || phase == 3) {
        arrive<11>();
      } else if (phase == 1) {
        arrive<14>();
      } else {
        arrive<16>();
      }
#pragma unroll
      for (int j = 0; j < RM; ++j) {
        const int q = RM * phase + j, last = (q + RN * RM - 1) % (RN * RM);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // (the form without scales)
          c[q & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv[phase & 1][half], xv[j][half], half ? c[q & 1] : zero, 0, 0, 0,
                                                                     0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (kMore) {
          if (j == 0) load_share(b + 2, phase);
        }
        // (past the last step: what is there, not used)
        if (j == 0) read_weights(phase < 3 ? b : b + 1, (phase + 1) % RN, wv[(phase + 1) & 1]);
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[last / RM][last % RM][e] = fmaf(c[(q + 1) & 1][e], last_f, acc[last / RM][last % RM][e]);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" : "+v"(c[q & 1]), "+v"(acc[last / RM][last % RM]));  // not past the next barrier
        if (q == 0) {
#pragma unroll
          for (int i = 0; i < RM; ++i) f[i] = next_w * next_f[i];
        }
        last_f = f[j];
        if (phase == 3) {
          read_tokens(b + 1, j);
          if (j == 1) read_scales(b + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  int b = 0;
  for (; b + 2 < blocks; ++b) step(b, std::true_type{});
  for (; b < blocks; ++b) step(b, std::false_type{});

#pragma unroll
  for (int e = 0; e < 16; ++e) acc[RN - 1][RM - 1][e] = fmaf(c[1][e], last_f, acc[RN - 1][RM - 1][e]);

  // ---- a lane has weights 8 g + 4 h .. + 3 (g < 4) of token r of each part
  static_assert(kTile * kTileRow<kTile, _Float16> <= 2 * kSlot, "the tile fits");
  __syncthreads();  // every wave has left its operands
#pragma unroll
  for (int j = 0; j < RM; ++j)
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        tile_put<kTile, _Float16>(lds, 64 * wm + 32 * j + r, 128 * wn + 32 * i + 8 * g + 4 * h, acc[i][j][4 * g],
                                  acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
  __syncthreads();
  tile_store<kTile, kTile, kWaves * kWave, _Float16>(lds, p, n0, m0);
}

}  // namespace

void f8_large(const F8Product& p) {
  const int tiles_m = (p.m + kTile - 1) / kTile, tiles_n = (p.n + kTile - 1) / kTile;
  f8_large_kernel<<<dim3((unsigned)(tiles_m * tiles_n)), kWaves * kWave, 2 * kSlot, current_stream()>>>(p, tiles_m, tiles_n);
  check_launch("f8_large_kernel");
}

}  // namespace weft
