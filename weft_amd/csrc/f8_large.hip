// The product of 8-bit floats in tiles of 256 weights x 256 tokens, for calls that fill the card
// with them and end in 16 bits.
//
// Eight waves of 128 weights x 64 tokens, a step a block of K: operands are widened to 16-bit floats
// on their way from LDS (f8_many.hip says why), a wave's tokens once a step and its weights 16 rows
// (a phase) at a time, so that a matrix instruction of 16 x 16 x 32 needs one and a half conversions and
// one multiply-add.  The codes of a phase's weights and, in a step's last phase, of the next
// step's tokens are read a phase ahead; so at the last phase's barrier all of the step's operands are in
// registers, its place in LDS is loaded again at once, for the step after the next, and loads
// have a whole step to arrive.
//
// Bound by the matrix pipe (busy 54 % of the time), the VALU (51 %) and waits (31 % of the waves' time): 8192^3 of random
// codes takes 864 to 920 us, by the card (1.2 to 1.27 PF, at 2.2 GHz; tiles of 128 x 128 1010 to 1060), 4096^3 111 to 118 (137).
#include "f8_tile.h"
#include "runtime.h"

namespace weft {

namespace {

constexpr int kTile = 256, kWavesN = 2, kWavesM = 4, kWaves = kWavesN * kWavesM;
constexpr int kData = kTile * kF8Block;                       // of either operand and step
constexpr int kSlot = 2 * kData + (kTile + kWave) * 4;        // and the tokens' scales, the weights'
constexpr int RN = kTile / kWavesN / 16, RM = kTile / kWavesM / 16;

// At least two blocks of K.
__global__ void __launch_bounds__(kWaves * kWave, 2) f8_large_kernel(F8Product p, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int tm, tn;
  place((int)blockIdx.x, tiles_m, tiles_n, tm, tn);
  const int n0 = tn * kTile, m0 = tm * kTile;
  const int blocks = p.k / kF8Block;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)lds;

  // ---- loads: unit u of a wave is rows 8 (8 u + wave) .. + 7 of the weights (tokens).  Rows past the ends are
  // read as the last one.
  const int row8 = lane >> 3, chunk = (lane & 7) ^ (4 * (wave & 1) + (row8 >> 1));
  const uint8_t* w_base = p.w.codes + n0 * p.w.row;
  const uint8_t* x_base = p.x.codes + m0 * p.x.row;
  const uint32_t w_step = 64 * (uint32_t)p.w.row, x_step = 64 * (uint32_t)p.x.row;
  const uint32_t w_off = (uint32_t)(8 * wave + row8) * (uint32_t)p.w.row + 16 * chunk;
  const uint32_t x_off = (uint32_t)(8 * wave + row8) * (uint32_t)p.x.row + 16 * chunk;
  const uint32_t w_most = (uint32_t)(min(kTile, p.n - n0) - 1) * (uint32_t)p.w.row + 16 * chunk;
  const uint32_t x_most = (uint32_t)(min(kTile, p.m - m0) - 1) * (uint32_t)p.x.row + 16 * chunk;
  const bool of_tokens = wave < kTile / kWave;
  const int w_blocks = (p.n + kF8Block - 1) / kF8Block;
  const float* s_at = of_tokens ? p.x.scales + min(m0 + kWave * wave + lane, p.m - 1) * p.x.s_row
                                : p.w.scales + min(n0 / kF8Block + lane, w_blocks - 1) * p.w.s_row;
  const long long s_step = of_tokens ? p.x.s_block : p.w.s_block;
  const uint32_t s_lds = 2 * kData + (of_tokens ? wave * kWave * 4 : kTile * 4);
  constexpr int kLoads = 9;
  auto load = [&](int b) {
    const uint32_t to = lds0 + (b & 1) * kSlot;
    // offsets are computed anew each time: kept, they would not fit the registers
    uint32_t w = w_off, x = x_off;
    asm volatile("" : "+v"(w), "+v"(x));
#pragma unroll
    for (int u = 0; u < 4; ++u)
      dma16(w_base + (long long)b * kF8Block, min(w + u * w_step, w_most), to + (64 * u + 8 * wave) * kF8Block);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      dma16(x_base + (long long)b * kF8Block, min(x + u * x_step, x_most), to + kData + (64 * u + 8 * wave) * kF8Block);
    dma4(s_at + b * s_step, to + s_lds);
  };

  // ---- the wave's parts of 16 x 16.  A lane has two chunks of 16 of a row's codes (which of them an
  // instruction takes does not matter as weights and tokens have the same), the second 64 bytes from the first.
  const int r = lane & 15, g = lane >> 4;
  const int wn = wave % kWavesN, wm = wave / kWavesN;
  const int chunk16 = (g ^ (r >> 1)) * 16;
  auto codes = [&](int b, int row, int second) {
    return *reinterpret_cast<const int4*>(lds + (b & 1) * kSlot + row * kF8Block + ((chunk16 ^ 64 * second)));
  };
  const int w_row = 128 * wn + r, x_row = kTile + 64 * wm + r;
  half8 xh[RM][4];
  auto widen_tokens = [&](const int4 (&v)[RM], int second) {
#pragma unroll
    for (int j = 0; j < RM; ++j) {
      xh[j][2 * second] = halves(v[j].x, v[j].y);
      xh[j][2 * second + 1] = halves(v[j].z, v[j].w);
    }
  };
  auto read_tokens = [&](int b, int second, int4 (&v)[RM]) {
#pragma unroll
    for (int j = 0; j < RM; ++j) v[j] = codes(b, x_row + 16 * j, second);
  };

  v4f acc[RN][RM] = {};
  const v4f zero = {};
  load(0);
  load(1);
  arrive<kLoads>();
  int4 wc[2] = {codes(0, w_row, 0), codes(0, w_row, 1)}, xc[RM];
  read_tokens(0, 0, xc);
  widen_tokens(xc, 0);
  read_tokens(0, 1, xc);
  widen_tokens(xc, 1);
  for (int b = 0; b < blocks; ++b) {
    const float* scales = reinterpret_cast<const float*>(lds + (b & 1) * kSlot + 2 * kData);
    float f[RM];
#pragma unroll
    for (int j = 0; j < RM; ++j) f[j] = scales[kTile + wn] * scales[64 * wm + 16 * j + r];
#pragma unroll
    for (int phase = 0; phase < RN; ++phase) {
      const half8 wh[4] = {halves(wc[0].x, wc[0].y), halves(wc[0].z, wc[0].w), halves(wc[1].x, wc[1].y), halves(wc[1].z, wc[1].w)};
      const bool last = phase == RN - 1;
      if (last) {
        // the next step has arrived, and no wave reads this one's place any more
        arrive<0>();
        if (b + 2 < blocks) load(b + 2);
      }
      // (past the last step: what is there, not used)
#pragma unroll
      for (int s = 0; s < 2; ++s) wc[s] = codes(last ? b + 1 : b, w_row + (last ? 0 : 16 * (phase + 1)), s);
      v4f c[RM];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (last && q == 2) read_tokens(b + 1, 0, xc);
#pragma unroll
        for (int j = 0; j < RM; ++j) c[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[q], xh[j][q], q ? c[j] : zero, 0, 0, 0);
      }
      if (last) {
        widen_tokens(xc, 0);
        read_tokens(b + 1, 1, xc);
      }
#pragma unroll
      for (int j = 0; j < RM; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[phase][j][e] = fmaf(c[j][e], f[j], acc[phase][j][e]);
#pragma unroll
      for (int j = 0; j < RM; ++j) asm volatile("" : "+v"(acc[phase][j]));  // here, not behind the step's last barrier
      if (last) widen_tokens(xc, 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // ---- a lane has weights 4 g .. + 3 of token r of each part
  static_assert(kTile * kTileRow<kTile, _Float16> <= 2 * kSlot, "the tile fits");
  __syncthreads();  // every wave has left its operands
#pragma unroll
  for (int j = 0; j < RM; ++j)
#pragma unroll
    for (int i = 0; i < RN; ++i)
      tile_put<kTile, _Float16>(lds, 64 * wm + 16 * j + r, 128 * wn + 16 * i + 4 * g, acc[i][j][0], acc[i][j][1], acc[i][j][2],
                                acc[i][j][3]);
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
