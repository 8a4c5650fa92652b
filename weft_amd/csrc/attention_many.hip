// Attention of many query rows a kv head: prompts and chunks.
//
// Bound by the matrix pipe and the softmax beside it, which two waves a SIMD overlap
// in part only: a prompt of 4096 16-bit tokens, 32 heads over 8 of 128 values, takes
// 169 to 180 us (0.76 to 0.81 PFLOP/s; the matrix pipe is busy for 34 % of it, the
// vector unit for 38 %, a quarter of a wave's time waits for records or the step's
// barrier); 512 tokens of 64 heads of 64 in a window of 4096 behind 32768 Q8_0 keys
// 73 us with the join (0.47 PFLOP/s); nine chunks of up to 640 tokens
// over up to 3001 Q4_0 keys with no shared heads 114 us (0.37 PFLOP/s: the
// longest tile's 47 steps; each workgroup converts the records for its 128 rows only).
//
// A workgroup owns 128 rows,
// 32 a wave, and walks the keys in steps of 64 (heads of 256: 32, for the
// registers' sake) that all waves share: the records
// are loaded into registers a step ahead, converted to 16-bit values once for the
// 128 rows, and written to one of two LDS buffers, one barrier a step.  Two
// workgroups fit a CU, so one's products run beside the other's softmax.
//
// As for few rows the scores are formed transposed (S^T = K Q^T, here with
// 32x32x16 products): a lane holds 32 keys of one query, the maximum needs one
// lane exchange, the accumulators' scale is one number a lane, and the weights
// are the right operand of O^T = V^T P^T without leaving their registers, V^T
// read by the transposing LDS read in the weights' key order.
//
// Numbers: queries, values of quantized keys and values, and weights are each
// rounded once to 16 bits (a second part of each would cost the matrix pipe as
// much again): against 64 bits the outputs are off by 3e-4 of their size over a
// 16-bit cache and 5e-4 over a quantized one, whose values' own rounding is 5e-3 and
// more.  Records of V that may be past 16 bits are added apart, in 32.  Products, maximum,
// sum and accumulators are in 32 bits.
#include <algorithm>

#include "attention.h"
#include "runtime.h"

namespace weft {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * kWave, kRows = 32;  // rows a wave

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int T, int NB>
struct Tile {
  static constexpr int kStep = many_step(32 * NB);
  static constexpr int kUnit = T == kKvF16 ? 4 * NB : T == kKvQ8_0 ? 2 * NB : NB;  // 16-byte units a row
  static constexpr int kUnits = (kUnit * kStep + kThreads - 1) / kThreads;          // a thread
  static constexpr bool kEven = kUnit * kStep % kThreads == 0;
  // rows in LDS: eight rows' 16 bytes of K fall on different banks, and four rows'
  // 64 of V (two quarters of a transposing read)
  static constexpr int kKRow = 64 * NB + 16, kVRow = 64 * NB + (NB % 2 ? 0 : 64);
  static constexpr int kV = kStep * kKRow, kBytes = kV + kStep * kVRow;
};

template <int T, int NB>
__global__ void __launch_bounds__(kThreads, NB <= 4 ? 2 : 1) attend_many_kernel(AttendArgs a) {
  using L = Tile<T, NB>;
  constexpr int D = 32 * NB, kStep = L::kStep, kPart = kStep / 32;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // two steps' tiles
  __shared__ unsigned long long spoiled_of[2][kWaves];
  __shared__ uint32_t met;  // whether any step had such a key, of quantized ones

  const int lane = threadIdx.x & (kWave - 1), wave = uniform((int)threadIdx.x / kWave), tid = threadIdx.x;
  const int c = lane & 31, h = lane >> 5;  // query column (or key, value) and half
  // a causal call's last tiles are its longest: they start first
  const int turn = a.first + (int)blockIdx.x, kvh = turn % a.kv_heads;
  const int tile = a.items / a.kv_heads - 1 - turn / a.kv_heads;
  const int split = (int)blockIdx.y;
  TileRows t;
  if (!locate(a, tile, -1, 0, t)) return;
  const int seq = t.seq;
  int step0 = 0, step1 = t.range.steps;
  bool whole = true;
  if (a.part != nullptr) {
    const int n = t.each;
    whole = n >= step1;
    step0 = min(split * n, step1);
    step1 = min(step0 + n, step1);
    if (split > 0 && step0 >= step1) return;
  }

  // this wave's queries, as right operands: lane c's row, values 16 b + 8 h + j
  f16x8 qf[2 * NB];
  const int wrow0 = t.row0 + min(kRows * wave, t.rows - 1), wrow1 = t.row0 + min(kRows * wave + kRows, t.rows) - 1;
  const bool idle = kRows * wave >= t.rows;  // no row of this wave
  const int row = t.row0 + min(kRows * wave + c, t.rows - 1);
  const int tok = row / a.share, head = kvh * a.share + row % a.share;
  const int qpos = (int)max(-1ll, t.pos0 + tok);
  const int first_pos = (int)max(-1ll, t.pos0 + wrow0 / a.share), last_pos = (int)max(-1ll, t.pos0 + wrow1 / a.share);
  // of the whole tile
  const int first_all = (int)max(-1ll, t.pos0 + t.row0 / a.share);
  const int last_all = (int)max(-1ll, t.pos0 + (t.row0 + t.rows - 1) / a.share);
  // The scale (at most 1: queries stay in range) goes into queries that are rounded
  // here anyway, and the scores' products begin at minus the row's reference, so that
  // they end as the weights' exponents.  16-bit queries stay exact.
  const bool folded = a.scale <= 1.f && !a.half_q;
  {
    const float qscale = folded ? a.sign * a.scale : a.sign;
    const uint8_t* src = a.q + (long long)(t.token0 + tok) * a.q_token + (long long)head * a.q_head;
    if (a.half_q) {
#pragma unroll
      for (int b = 0; b < 2 * NB; ++b)
        qf[b] = __builtin_bit_cast(f16x8, *reinterpret_cast<const Bytes16*>(src + 32 * b + 16 * h)) * (_Float16)a.sign;
    } else {
#pragma unroll
      for (int b = 0; b < 2 * NB; ++b) {
        const float* x = reinterpret_cast<const float*>(src) + 16 * b + 8 * h;
#pragma unroll
        for (int j = 0; j < 8; ++j) qf[b][j] = (_Float16)(x[j] * qscale);
      }
    }
  }

  f32x16 o[NB] = {};
  float ref = -INFINITY, l = 0.f;
  f32x16 minus = {};  // the reference, negative, in every place

  // The table's entry for a step's key `lane` (of 32: keys twice), looked up two steps
  // ahead and not looked at before it is needed: a check here would wait for the
  // load, and for the records loaded before it.  Past the table its last entry
  // stands in; no key there is present.
  auto entry_of = [&](int step) {
    if (step >= step1) return -1;
    const uint32_t pos = (uint32_t)(step_position<kStep>(t.range, step) + (lane & (kStep - 1)));
    const uint32_t entry = a.seqs.page_shift >= 0 ? pos >> a.seqs.page_shift : pos / (uint32_t)a.seqs.page_size;
    return a.seqs.pages[(long long)seq * a.seqs.pages_row + min(entry, (uint32_t)a.seqs.max_pages - 1)];
  };
  // -1 where that is no page
  auto page_of = [&](int entry) { return (uint32_t)entry < (uint32_t)a.seqs.n_pages ? entry : -1; };
  // the keys of a step that are there and that some row of the tile sees
  auto present_of = [&](int pos, int page) {
    unsigned long long present = __ballot(page >= 0);
    if (pos + kStep > t.range.end || (a.window > 0 && pos <= first_all - a.window)) {
      unsigned long long seen = first_bits(t.range.end - pos);
      if (a.window > 0) seen &= ~first_bits(first_all - a.window - pos + 1) | first_bits(a.sinks - pos);
      present &= seen;
    }
    return present;
  };
  Bytes16 rk[L::kUnits], rv[L::kUnits];
  uint32_t sk[L::kUnits], sv[L::kUnits];
  auto slot_of = [&](int at) {
    return a.seqs.page_shift >= 0 ? at & (a.seqs.page_size - 1) : (int)((uint32_t)at % (uint32_t)a.seqs.page_size);
  };
  // a unit of a row: 16 bytes of values or codes, and their step
  auto part_of = [&](int e) { return T == kKvF16 ? 16 * e : T == kKvQ8_0 ? 34 * (e / 2) + 2 + 16 * (e & 1) : 18 * e + 2; };
  auto step_of = [&](int e) { return T == kKvQ8_0 ? 34 * (e / 2) : 18 * e; };
  auto fetch = [&](const uint8_t* part, const uint8_t* step, Bytes16& b, uint32_t& s) {
    b = *reinterpret_cast<const Bytes16*>(part);
    if constexpr (T != kKvF16) s = ld_u16(step);
  };
  // Units per row a power of two: unit i of a thread is its unit 0 some whole rows
  // on, in the wave's half of the step, so one offset a thread serves them all.
  // Else (heads of 96 and 192) each unit's place is computed at each step, behind a
  // barrier to the optimizer, which would keep them all in registers.
  constexpr bool kSame = (L::kUnit & (L::kUnit - 1)) == 0;
  constexpr int kRowsOn = kThreads / L::kUnit;  // rows between a thread's units
  const int key0 = tid / L::kUnit, e0 = tid % L::kUnit;
  auto opaque_tid = [&] {
    int x = tid;
    asm volatile("" : "+v"(x));
    return x;
  };
  const uint32_t krow = (uint32_t)(key0 & 31) * (uint32_t)a.k.slot, vrow = (uint32_t)(key0 & 31) * (uint32_t)a.v.slot;
  const uint32_t koff = krow + part_of(e0), voff = vrow + part_of(e0);
  const uint32_t ksoff = krow + step_of(e0), vsoff = vrow + step_of(e0);
  auto load = [&](int step, int page) {
    const int pos = step_position<kStep>(t.range, step);
    const uint8_t* kh = a.k.data + (long long)kvh * a.k.head;
    const uint8_t* vh = a.v.data + (long long)kvh * a.v.head;
    if (a.whole32) {
      // 32 keys lie in one page
      const uint8_t *kb[2], *vb[2];
#pragma unroll
      for (int i = 0; i < kPart; ++i) {
        const uint32_t p = (uint32_t)max(__builtin_amdgcn_readlane(page, 32 * i), 0);
        const uint32_t slot = (uint32_t)(pos + 32 * i) & (uint32_t)(a.seqs.page_size - 1);
        kb[i] = kh + ((unsigned long long)p * (uint32_t)a.k.page + slot * (uint32_t)a.k.slot);
        vb[i] = vh + ((unsigned long long)p * (uint32_t)a.v.page + slot * (uint32_t)a.v.slot);
      }
      if constexpr (kSame) {
#pragma unroll
        for (int i = 0; i < L::kUnits; ++i) {
          // a wave's units lie in one half, whole rows on in it; those past the step
          // read its last rows again
          const bool half = kPart > 1 && (kRowsOn <= 32 ? i * kRowsOn >= 32 : uniform(key0) >= 32);
          constexpr int kOn = kRowsOn <= 32 ? kRowsOn : 32;
          const uint32_t on = (uint32_t)(i * kOn & 31);
          const uint8_t* kr = (half ? kb[1] : kb[0]) + on * (uint32_t)a.k.slot;
          const uint8_t* vr = (half ? vb[1] : vb[0]) + on * (uint32_t)a.v.slot;
          fetch(kr + koff, kr + ksoff, rk[i], sk[i]);
          fetch(vr + voff, vr + vsoff, rv[i], sv[i]);
        }
      } else {
        const int x = opaque_tid();
        const uint32_t ks = (uint32_t)a.k.slot, vs = (uint32_t)a.v.slot;
#pragma unroll
        for (int i = 0; i < L::kUnits; ++i) {
          const int u = i * kThreads + x, key = min(u / L::kUnit, kStep - 1), e = u % L::kUnit;
          const uint8_t* kr = (kPart > 1 && key & 32 ? kb[1] : kb[0]) + (key & 31) * ks;
          const uint8_t* vr = (kPart > 1 && key & 32 ? vb[1] : vb[0]) + (key & 31) * vs;
          fetch(kr + part_of(e), kr + step_of(e), rk[i], sk[i]);
          fetch(vr + part_of(e), vr + step_of(e), rv[i], sv[i]);
        }
      }
      return;
    }
    const int x = opaque_tid();
#pragma unroll
    for (int i = 0; i < L::kUnits; ++i) {
      const int u = i * kThreads + x, key = min(u / L::kUnit, kStep - 1), e = u % L::kUnit;
      const int p = __shfl(page, key, kWave);
      const long long slot = p < 0 ? 0 : slot_of(pos + key);
      const uint8_t* kr = kh + (long long)max(p, 0) * a.k.page + slot * a.k.slot;
      const uint8_t* vr = vh + (long long)max(p, 0) * a.v.page + slot * a.v.slot;
      fetch(kr + part_of(e), kr + step_of(e), rk[i], sk[i]);
      fetch(vr + part_of(e), vr + step_of(e), rv[i], sv[i]);
    }
  };
  // a unit's values, in 16 bits, into a row in LDS
  auto put = [&](const Bytes16& b, uint32_t step16, bool zero, uint8_t* dst, int e) {
    if constexpr (T == kKvF16) {
      uint4 x = make_uint4(b.w[0], b.w[1], b.w[2], b.w[3]);
      if (zero) x = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(dst + 16 * e) = x;
    } else {
      const _Float16 s1 = zero ? (_Float16)0.f : __builtin_bit_cast(_Float16, (uint16_t)step16);
      const f16x2 s = {s1, s1};
      f16x2 x[2][8];
      if constexpr (T == kKvQ8_0) {
#pragma unroll
        for (int w = 0; w < 4; ++w) codes4<128>(b.w[w] ^ 0x80808080u, x[0][2 * w], x[0][2 * w + 1]);
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          codes4<8>(b.w[w] & 0x0f0f0f0fu, x[0][2 * w], x[0][2 * w + 1]);
          codes4<8>(b.w[w] >> 4 & 0x0f0f0f0fu, x[1][2 * w], x[1][2 * w + 1]);
        }
      }
#pragma unroll
      for (int i = 0; i < (T == kKvQ8_0 ? 1 : 2); ++i) {
        uint32_t y[8];
#pragma unroll
        for (int w = 0; w < 8; ++w) y[w] = __builtin_bit_cast(uint32_t, x[i][w] * s);
        uint4* to = reinterpret_cast<uint4*>(dst + (T == kKvQ8_0 ? 32 * e : 64 * e + 32 * i));
        to[0] = make_uint4(y[0], y[1], y[2], y[3]);
        to[1] = make_uint4(y[4], y[5], y[6], y[7]);
      }
    }
  };
  // a step in which the tile's rows see different keys, or not all of them
  auto is_edge = [&](int pos, unsigned long long present) {
    return pos + kStep - 1 > first_all || (a.window > 0 && pos <= last_all - a.window && pos + kStep - 1 >= a.sinks) ||
           present != ~0ull;
  };
  // the loaded step into LDS buffer `buf`; V of a key that no row sees is zeros
  auto store = [&](int step, int page, int buf) {
    const int x = kSame ? tid : opaque_tid();
    const int pos = step_position<kStep>(t.range, step);
    const unsigned long long present = present_of(pos, page);
    const bool edge = is_edge(pos, present);
    uint8_t* base = lds + buf * L::kBytes;
    // keys whose rows (records, where there are some) stay out of the products
    unsigned long long spoiled = 0;
    bool past = false;
#pragma unroll
    for (int i = 0; i < L::kUnits; ++i) {
      const int u = i * kThreads + x;
      const int key = kSame ? i * kRowsOn + key0 : u / L::kUnit, e = kSame ? e0 : u % L::kUnit;
      if (!L::kEven && key >= kStep) continue;
      put(rk[i], sk[i], false, base + key * L::kKRow, e);
      bool zero = false;
      if (edge) {
        zero = !((uint32_t)(key & 32 ? present >> 32 : present) >> (key & 31) & 1u);
        if constexpr (T == kKvF16) {
          bool bad = false;
#pragma unroll
          for (int w = 0; w < 4; ++w) bad = bad || half_not_finite(rv[i].w[w]) || half_not_finite(rv[i].w[w] >> 16);
          if (bad && !zero) spoiled |= 1ull << key;
        }
      }
      if constexpr (T != kKvF16) {
        const bool mine = past_half<T>(sv[i]);
        past = past || mine;
        zero = zero || mine;
      }
      put(rv[i], sv[i], zero, base + L::kV + key * L::kVRow, e);
    }
    if (T != kKvF16 && __ballot(past)) {  // hardly ever
#pragma unroll
      for (int i = 0; i < L::kUnits; ++i) {
        const int u = i * kThreads + x, key = kSame ? i * kRowsOn + key0 : u / L::kUnit;
        if (key < kStep && past_half<T>(sv[i]) && present >> key & 1) spoiled |= 1ull << key;
      }
    }
    if (T != kKvF16 || edge) {
      if (__ballot(spoiled != 0)) {  // hardly ever
#pragma unroll
        for (int s = 32; s > 0; s >>= 1)
          spoiled |= (unsigned long long)__shfl_xor((long long)spoiled, s, kWave);
      }
      if (lane == 0) spoiled_of[buf][wave] = spoiled;
      if (T != kKvF16 && spoiled != 0) met = 1;
    }
  };

  if constexpr (T != kKvF16) {
    if (tid == 0) met = 0;
    __syncthreads();
  }
  int page = page_of(entry_of(step0)), next = entry_of(step0 + 1);
  if (step0 < step1) {
    load(step0, page);
    store(step0, page, 0);
  }
  __syncthreads();
  for (int step = step0; step < step1; ++step) {
    const int buf = (step - step0) & 1;
    const int pos = step_position<kStep>(t.range, step);
    const unsigned long long present = present_of(pos, page);
    const int next_page = page_of(next);
    if (step + 1 < step1) load(step + 1, next_page);
    next = entry_of(step + 2);

    // Keys with values that are not finite, where rows see different keys: their whole
    // rows are cleared, once every thread's part is there, and reach the rows that see
    // them at the end.  Of a quantized key the records past 16 bits were not stored.
    unsigned long long spoiled = 0;
    uint32_t any = 0;
    if constexpr (T != kKvF16) any = met;  // looked at after the products
    if (T == kKvF16 && is_edge(pos, present)) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) spoiled |= spoiled_of[buf][w];
      spoiled = (unsigned long long)(uint32_t)uniform((int)(spoiled >> 32)) << 32 | (uint32_t)uniform((int)spoiled);
      if (spoiled != 0) {  // for all of the workgroup's threads, or none
        for (unsigned long long left = spoiled; left != 0; left &= left - 1)
          if (const int i = opaque_tid(); i < 16 * NB)
            *reinterpret_cast<uint32_t*>(lds + buf * L::kBytes + L::kV + __builtin_ctzll(left) * L::kVRow + 4 * i) = 0;
        __syncthreads();
      }
    }

    // rows of this wave see none, different, or all of the step's keys
    const bool none = idle || pos > last_pos ||
                      (a.window > 0 && pos + kStep - 1 <= first_pos - a.window && pos >= a.sinks);
    const bool masked = pos + kStep - 1 > first_pos ||
                        (a.window > 0 && pos <= last_pos - a.window && pos + kStep - 1 >= a.sinks) || present != ~0ull;
    if (!none) {
      const uint8_t* base = lds + buf * L::kBytes;
      f32x16 s[kPart];
      // operands come two blocks ahead of their products; the barriers keep the
      // scheduler from fetching them all at once, which the registers would not hold
      constexpr int kAhead = 2;
      // the SIMD's other wave gets what the products leave: its softmax or its loads
      __builtin_amdgcn_s_setprio(1);
      f16x8 kf[kAhead][kPart];
      auto k_at = [&](int b, int i) {
        return *reinterpret_cast<const f16x8*>(base + (32 * i + c) * L::kKRow + 32 * b + 16 * h);
      };
#pragma unroll
      for (int b = 0; b < kAhead; ++b)
#pragma unroll
        for (int i = 0; i < kPart; ++i) kf[b][i] = k_at(b, i);
#pragma unroll
      for (int b = 0; b < 2 * NB; ++b) {
#pragma unroll
        for (int i = 0; i < kPart; ++i) {
          s[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[b % kAhead][i], qf[b], b == 0 ? minus : s[i], 0, 0, 0);
          if (b + kAhead < 2 * NB) kf[b % kAhead][i] = k_at(b + kAhead, i);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      const bool first = ref == -INFINITY;
      const float ref0 = first ? 0.f : ref;
      if (!folded) {
#pragma unroll
        for (int i = 0; i < kPart; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[i][e] = fmaf(s[i][e], a.scale, -ref0);
      }
      float top;
      if (masked) {
        // value e of half i: key 32 i + 8 (e / 4) + 4 h + e % 4
        const unsigned long long seen = seen_bits(a, present, pos, qpos) >> (4 * h);
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPart; ++i) {
          const uint32_t bits = (uint32_t)(seen >> (32 * i));
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s[i][e] = bits & 1u << (8 * (e / 4) + e % 4) ? s[i][e] : -INFINITY;
            top = fmaxf(top, s[i][e]);
          }
        }
      } else {
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPart; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) top = fmaxf(top, s[i][e]);
      }
      {
        typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
      }
      if (__ballot(top > (first ? -INFINITY : kMost))) {
        // the scores are over the reference already; it moves by
        float by = reference(top);
        if (top == -INFINITY || (!first && by < 0.f)) by = 0.f;
        const float now = ref0 + by;
        if (fabsf(now) < 0x1p22f) by = now - ref0;  // as it is rounded
        const float f = first ? 0.f : exp2_fast(-by);  // at first there are no sums
        if (!first || top != -INFINITY) ref = now;
        l *= f;
#pragma unroll
        for (int v = 0; v < NB; ++v) o[v] *= f;
#pragma unroll
        for (int i = 0; i < kPart; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[i][e] -= by;
        if (folded) {
#pragma unroll
          for (int e = 0; e < 16; ++e) minus[e] = -now;
        }
      }
      f16x8 p[2 * kPart];
      auto weigh = [&](int k, int from, int to) {  // weights [from, to) of p[k]
#pragma unroll
        for (int e = from; e < to; ++e) {
          const float w = exp2_fast(s[k / 2][8 * (k & 1) + e]);
          l += w;
          p[k][e] = (_Float16)w;
        }
      };
      weigh(0, 0, 8);
      // O^T += V^T P^T: 16 keys a product, four of a quarter's and four 8 on; the next
      // products' weights are computed while these run
      {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4* LdsPtr;
        const int i = lane & 15;
        uint8_t* const vbase = lds + buf * L::kBytes + L::kV + (4 * h + i / 4) * L::kVRow + 32 * (lane >> 4 & 1) + 8 * (i & 3);
        auto v_at = [&](int n) {  // product n: keys 16 (n / NB), values 32 (n % NB)
          uint8_t* at = vbase + 16 * (n / NB) * L::kVRow + 64 * (n % NB);
          const f16x4 lo = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at)));
          const f16x4 hi = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at + 8 * L::kVRow)));
          return f16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        };
        constexpr int kAheadV = 4;
        f16x8 vf[kAheadV];
#pragma unroll
        for (int n = 0; n < kAheadV; ++n) vf[n] = v_at(n);
#pragma unroll
        for (int n = 0; n < 2 * kPart * NB; ++n) {
          o[n % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[n % kAheadV], p[n / NB], o[n % NB], 0, 0, 0);
          if (n + kAheadV < 2 * kPart * NB) vf[n % kAheadV] = v_at(n + kAheadV);
          const int k = n / NB + 1, v = n % NB;
          if (k < 2 * kPart) weigh(k, 4 * v / NB * 2, 4 * (v + 1) / NB * 2);
          __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("" : "+v"(l));  // summed here: 32 weights more in registers would not fit
      }
      if constexpr (T != kKvF16) {
        if (uniform((int)any) != 0) {
#pragma unroll
          for (int w = 0; w < kWaves; ++w) spoiled |= spoiled_of[buf][w];
        }
      }
      while (spoiled) {
        const int key = __builtin_ctzll(spoiled);
        spoiled &= spoiled - 1;
        int pg, slot;
        if (!kv_place(a.seqs, seq, pos + key, pg, slot)) continue;
        const uint8_t* vr = a.v.data + (long long)kvh * a.v.head + pg * a.v.page + slot * a.v.slot;
        const int want = 16 * (key / 32) + 4 * (key % 32 / 8) + key % 4;
        float w = 0.f;
#pragma unroll
        for (int k = 0; k < 2 * kPart; ++k) {
          f16x8 pk = p[k];
          asm volatile("" : "+v"(pk));  // converted here, not beside every step's weights
#pragma unroll
          for (int e = 0; e < 8; ++e) w = 8 * k + e == want ? (float)pk[e] : w;
        }
        w = __shfl(w, 32 * (key / 4 & 1) + c, kWave);
        if (seen_bits(a, 1ull, pos + key, qpos)) {
#pragma unroll
          for (int v = 0; v < NB; ++v) {
            if (T != kKvF16 && !past_half<T>(uniform((int)ld_u16(vr + v * KvRecord<T>::kBytes)))) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              o[v][e] += w * value_of<T>(vr, 32 * v + 8 * (e / 4) + 4 * h + e % 4);
              asm volatile("" ::: "memory");  // one value at a time: no registers for this path
            }
          }
        }
      }
    }
    page = next_page;
    if (step + 1 < step1) store(step + 1, page, buf ^ 1);
    __syncthreads();
  }

  // a lane has value 32 v + 8 (e / 4) + 4 h + e % 4 of its row
  if (kRows * wave + c >= t.rows) return;
  {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if (!whole) {
    // the item's number in the sequences' order, as the join counts it
    const long long item = (long long)tile * a.kv_heads + kvh;
    float* part = a.part + (item * a.splits + split) * (kWaves * kRows) * (D + 2) + (kRows * wave + c) * (D + 2);
#pragma unroll
    for (int v = 0; v < NB; ++v)
#pragma unroll
      for (int e = 0; e < 16; ++e) part[32 * v + 8 * (e / 4) + 4 * h + e % 4] = o[v][e];
    if (h == 0) part[D] = ref, part[D + 1] = l;
    return;
  }
  const float f = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: zeros
  uint8_t* dst = a.o + (long long)(t.token0 + tok) * a.o_token + (long long)head * a.o_head;
#pragma unroll
  for (int v = 0; v < NB; ++v)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int e = 32 * v + 8 * g + 4 * h;
      const float x[4] = {o[v][4 * g] * f, o[v][4 * g + 1] * f, o[v][4 * g + 2] * f, o[v][4 * g + 3] * f};
      if (a.half_o) {
        const f16x4 y = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
        *reinterpret_cast<Bytes8*>(dst + 2 * e) = __builtin_bit_cast(Bytes8, y);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<float*>(dst)[e + i] = x[i];
      }
    }
}

template <int T, int NB>
void launch(const AttendArgs& a, dim3 grid, hipStream_t st) {
  constexpr size_t kLds = 2 * Tile<T, NB>::kBytes;
  attend_many_kernel<T, NB><<<grid, kThreads, kLds, st>>>(a);
}

template <int T>
void launch_d(int d, const AttendArgs& a, dim3 grid, hipStream_t st) {
  switch (d) {
    case 64: launch<T, 2>(a, grid, st); break;
    case 96: launch<T, 3>(a, grid, st); break;
    case 128: launch<T, 4>(a, grid, st); break;
    case 192: launch<T, 6>(a, grid, st); break;
    default: launch<T, 8>(a, grid, st); break;
  }
}

}  // namespace

void attend_many(int type, int d, AttendArgs a, hipStream_t st) {
  for (; a.first < a.items; a.first += kMostItems) {
    const dim3 grid((unsigned)std::min(a.items - a.first, kMostItems), (unsigned)a.splits);
    switch (type) {
      case kKvF16: launch_d<kKvF16>(d, a, grid, st); break;
      case kKvQ8_0: launch_d<kKvQ8_0>(d, a, grid, st); break;
      default: launch_d<kKvQ4_0>(d, a, grid, st); break;
    }
    check_launch("attend_many_kernel");
    if (a.items - a.first <= kMostItems) break;  // first stays in 32 bits
  }
}

}  // namespace weft
