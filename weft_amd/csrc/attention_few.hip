// Attention of few query rows a kv head: decode steps and short chunks.
//
// Bound by reading the cache, 4-bit codes by converting them beside that: 48
// sequences of up to 8192 Q8_0 tokens, 32 heads over 8 of 128 values, take 126 us
// (4.0 TB/s); one of 131072 Q4_0 tokens 52 us (2.9 TB/s, about 450 VALU
// instructions a wave and step, 65 % of the busy cycles); 1023 Q8_0 tokens 11.6 us
// with the join, both launches and a dozen dependent trips to memory.
//
// Each of a workgroup's four waves takes every
// fourth step of 32 keys of its split, alone, for the 16 rows of the tile,
// and the waves' results are joined in LDS at the end; splits are joined
// by a second kernel (attention.hip).
//
// The scores are formed transposed, S^T = K Q^T, with 16x16x32 products: keys
// down the rows, so a lane holds four keys of its own query in each and the
// softmax's maximum over keys is seven comparisons and two lane exchanges.  The
// weights are then already the right operand of O^T = V^T P^T: a lane's eight
// keys in any order serve as its eight contraction values, as long as V^T is
// read in the same order, which the transposing LDS read gives (four keys of one
// value column a lane).
//
// A product's left operand is eight values of a key a lane (Q4_0: four bytes, the
// values of both halves, the queries permuted to match).  Where a page's slots
// follow each other, 16 rows are whole 16-byte lines: those are loaded, put into
// LDS and taken from there as operands (read directly, 18- and 34-byte records cost
// the L1 cache 75 accesses a load instruction: 166 us for the batch above).  Other
// layouts load the records directly.  V's records are converted into LDS rows.
//
// Numbers: the codes of a quantized K are exact in 16 bits, so its products are
// too, and a record's step multiplies their 32-bit sum.  A query in 32 bits is
// two 16-bit parts, two products.  V's values are rounded to 16 bits (code times
// step); against them the weights are two parts as well, so that V's rounding is
// all that the sum carries, down to weights of 2^-25 of a row's largest.  A 16-bit V is exact and takes rounded weights.  A V whose
// values may be past 16 bits is added apart, in 32.
// Maximum, sum and accumulators are in 32 bits.
#include <algorithm>
#include <type_traits>

#include "attention.h"
#include "runtime.h"

namespace weft {
namespace {

constexpr int kWaves = 4, kStep = 32;

// A step's records as they are loaded.  kDense: whole 16-byte lines of them, 32
// rows one after the other, which LDS hands out as operands and units.
template <int T, int NB, bool kDense>
struct Raw {
  static constexpr int kVUnit = T == kKvF16 ? 4 * NB : T == kKvQ8_0 ? 2 * NB : NB;  // 16-byte units a row
  static constexpr int kV = (kVUnit * kStep + kWave - 1) / kWave;                  // units a lane
  static constexpr int kS = T == kKvF16 ? 1 : (NB + 3) / 4;                        // K steps a lane and 16 keys
  static constexpr int kKWords = T == kKvF16 ? 4 : T == kKvQ8_0 ? 2 : 1;
  static constexpr int kRowBytes = KvRecord<T>::kBytes * NB;
  static constexpr int kLines = kStep * kRowBytes / 16;  // a step's
  // those of a last part of at most 32 of K and V go together: lanes 0.. and 32..
  static constexpr int kRest = kLines % kWave <= 32 ? kLines % kWave : 0;
  static constexpr int kLine = (kLines - kRest + kWave - 1) / kWave;  // a lane's besides
  uint32_t k[2][NB][kKWords];
  uint32_t ks[2][kS];
  Bytes16 v[kV];
  uint32_t vs[T == kKvF16 ? 1 : kV];
};

// A line of records, read once a tile, which the caches need not keep: one token
// over 131072 Q8_0 keys takes 66 us instead of 70, 48 over up to 8192 124 instead of
// 125; 32 heads over one kv head, two tiles on the same lines, 26.5 instead of 25.9.
// (16-bit rows are not whole lines a load: eight chunks of 8 tokens would take 76 us instead of 64.)
__device__ __forceinline__ u32x4 once(const uint8_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

// a wave's place in LDS: V rows (padded by 32 bytes, so that eight rows of 32
// bytes fall on different banks), K's steps; O at the end lies over them
template <int NB>
struct Lds {
  static constexpr int kRow = 64 * NB + 32;
  static constexpr int kSteps = kStep * kRow;
  static constexpr int kBytes = kSteps + NB * kStep * 4;
  static constexpr int kORow = 32 * NB + 4;  // floats
  static_assert(16 * kORow * 4 <= kBytes && 2 * kStep * 34 * NB <= kSteps && 16 * kRow + kStep * 34 * NB <= kSteps,
                "the rows' sums, and a step's records beside half its V rows");
};

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int T, int NB, bool kDense>
__global__ void __launch_bounds__(kWaves* kWave, NB <= 4 ? 3 : 1) attend_few_kernel(AttendArgs a) {
  using L = Lds<NB>;
  using R = Raw<T, NB, kDense>;
  constexpr int D = 32 * NB;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves][L::kBytes];
  constexpr int kQRow = 64 * NB + 16;
  __shared__ __attribute__((aligned(16))) uint8_t qs[2][16 * kQRow];
  __shared__ float ml[kWaves][16][2];

  const int lane = threadIdx.x & (kWave - 1), wave = uniform((int)threadIdx.x / kWave);
  const int c = lane & 15, g = lane >> 4;  // query column (or key, value) and quarter
  const int item = a.first + (int)blockIdx.x, kvh = item % a.kv_heads;
  const int split = (int)blockIdx.y;
  TileRows t;
  if (!locate(a, item / a.kv_heads, -1, 0, t)) return;
  const int seq = t.seq;
  int step0 = 0, step1 = t.range.steps;
  bool whole = true;  // the tile has one split
  if (a.part != nullptr) {
    const int n = t.each;
    whole = n >= step1;
    step0 = min(split * n, step1);
    step1 = min(step0 + n, step1);
    if (split > 0 && step0 >= step1) return;
  }

  // The queries into LDS, as right operands: lane (c, g) reads row c's values
  // 8 g .. 8 g + 7 of a block (Q4_0: 4 g + j and 16 + 4 g + j) as 16 bytes; two
  // parts of 16 bits where they have 32.
  for (int i = threadIdx.x; i < 16 * 8 * NB; i += kWaves * kWave) {
    const int r = i / (8 * NB), e = i % (8 * NB), b = e / 8, four = e % 8;
    const int row = t.row0 + min(r, t.rows - 1);
    const int tok = row / a.share, head = kvh * a.share + row % a.share;
    const uint8_t* src = a.q + (long long)(t.token0 + tok) * a.q_token + (long long)head * a.q_head;
    f16x4 hi, lo;
    if (a.half_q) {
      hi = __builtin_bit_cast(f16x4, *reinterpret_cast<const Bytes8*>(src + 8 * e)) * (_Float16)a.sign;
      lo = f16x4{};
    } else {
      const float* x = reinterpret_cast<const float*>(src) + 4 * e;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = x[j] * a.sign;
        hi[j] = (_Float16)v;
        lo[j] = (_Float16)(v - (float)hi[j]);
      }
    }
    uint8_t* dst = qs[0] + r * kQRow + 64 * b + (T != kKvQ4_0 ? 8 * four : four < 4 ? 16 * four : 16 * (four - 4) + 8);
    *reinterpret_cast<f16x4*>(dst) = hi;
    *reinterpret_cast<f16x4*>(dst + 16 * kQRow) = lo;
  }
  int qpos;  // of lane c's row; -1: before the sequence
  {
    const int row = t.row0 + min(c, t.rows - 1);
    qpos = (int)max(-1ll, t.pos0 + row / a.share);
  }
  int qoff = c * kQRow + 16 * g;
  const int first_pos = (int)max(-1ll, t.pos0 + t.row0 / a.share);
  const int last_pos = (int)max(-1ll, t.pos0 + (t.row0 + t.rows - 1) / a.share);

  f32x4 o[2 * NB] = {};
  float ref = -INFINITY, l = 0.f;

  uint8_t* const vrow = lds[wave];
  float* const ksteps = reinterpret_cast<float*>(lds[wave] + L::kSteps);

  // The table's entry for a step's key `lane` (32 keys), looked up two steps
  // ahead and not looked at before it is needed: a check here would wait for the
  // load, and for the records loaded before it.  Past the table its last entry
  // stands in; no key there is present.
  auto entry_of = [&](int step) {
    if (step >= step1) return -1;
    const uint32_t pos = (uint32_t)(step_position<kStep>(t.range, step) + (lane & 31));
    const uint32_t entry = a.seqs.page_shift >= 0 ? pos >> a.seqs.page_shift : pos / (uint32_t)a.seqs.page_size;
    return a.seqs.pages[(long long)seq * a.seqs.pages_row + min(entry, (uint32_t)a.seqs.max_pages - 1)];
  };
  // -1 where that is no page
  auto page_of = [&](int entry) { return (uint32_t)entry < (uint32_t)a.seqs.n_pages ? entry : -1; };
  // A step's records: K as operands (lane c's key of each 16, quarter g's values),
  // V as rows of 16-byte units.  With whole groups of 16 keys in a page the bases
  // are scalars and a lane's offsets constants; where a row's units are a power of
  // two (>= 4), unit i of a lane is its unit 0 some whole rows on.  Else places are
  // computed at each step, behind a barrier to the optimizer, which would keep them
  // all in registers.  Absent keys read the pool's first row.
  constexpr bool kSame = R::kVUnit >= 4 && (R::kVUnit & (R::kVUnit - 1)) == 0;
  constexpr int kRowsOn = kWave / R::kVUnit;
  // where a lane's part of a row begins: K's values and steps, V's unit and its step
  auto k_part = [&](int quarter) { return T == kKvF16 ? 16 * quarter : T == kKvQ8_0 ? 2 + 8 * quarter : 2 + 4 * quarter; };
  auto v_part = [&](int e) { return T == kKvF16 ? 16 * e : T == kKvQ8_0 ? 34 * (e / 2) + 2 + 16 * (e & 1) : 18 * e + 2; };
  auto v_step = [&](int e) { return T == kKvQ8_0 ? 34 * (e / 2) : 18 * e; };
  const uint32_t krow = (uint32_t)c * (uint32_t)a.k.slot, vrow_off = (uint32_t)(lane / R::kVUnit) * (uint32_t)a.v.slot;
  const int e0 = lane % R::kVUnit;
  const uint32_t koff = krow + k_part(g), voff = vrow_off + v_part(e0), vsoff = vrow_off + v_step(e0);
  auto fetch_k = [&](const uint8_t* row, const uint8_t* part, R& r, int i) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
      __builtin_memcpy(r.k[i][b], __builtin_assume_aligned(part + b * KvRecord<T>::kBytes, 2), 4 * R::kKWords);
    if constexpr (T != kKvF16) {
#pragma unroll
      for (int s = 0; s < R::kS; ++s) r.ks[i][s] = ld_u16(row + KvRecord<T>::kBytes * min(4 * s + g, NB - 1));
    }
  };
  auto fetch_v = [&](const uint8_t* part, const uint8_t* step, R& r, int i) {
    r.v[i] = *reinterpret_cast<const Bytes16*>(part);
    if constexpr (T != kKvF16) r.vs[i] = ld_u16(step);
  };
  auto opaque_lane = [&] {
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  u32x4 klines[kDense ? R::kLine : 1], vlines[kDense ? R::kLine : 1], rest;
  auto load = [&](int step, int page, R& r, bool keys, bool values) {
    const int pos = step_position<kStep>(t.range, step);
    const uint8_t* kh = a.k.data + (long long)kvh * a.k.head;
    const uint8_t* vh = a.v.data + (long long)kvh * a.v.head;
    if (kDense || a.whole16) {
      const uint8_t *kb[2], *vb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t p = (uint32_t)max(__builtin_amdgcn_readlane(page, 16 * i), 0);
        const uint32_t slot = (uint32_t)(pos + 16 * i) & (uint32_t)(a.seqs.page_size - 1);
        kb[i] = kh + ((unsigned long long)p * (uint32_t)a.k.page + slot * (uint32_t)a.k.slot);
        vb[i] = vh + ((unsigned long long)p * (uint32_t)a.v.page + slot * (uint32_t)a.v.slot);
      }
      if constexpr (kDense) {
        // 16 rows are kHalf lines, the second 16 rows' may lie elsewhere
        constexpr int kHalf = R::kLines / 2, kWhole = R::kLines - R::kRest;
        static_assert(R::kRest == 0 || kWhole >= kHalf, "");
        auto lines = [&](const uint8_t* b0, const uint8_t* b1, u32x4 (&to)[kDense ? R::kLine : 1]) {
          b1 -= 16 * kHalf;
#pragma unroll
          for (int i = 0; i < R::kLine; ++i) {
            const int n0 = i * kWave, u = n0 + kWave <= kWhole ? n0 + lane : min(n0 + lane, kWhole - 1);
            const uint8_t* from = n0 + kWave <= kHalf ? b0 : n0 >= kHalf ? b1 : u < kHalf ? b0 : b1;
            to[i] = once(from + (uint32_t)(16 * u));
          }
        };
        if (values && R::kRest > 0)
          rest = once((lane < 32 ? kb[1] : vb[1]) + (uint32_t)(16 * (kWhole - kHalf + min(lane & 31, R::kRest - 1))));
        if (keys) lines(kb[0], kb[1], klines);
        if (values) lines(vb[0], vb[1], vlines);
        return;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (keys) fetch_k(kb[i] + krow, kb[i] + koff, r, i);
      }
      if (!values) return;
      if constexpr (kSame) {
#pragma unroll
        for (int i = 0; i < R::kV; ++i) {
          const uint8_t* base = vb[i * kRowsOn >= 16 ? 1 : 0] + (uint32_t)(i * kRowsOn & 15) * (uint32_t)a.v.slot;
          fetch_v(base + voff, base + vsoff, r, i);
        }
      } else {
        const int x = opaque_lane();
#pragma unroll
        for (int i = 0; i < R::kV; ++i) {
          const int u = i * kWave + x, key = min(u / R::kVUnit, kStep - 1), e = u % R::kVUnit;
          const uint8_t* row = (key & 16 ? vb[1] : vb[0]) + (uint32_t)(key & 15) * (uint32_t)a.v.slot;
          fetch_v(row + v_part(e), row + v_step(e), r, i);
        }
      }
      asm volatile("; whole groups");  // kept apart: merged with those below, the loads' addresses would all be kept
      return;
    }
    auto slot_of = [&](int at) {
      return a.seqs.page_shift >= 0 ? at & (a.seqs.page_size - 1) : (int)((uint32_t)at % (uint32_t)a.seqs.page_size);
    };
    const int x = opaque_lane();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = 16 * i + (x & 15), p = __shfl(page, key, kWave);
      const long long slot = p < 0 ? 0 : slot_of(pos + key);
      const uint8_t* row = kh + (long long)max(p, 0) * a.k.page + slot * a.k.slot;
      if (keys) fetch_k(row, row + k_part(g), r, i);
    }
#pragma unroll
    for (int i = 0; values && i < R::kV; ++i) {
      const int u = i * kWave + x, key = min(u / R::kVUnit, kStep - 1), e = u % R::kVUnit;
      const int p = __shfl(page, key, kWave);
      const long long slot = p < 0 ? 0 : slot_of(pos + key);
      const uint8_t* row = vh + (long long)max(p, 0) * a.v.page + slot * a.v.slot;
      fetch_v(row + v_part(e), row + v_step(e), r, i);
    }
  };

  __syncthreads();
  // heads up to 128: three waves a SIMD leave no registers for the next step's keys
  // beside this step's, which are loaded when its scores are done
  constexpr bool kLate = NB <= 4;
  // dense: V's lines in LDS; records lie at odd halfwords, but whole words are read
  // (LDS stalls on others) and shifted
  constexpr int kVRaw = L::kSteps - kStep * R::kRowBytes;
  auto word = [&](const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(__builtin_assume_aligned(p, 4)); };
  R raw;
  int step = step0 + wave;
  int page = page_of(entry_of(step)), next = entry_of(step + kWaves);
  if (step < step1) load(step, page, raw, true, true);
  for (; step < step1; step += kWaves) {
    const int pos = step_position<kStep>(t.range, step);
    // the keys that are there and that some row sees, key i as bit i
    uint32_t present = (uint32_t)__ballot(page >= 0);
    if (pos + kStep > t.range.end) present &= (uint32_t)first_bits(t.range.end - pos);
    if (a.window > 0 && pos <= first_pos - a.window)
      present &= (uint32_t)(~first_bits(first_pos - a.window - pos + 1) | first_bits(a.sinks - pos));
    // rows see different keys of this step
    const bool mixed = pos + kStep - 1 > first_pos ||
                       (a.window > 0 && pos <= last_pos - a.window && pos + kStep - 1 >= a.sinks);
    const bool masked = mixed || present != 0xffffffffu;

    if constexpr (kDense) {
      // the lines into the place of the V rows, V's at its end, and out as operands
      // and units
      constexpr int kWhole = R::kLines - R::kRest;
#pragma unroll
      for (int i = 0; i < R::kLine; ++i) {
        const int u = i * kWave + lane;
        if (u < kWhole) {
          *reinterpret_cast<u32x4*>(vrow + 16 * u) = klines[i];
          *reinterpret_cast<u32x4*>(vrow + kVRaw + 16 * u) = vlines[i];
        }
      }
      const int z = opaque_lane();
      if ((z & 31) < R::kRest)
        *reinterpret_cast<u32x4*>(vrow + (z < 32 ? 0 : kVRaw) + 16 * (kWhole + (z & 31))) = rest;
      wave_sync();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = (16 * i + c) * R::kRowBytes;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int at = row + b * KvRecord<T>::kBytes + k_part(g);
          if (R::kRowBytes % 4 == 0 && (b * KvRecord<T>::kBytes + 2) % 4 == 0) {
#pragma unroll
            for (int j = 0; j < R::kKWords; ++j) raw.k[i][b][j] = word(vrow + at + 4 * j);
            continue;
          }
          const uint8_t* from = vrow + (at & ~3);
          uint32_t w[R::kKWords + 1];
#pragma unroll
          for (int j = 0; j <= R::kKWords; ++j) w[j] = word(from + 4 * j);
#pragma unroll
          for (int j = 0; j < R::kKWords; ++j) raw.k[i][b][j] = __builtin_amdgcn_alignbyte(w[j + 1], w[j], at & 3);
        }
#pragma unroll
        for (int s = 0; s < R::kS; ++s) raw.ks[i][s] = ld_u16(vrow + row + KvRecord<T>::kBytes * min(4 * s + g, NB - 1));
      }
    }
    // a V unit out of the lines
    auto unit = [&](int i) {
      if constexpr (kDense) {
        int row, at, shift;
        if constexpr (kSame) {  // whole rows on, a multiple of four bytes
          constexpr int kOn = kRowsOn * R::kRowBytes;
          static_assert(kOn % 4 == 0, "");
          const int first = kVRaw + lane / R::kVUnit * R::kRowBytes;
          row = first + i * kOn;
          at = ((first + v_part(e0)) & ~3) + i * kOn;
          shift = (first + v_part(e0)) & 3;
          row += v_step(e0);
        } else {
          const int u = i * kWave + opaque_lane(), key = min(u / R::kVUnit, kStep - 1), e = u % R::kVUnit;
          row = kVRaw + key * R::kRowBytes;
          at = (row + v_part(e)) & ~3;
          shift = (row + v_part(e)) & 3;
          row += v_step(e);
        }
        const uint8_t* from = vrow + at;
        uint32_t w[5];
#pragma unroll
        for (int j = 0; j < 5; ++j) w[j] = word(from + 4 * j);
#pragma unroll
        for (int j = 0; j < 4; ++j) raw.v[i].w[j] = __builtin_amdgcn_alignbyte(w[j + 1], w[j], shift);
        raw.vs[i] = ld_u16(vrow + row);
      }
    };
    // The rows overwrite the lines: those of the first 16 keys lie before V's (and
    // over K's, which are read), so units that come in halves take half the registers.
    constexpr bool kHalves = kSame && R::kV % 2 == 0;
    // V into LDS rows; a key that no row sees is zeros (its memory may hold anything)
    // keys that some rows see whose values are not all finite, in steps whose rows see
    // different keys, or not all within 16 bits
    uint32_t spoiled = 0;
    unsigned long long past[R::kV];  // lanes whose unit i is past 16 bits
    const int x0 = kSame ? lane : opaque_lane();
#pragma unroll
    for (int i = 0; i < R::kV; ++i) {
      if constexpr (kDense) {
        constexpr int kEach = kHalves ? R::kV / 2 : R::kV;
        if (i % kEach == 0) {
#pragma unroll
          for (int j = 0; j < kEach; ++j) unit(i + j);
          wave_sync();
        }
      }
      const int u = i * kWave + x0;
      const int key = kSame ? i * kRowsOn + lane / R::kVUnit : u / R::kVUnit, e = kSame ? e0 : u % R::kVUnit;
      const bool live = R::kVUnit * kStep % kWave == 0 || key < kStep;
      bool zero = masked && !(present >> (key & 31) & 1u);
      if constexpr (T != kKvF16) past[i] = __ballot(past_half<T>(raw.vs[i]));
      if (T == kKvF16 && masked) {
        bool bad = false;
#pragma unroll
        for (int w = 0; w < 4; ++w) bad = bad || half_not_finite(raw.v[i].w[w]) || half_not_finite(raw.v[i].w[w] >> 16);
        bad = bad && !zero && live;  // the row is cleared below
        if (__ballot(bad)) {  // hardly ever
          uint32_t mine = bad ? 1u << (key & 31) : 0u;
#pragma unroll
          for (int s = 32; s > 0; s >>= 1) mine |= (uint32_t)__shfl_xor((int)mine, s, kWave);
          spoiled |= mine;
        }
      }
      if (live) {
        uint8_t* dst = vrow + key * L::kRow;
        if constexpr (T == kKvF16) {
          uint4 x = make_uint4(raw.v[i].w[0], raw.v[i].w[1], raw.v[i].w[2], raw.v[i].w[3]);
          if (zero) x = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(dst + 16 * e) = x;
        } else {
          const _Float16 s1 = zero ? (_Float16)0.f : __builtin_bit_cast(_Float16, (uint16_t)raw.vs[i]);
          const f16x2 s = {s1, s1};
          f16x2 x[2][8];
          if constexpr (T == kKvQ8_0) {
#pragma unroll
            for (int w = 0; w < 4; ++w) codes4<128>(raw.v[i].w[w] ^ 0x80808080u, x[0][2 * w], x[0][2 * w + 1]);
          } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              codes4<8>(raw.v[i].w[w] & 0x0f0f0f0fu, x[0][2 * w], x[0][2 * w + 1]);
              codes4<8>(raw.v[i].w[w] >> 4 & 0x0f0f0f0fu, x[1][2 * w], x[1][2 * w + 1]);
            }
          }
#pragma unroll
          for (int h = 0; h < (T == kKvQ8_0 ? 1 : 2); ++h) {
            uint32_t y[8];
#pragma unroll
            for (int w = 0; w < 8; ++w) y[w] = __builtin_bit_cast(uint32_t, x[h][w] * s);
            uint4* to = reinterpret_cast<uint4*>(dst + (T == kKvQ8_0 ? 32 * e : 64 * e + 32 * h));
            to[0] = make_uint4(y[0], y[1], y[2], y[3]);
            to[1] = make_uint4(y[4], y[5], y[6], y[7]);
          }
        }
      }
    }
    if constexpr (T != kKvF16) {
      unsigned long long any = 0;
#pragma unroll
      for (int i = 0; i < R::kV; ++i) any |= past[i];
      if (any) {  // hardly ever
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < R::kV; ++i) {
          const int u = i * kWave + opaque_lane();
          if (u < R::kVUnit * kStep && past[i] >> (u % kWave) & 1) mine |= 1u << (u / R::kVUnit);
        }
#pragma unroll
        for (int s = 32; s > 0; s >>= 1) mine |= (uint32_t)__shfl_xor((int)mine, s, kWave);
        spoiled = mine & present;
      }
    }
    // whole rows: their finite values too are added with the others, at the end
    if (spoiled != 0) wave_sync();
    for (uint32_t left = spoiled; left != 0; left &= left - 1)
      for (int i = opaque_lane(); i < 16 * NB; i += kWave)
        *reinterpret_cast<uint32_t*>(vrow + (__ffs(left) - 1) * L::kRow + 4 * i) = 0;
    // K's steps, times the scale, as [block][key]
    if constexpr (T != kKvF16) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 0; s < R::kS; ++s)
          if (4 * s + g < NB) ksteps[(4 * s + g) * kStep + 16 * i + c] = fp16_to_fp32(raw.ks[i][s]) * a.scale;
    }
    // K as operands
    auto k_operand = [&](int i, int b) {
      if constexpr (T == kKvF16) {
        return __builtin_bit_cast(f16x8, make_uint4(raw.k[i][b][0], raw.k[i][b][1], raw.k[i][b][2], raw.k[i][b][3]));
      } else {
        uint32_t w[R::kKWords];
#pragma unroll
        for (int j = 0; j < R::kKWords; ++j) {
          w[j] = raw.k[i][b][j];
          if constexpr (kLate) asm volatile("" : "+v"(w[j]));  // converted where it is used, not all at once before
        }
        f16x2 x[4];
        if constexpr (T == kKvQ8_0) {
          codes4<128>(w[0] ^ 0x80808080u, x[0], x[1]);
          codes4<128>(w[1] ^ 0x80808080u, x[2], x[3]);
        } else {
          codes4<8>(w[0] & 0x0f0f0f0fu, x[0], x[1]);
          codes4<8>(w[0] >> 4 & 0x0f0f0f0fu, x[2], x[3]);
        }
        return f16x8{x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
      }
    };
    f16x8 kf[2][NB];
    if constexpr (!kLate) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int b = 0; b < NB; ++b) kf[i][b] = k_operand(i, b);
    }
    wave_sync();
    // the next step's records are on their way while this one is worked on
    page = page_of(next);
    if (step + kWaves < step1) load(step + kWaves, page, raw, !kLate, true);
    next = entry_of(step + 2 * kWaves);

    // scores: key 16 i + 4 g + e of the lane's query
    f32x4 s[2] = {};
    asm volatile("" : "+v"(qoff));  // read at every step: in registers they would halve the waves
    auto scores = [&](auto two) {  // two: queries of two parts
      constexpr bool kTwo = decltype(two)::value;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const f16x8 qh = *reinterpret_cast<const f16x8*>(qs[0] + qoff + 64 * b);
        f16x8 ql;
        if constexpr (kTwo) ql = *reinterpret_cast<const f16x8*>(qs[1] + qoff + 64 * b);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f16x8 kx = kLate ? k_operand(i, b) : kf[i][b];
          f32x4 x = {};
          if constexpr (T == kKvF16) x = s[i];
          x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kx, qh, x, 0, 0, 0);
          if constexpr (kTwo) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kx, ql, x, 0, 0, 0);
          if constexpr (T == kKvF16) {
            s[i] = x;
          } else {
            const f32x4 step4 = *reinterpret_cast<const f32x4*>(ksteps + b * kStep + 16 * i + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] = fmaf(x[e], step4[e], s[i][e]);
          }
        }
      }
    };
    if (a.half_q)
      scores(std::false_type{});
    else
      scores(std::true_type{});
    if (kLate && step + kWaves < step1) load(step + kWaves, page, raw, true, false);

    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = s[e / 4][e % 4];
      if constexpr (T == kKvF16) x[e] *= a.scale;
    }
    if (masked) {
      // value e: key 16 (e / 4) + 4 g + e % 4
      const uint32_t seen = (uint32_t)seen_bits(a, present, pos, qpos) >> (4 * g);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = seen & 1u << (16 * (e / 4) + e % 4) ? x[e] : -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    top = quarters_max(top);
    if (__ballot(top - ref > kMost)) {
      const float now = fmaxf(ref, reference(top));
      const float f = now == -INFINITY ? 1.f : exp2_fast(ref - now);
      ref = now;
      l *= f;
#pragma unroll
      for (int v = 0; v < 2 * NB; ++v) o[v] *= f;
    }
    const float from = ref == -INFINITY ? 0.f : ref;
    f16x8 ph, pl;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = exp2_fast(x[e] - from);
      l += p;
      ph[e] = (_Float16)p;
      if constexpr (T != kKvF16) pl[e] = (_Float16)(p - (float)ph[e]);
    }

    // O^T += V^T P^T
    const int y = opaque_lane();  // addresses made here: kept, they would be one register too many
    uint8_t* const vfrom = vrow + (4 * (y >> 4) + (y & 15) / 4) * L::kRow + 8 * (y & 3);
#pragma unroll
    for (int v = 0; v < 2 * NB; ++v) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* LdsPtr;
      // a quarter's lane i: key 4 g + i / 4, values 4 (i % 4) .. of the 16 columns
      uint8_t* at = vfrom + 32 * v;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at + 16 * L::kRow));
      const f16x4 lo4 = __builtin_bit_cast(f16x4, lo), hi4 = __builtin_bit_cast(f16x4, hi);
      const f16x8 vf = {lo4[0], lo4[1], lo4[2], lo4[3], hi4[0], hi4[1], hi4[2], hi4[3]};
      o[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph, o[v], 0, 0, 0);
      if constexpr (T != kKvF16) o[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, o[v], 0, 0, 0);
    }
    // those keys reach the rows that see them, and no other
    while (spoiled) {
      const int key = __ffs(spoiled) - 1;
      spoiled &= spoiled - 1;
      int pg, slot;
      if (!kv_place(a.seqs, seq, pos + key, pg, slot)) continue;
      const uint8_t* row = a.v.data + (long long)kvh * a.v.head + pg * a.v.page + slot * a.v.slot;
      const int at = 4 * (key / 16) + key % 4;  // among the lane's weights
      float p = 0.f;
      f16x8 wh = ph, wl = pl;
      asm volatile("" : "+v"(wh), "+v"(wl));  // converted here, not beside every step's weights
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float w = (float)wh[e];
        if constexpr (T != kKvF16) w += (float)wl[e];
        p = e == at ? w : p;
      }
      p = __shfl(p, 16 * (key % 16 / 4) + c, kWave);
      if (seen_bits(a, 1ull, pos + key, qpos)) {
#pragma unroll
        for (int v = 0; v < 2 * NB; ++v)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[v][e] += p * value_of<T>(row, 16 * v + 4 * g + e);
            asm volatile("" ::: "memory");  // one value at a time: no registers for this path
          }
      }
    }
    wave_sync();
  }

  // join the waves through LDS
  __syncthreads();
  const float sum = quarters_sum(l);
  const int last = opaque_lane(), col = last & 15;
  float* mine = reinterpret_cast<float*>(lds[wave]) + col * L::kORow + last / 16 * 4;
#pragma unroll
  for (int v = 0; v < 2 * NB; ++v) *reinterpret_cast<f32x4*>(mine + 16 * v) = o[v];
  if (last < 16) ml[wave][col][0] = ref, ml[wave][col][1] = sum;
  __syncthreads();
  const int row = threadIdx.x / 16;
  if (row >= t.rows) return;
  float top = -INFINITY, w[kWaves], all = 0.f;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) top = fmaxf(top, ml[i][row][0]);
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    w[i] = top == -INFINITY ? 0.f : exp2_fast(ml[i][row][0] - top);
    all += w[i] * ml[i][row][1];
  }
  const int r = t.row0 + row;
  const float f = !whole ? 1.f : all == 0.f ? 0.f : 1.f / all;  // a row that sees nothing: zeros
  float* part = nullptr;
  if (!whole) {
    part = a.part + ((long long)item * a.splits + split) * 16 * (D + 2) + row * (D + 2);
    if (threadIdx.x % 16 == 0) part[D] = top, part[D + 1] = all;
  }
  uint8_t* dst =
      a.o + (long long)(t.token0 + r / a.share) * a.o_token + (long long)(kvh * a.share + r % a.share) * a.o_head;
  for (int e = 4 * (threadIdx.x % 16); e < D; e += 64) {
    f32x4 x = {};
#pragma unroll
    for (int i = 0; i < kWaves; ++i)
      x += w[i] * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds[i]) + row * L::kORow + e);
    x *= f;
    if (part != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) part[e + i] = x[i];
    } else if (a.half_o) {
      const f16x4 h = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
      *reinterpret_cast<Bytes8*>(dst + 2 * e) = __builtin_bit_cast(Bytes8, h);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<float*>(dst)[e + i] = x[i];
    }
  }
}

template <int T, int NB>
void launch(const AttendArgs& a, dim3 grid, hipStream_t st) {
  if constexpr (T != kKvF16) {
    if (a.dense) {
      attend_few_kernel<T, NB, true><<<grid, kWaves * kWave, 0, st>>>(a);
      return;
    }
  }
  attend_few_kernel<T, NB, false><<<grid, kWaves * kWave, 0, st>>>(a);
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

void attend_few(int type, int d, AttendArgs a, hipStream_t st) {
  for (; a.first < a.items; a.first += kMostItems) {
    const dim3 grid((unsigned)std::min(a.items - a.first, kMostItems), (unsigned)a.splits);
    switch (type) {
      case kKvF16: launch_d<kKvF16>(d, a, grid, st); break;
      case kKvQ8_0: launch_d<kKvQ8_0>(d, a, grid, st); break;
      default: launch_d<kKvQ4_0>(d, a, grid, st); break;
    }
    check_launch("attend_few_kernel");
    if (a.items - a.first <= kMostItems) break;  // first stays in 32 bits
  }
}

}  // namespace weft
