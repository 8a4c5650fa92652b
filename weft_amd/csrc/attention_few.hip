// Attention of few query rows a kv head: decode steps and short chunks.
//
// Bound by reading the cache.  Each of a workgroup's four waves takes every
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
// K never passes through LDS: a product's left operand is eight values of a key
// a lane, which is a direct load of the record (Q4_0: four bytes, the values of
// both halves, the queries permuted to match).  V's records are converted into
// LDS rows.
//
// Numbers: the codes of a quantized K are exact in 16 bits, so its products are
// too, and a record's step multiplies their 32-bit sum.  A query in 32 bits is
// two 16-bit parts, two products.  V's values are rounded to 16 bits (code times
// step); against them the weights are two parts as well, so that V's rounding is
// all that the sum carries.  A 16-bit V is exact and takes rounded weights.
// Maximum, sum and accumulators are in 32 bits.
#include "attention.h"
#include "runtime.h"

namespace weft {
namespace {

constexpr int kWaves = 4, kStep = 32;

template <int T, int NB>
struct Raw {  // a step's records: K as operands, V as rows
  static constexpr int kVUnit = T == kKvF16 ? 4 * NB : T == kKvQ8_0 ? 2 * NB : NB;  // 16-byte units a row
  static constexpr int kV = (kVUnit * kStep + kWave - 1) / kWave;                  // units a lane
  static constexpr int kS = T == kKvF16 ? 1 : (NB + 3) / 4;                        // K steps a lane and 16 keys
  static constexpr int kKWords = T == kKvF16 ? 4 : T == kKvQ8_0 ? 2 : 1;
  uint32_t k[2][NB][kKWords];
  uint32_t ks[2][kS];
  Bytes16 v[kV];
  uint32_t vs[T == kKvF16 ? 1 : kV];
};

// a wave's place in LDS: V rows (padded by 32 bytes, so that eight rows of 32
// bytes fall on different banks), K's steps; O at the end lies over them
template <int NB>
struct Lds {
  static constexpr int kRow = 64 * NB + 32;
  static constexpr int kSteps = kStep * kRow;
  static constexpr int kBytes = kSteps + NB * kStep * 4;
  static constexpr int kORow = 32 * NB + 4;  // floats
  static_assert(16 * kORow * 4 <= kBytes, "a group of rows' sums fit");
};

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int T, int NB, int RT>
__global__ void __launch_bounds__(kWaves* kWave, NB <= 4 ? 2 : 1) attend_few_kernel(AttendArgs a) {
  using L = Lds<NB>;
  using R = Raw<T, NB>;
  constexpr int D = 32 * NB;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kWaves][L::kBytes];
  __shared__ float ml[kWaves][16][2];

  const int lane = threadIdx.x & (kWave - 1), wave = uniform((int)threadIdx.x / kWave);
  const int c = lane & 15, g = lane >> 4;  // query column (or key, value) and quarter
  const int kvh = (int)blockIdx.x % a.kv_heads;
  const int split = (int)blockIdx.y;
  int tile;
  const int seq = find_tile(a, (int)blockIdx.x / a.kv_heads, tile);
  TileRows t;
  if (seq < 0 || !tile_rows(a, seq, tile, t)) return;
  int step0 = 0, step1 = t.range.steps;
  bool whole = true;  // the tile has one split
  if (a.part != nullptr) {
    const int n = split_steps(a);
    whole = n >= step1;
    step0 = min(split * n, step1);
    step1 = min(step0 + n, step1);
    if (split > 0 && step0 >= step1) return;
  }

  // the queries, as right operands: lane c's row, values 8 g + j of each block
  // (Q4_0: 4 g + j and 16 + 4 g + j)
  f16x8 qh[RT][NB], ql[RT][NB];
  int qpos[RT];  // -1: before the sequence
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = t.row0 + min(16 * rt + c, t.rows - 1);
    const int tok = row / a.share, head = kvh * a.share + row % a.share;
    qpos[rt] = (int)max(-1ll, t.pos0 + tok);
    const uint8_t* src = a.q + (long long)(t.token0 + tok) * a.q_token + (long long)head * a.q_head;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int e = 32 * b + (T == kKvQ4_0 ? 4 * g + (j & 3) + 4 * (j & 4) : 8 * g + j);
        const float x = a.sign * (a.half_q ? (float)*reinterpret_cast<const _Float16*>(src + 2 * e)
                                           : *reinterpret_cast<const float*>(src + 4 * e));
        qh[rt][b][j] = (_Float16)x;
        ql[rt][b][j] = (_Float16)(x - (float)qh[rt][b][j]);
      }
  }
  const int first_pos = (int)max(-1ll, t.pos0 + t.row0 / a.share);
  const int last_pos = (int)max(-1ll, t.pos0 + (t.row0 + t.rows - 1) / a.share);

  f32x4 o[RT][2 * NB] = {};
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) m[rt] = -INFINITY, l[rt] = 0.f;

  uint8_t* const vrow = lds[wave];
  float* const ksteps = reinterpret_cast<float*>(lds[wave] + L::kSteps);

  // page of a step's key `lane & 31`, -1 where it is absent
  auto pages_of = [&](int step) {
    int page = -1, slot;
    if (step < step1 && !kv_place(a.seqs, seq, step_position<kStep>(t.range, step) + (lane & 31), page, slot)) page = -1;
    return page;
  };
  // addresses: key's row in a pool, absent keys at the pool's first row
  auto load = [&](int step, int page, R& r) {
    const int pos = step_position<kStep>(t.range, step);
    const long long kh = (long long)kvh * a.k.head, vh = (long long)kvh * a.v.head;
    if (a.whole16) {
      const uint8_t *kb[2], *vb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t p = (uint32_t)max(__builtin_amdgcn_readlane(page, 16 * i), 0);
        const uint32_t slot = (uint32_t)(pos + 16 * i) & (uint32_t)(a.seqs.page_size - 1);
        kb[i] = a.k.data + kh + ((unsigned long long)p * (uint32_t)a.k.page + slot * (uint32_t)a.k.slot);
        vb[i] = a.v.data + vh + ((unsigned long long)p * (uint32_t)a.v.page + slot * (uint32_t)a.v.slot);
      }
      const int ks = (int)a.k.slot, vs = (int)a.v.slot;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int off = c * ks + (T == kKvF16 ? 64 * b + 16 * g : T == kKvQ8_0 ? 34 * b + 2 + 8 * g : 18 * b + 2 + 4 * g);
          __builtin_memcpy(r.k[i][b], __builtin_assume_aligned(kb[i] + off, 2), 4 * R::kKWords);
        }
        if constexpr (T != kKvF16) {
#pragma unroll
          for (int s = 0; s < R::kS; ++s)
            r.ks[i][s] = ld_u16(kb[i] + c * ks + KvRecord<T>::kBytes * min(4 * s + g, NB - 1));
        }
      }
#pragma unroll
      for (int i = 0; i < R::kV; ++i) {
        const int u = i * kWave + lane, key = min(u / R::kVUnit, kStep - 1), e = u % R::kVUnit;
        const uint8_t* row = (key & 16 ? vb[1] : vb[0]) + (key & 15) * vs;
        if constexpr (T == kKvF16) {
          r.v[i] = *reinterpret_cast<const Bytes16*>(row + 16 * e);
        } else if constexpr (T == kKvQ8_0) {
          r.v[i] = *reinterpret_cast<const Bytes16*>(row + 34 * (e / 2) + 2 + 16 * (e & 1));
          r.vs[i] = ld_u16(row + 34 * (e / 2));
        } else {
          r.v[i] = *reinterpret_cast<const Bytes16*>(row + 18 * e + 2);
          r.vs[i] = ld_u16(row + 18 * e);
        }
      }
      return;
    }
    auto slot_of = [&](int at) {
      return a.seqs.page_shift >= 0 ? at & (a.seqs.page_size - 1) : (int)((uint32_t)at % (uint32_t)a.seqs.page_size);
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = __shfl(page, 16 * i + c, kWave);
      const uint8_t* row = a.k.data + kh + (long long)max(p, 0) * a.k.page +
                           (long long)(p < 0 ? 0 : slot_of(pos + 16 * i + c)) * a.k.slot;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int off = T == kKvF16 ? 64 * b + 16 * g : T == kKvQ8_0 ? 34 * b + 2 + 8 * g : 18 * b + 2 + 4 * g;
        __builtin_memcpy(r.k[i][b], __builtin_assume_aligned(row + off, 2), 4 * R::kKWords);
      }
      if constexpr (T != kKvF16) {
#pragma unroll
        for (int s = 0; s < R::kS; ++s) r.ks[i][s] = ld_u16(row + KvRecord<T>::kBytes * min(4 * s + g, NB - 1));
      }
    }
#pragma unroll
    for (int i = 0; i < R::kV; ++i) {
      const int u = i * kWave + lane, key = min(u / R::kVUnit, kStep - 1), e = u % R::kVUnit;
      const int p = __shfl(page, key, kWave);
      const uint8_t* row = a.v.data + vh + (long long)max(p, 0) * a.v.page +
                           (long long)(p < 0 ? 0 : slot_of(pos + key)) * a.v.slot;
      if constexpr (T == kKvF16) {
        r.v[i] = *reinterpret_cast<const Bytes16*>(row + 16 * e);
      } else if constexpr (T == kKvQ8_0) {
        r.v[i] = *reinterpret_cast<const Bytes16*>(row + 34 * (e / 2) + 2 + 16 * (e & 1));
        r.vs[i] = ld_u16(row + 34 * (e / 2));
      } else {
        r.v[i] = *reinterpret_cast<const Bytes16*>(row + 18 * e + 2);
        r.vs[i] = ld_u16(row + 18 * e);
      }
    }
  };

  R raw;
  int step = step0 + wave;
  int page = pages_of(step), next_page = pages_of(step + kWaves);
  if (step < step1) load(step, page, raw);
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

    // V into LDS rows; a key that no row sees is zeros (its memory may hold anything)
    uint32_t spoiled = 0;  // keys some rows see whose values are not all finite
#pragma unroll
    for (int i = 0; i < R::kV; ++i) {
      const int u = i * kWave + lane, key = u / R::kVUnit, e = u % R::kVUnit;
      const bool live = R::kVUnit * kStep % kWave == 0 || key < kStep;
      bool zero = masked && !(present >> (key & 31) & 1u);
      if (masked) {
        bool bad;
        if constexpr (T == kKvF16) {
          bad = false;
#pragma unroll
          for (int w = 0; w < 4; ++w) bad = bad || half_not_finite(raw.v[i].w[w]) || half_not_finite(raw.v[i].w[w] >> 16);
        } else {
          bad = half_not_finite(raw.vs[i]);
        }
        bad = bad && !zero && live;
        if (__ballot(bad)) {  // hardly ever
          uint32_t mine = bad ? 1u << (key & 31) : 0u;
#pragma unroll
          for (int s = 32; s > 0; s >>= 1) mine |= (uint32_t)__shfl_xor((int)mine, s, kWave);
          spoiled |= mine;
        }
        zero = zero || bad;
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
    // K's steps, times the scale, as [block][key]; K as operands
    f16x8 kf[2][NB];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (T != kKvF16) {
#pragma unroll
        for (int s = 0; s < R::kS; ++s)
          if (4 * s + g < NB) ksteps[(4 * s + g) * kStep + 16 * i + c] = fp16_to_fp32(raw.ks[i][s]) * a.scale;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if constexpr (T == kKvF16) {
          kf[i][b] = __builtin_bit_cast(f16x8, make_uint4(raw.k[i][b][0], raw.k[i][b][1], raw.k[i][b][2], raw.k[i][b][3]));
        } else {
          f16x2 x[4];
          if constexpr (T == kKvQ8_0) {
            codes4<128>(raw.k[i][b][0] ^ 0x80808080u, x[0], x[1]);
            codes4<128>(raw.k[i][b][1] ^ 0x80808080u, x[2], x[3]);
          } else {
            codes4<8>(raw.k[i][b][0] & 0x0f0f0f0fu, x[0], x[1]);
            codes4<8>(raw.k[i][b][0] >> 4 & 0x0f0f0f0fu, x[2], x[3]);
          }
          kf[i][b] = f16x8{x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
        }
      }
    }
    wave_sync();
    // the next step's records are on their way while this one is worked on
    page = next_page;
    if (step + kWaves < step1) load(step + kWaves, page, raw);
    next_page = pages_of(step + 2 * kWaves);

    f32x4 s[RT][2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        f32x4 step4;
        if constexpr (T != kKvF16) step4 = *reinterpret_cast<const f32x4*>(ksteps + b * kStep + 16 * i + 4 * g);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          f32x4 x = {};
          if constexpr (T == kKvF16) x = s[rt][i];
          x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i][b], qh[rt][b], x, 0, 0, 0);
          if (!a.half_q) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[i][b], ql[rt][b], x, 0, 0, 0);
          if constexpr (T == kKvF16) {
            s[rt][i] = x;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[rt][i][e] = fmaf(x[e], step4[e], s[rt][i][e]);
          }
        }
      }

    f16x8 ph[RT], pl[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = s[rt][e / 4][e % 4];
        if constexpr (T == kKvF16) x[e] *= a.scale;
      }
      if (masked) {
        // value e: key 16 (e / 4) + 4 g + e % 4
        const uint32_t seen = (uint32_t)seen_bits(a, present, pos, qpos[rt]) >> (4 * g);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = seen & 1u << (16 * (e / 4) + e % 4) ? x[e] : -INFINITY;
      }
      float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
      top = quarters_max(top);
      if (__ballot(top > m[rt] + kLag)) {
        const float now = fmaxf(m[rt], top);
        const float f = now == -INFINITY ? 1.f : exp2_fast(m[rt] - now);
        m[rt] = now;
        l[rt] *= f;
#pragma unroll
        for (int v = 0; v < 2 * NB; ++v) o[rt][v] *= f;
      }
      const float base = m[rt] == -INFINITY ? 0.f : m[rt];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = exp2_fast(x[e] - base);
        l[rt] += p;
        ph[rt][e] = (_Float16)p;
        if constexpr (T != kKvF16) pl[rt][e] = (_Float16)(p - (float)ph[rt][e]);
      }
    }

    // O^T += V^T P^T
#pragma unroll
    for (int v = 0; v < 2 * NB; ++v) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* LdsPtr;
      // a quarter's lane i: key 4 g + i / 4, values 4 (i % 4) .. of the 16 columns
      uint8_t* at = vrow + (4 * g + c / 4) * L::kRow + 32 * v + 8 * (c & 3);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsPtr)(at + 16 * L::kRow));
      const f16x4 lo4 = __builtin_bit_cast(f16x4, lo), hi4 = __builtin_bit_cast(f16x4, hi);
      const f16x8 vf = {lo4[0], lo4[1], lo4[2], lo4[3], hi4[0], hi4[1], hi4[2], hi4[3]};
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        o[rt][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[rt], o[rt][v], 0, 0, 0);
        if constexpr (T != kKvF16) o[rt][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[rt], o[rt][v], 0, 0, 0);
      }
    }
    // values that are not finite reach the rows that see their key, and no other
    while (spoiled) {
      const int key = __ffs(spoiled) - 1;
      spoiled &= spoiled - 1;
      int pg, slot;
      if (!kv_place(a.seqs, seq, pos + key, pg, slot)) continue;
      const uint8_t* row = a.v.data + (long long)kvh * a.v.head + pg * a.v.page + slot * a.v.slot;
      const int at = 4 * (key / 16) + key % 4;  // among the lane's weights
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float p = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float w = (float)ph[rt][e];
          if constexpr (T != kKvF16) w += (float)pl[rt][e];
          p = e == at ? w : p;
        }
        p = __shfl(p, 16 * (key % 16 / 4) + c, kWave);
        if (seen_bits(a, 1ull, pos + key, qpos[rt])) {
#pragma unroll
          for (int v = 0; v < 2 * NB; ++v)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              o[rt][v][e] += p * value_of<T>(row, 16 * v + 4 * g + e);
              asm volatile("" ::: "memory");  // one value at a time: no registers for this path
            }
        }
      }
    }
    wave_sync();
  }

  // join the waves: sixteen rows at a time through LDS
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    __syncthreads();
    const float sum = quarters_sum(l[rt]);
    float* mine = reinterpret_cast<float*>(lds[wave]) + c * L::kORow;
#pragma unroll
    for (int v = 0; v < 2 * NB; ++v) *reinterpret_cast<f32x4*>(mine + 16 * v + 4 * g) = o[rt][v];
    if (g == 0) ml[wave][c][0] = m[rt], ml[wave][c][1] = sum;
    __syncthreads();
    const int row = threadIdx.x / 16;
    if (16 * rt + row >= t.rows) continue;
    float top = -INFINITY, w[kWaves], all = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, ml[i][row][0]);
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      w[i] = top == -INFINITY ? 0.f : exp2_fast(ml[i][row][0] - top);
      all += w[i] * ml[i][row][1];
    }
    const int r = t.row0 + 16 * rt + row;
    const float f = !whole ? 1.f : all == 0.f ? 0.f : 1.f / all;  // a row that sees nothing: zeros
    float* part = nullptr;
    if (!whole) {
      part = a.part + ((long long)blockIdx.x * a.splits + split) * (16 * RT) * (D + 2) + (16 * rt + row) * (D + 2);
      if (threadIdx.x % 16 == 0) part[D] = top, part[D + 1] = all;
    }
    uint8_t* dst = a.o + (long long)(t.token0 + r / a.share) * a.o_token +
                   (long long)(kvh * a.share + r % a.share) * a.o_head;
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
}

template <int T, int NB>
void launch(const AttendArgs& a, dim3 grid, hipStream_t st) {
  attend_few_kernel<T, NB, 1><<<grid, kWaves * kWave, 0, st>>>(a);
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

void attend_few(int type, int d, const AttendArgs& a, int items, hipStream_t st) {
  const dim3 grid((unsigned)items, (unsigned)a.splits);
  switch (type) {
    case kKvF16: launch_d<kKvF16>(d, a, grid, st); break;
    case kKvQ8_0: launch_d<kKvQ8_0>(d, a, grid, st); break;
    default: launch_d<kKvQ4_0>(d, a, grid, st); break;
  }
  check_launch("attend_few_kernel");
}

}  // namespace weft
