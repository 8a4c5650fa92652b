// What the attention kernels share: the call's arguments, which keys a tile of
// query rows can see, and how the key axis is split.
//
// The queries of one kv head of a sequence are rows r = token * share + head:
// they read the same keys and values, so a tile of rows may hold several heads
// of one token, several tokens, or both.  Keys go in steps of 32 or 64 at
// positions that are multiples of that: first those that hold visible sinks, then
// those of the rows' windows.
#pragma once

#include "kv_cache.h"

namespace weft {

struct AttendArgs {
  KvSeqs seqs;
  KvPool k, v;
  const uint8_t* q;
  uint8_t* o;
  float* part;  // the splits' partial results, nullptr where none are made
  long long q_head, q_token, o_head, o_token;  // byte strides
  int share, kv_heads, window, sinks;
  int first, items;  // this launch's first (tile, kv head) and all of the call's
  int tile;        // rows a tile
  int step_shift;  // log2 of the keys a step, 5 or 6
  int splits;      // the most splits of a tile's steps
  int least;       // the fewest steps a split is made for
  float scale;     // its magnitude times log2 e, > 0; the queries take its sign (0: they are zeros)
  float sign;
  bool half_q, half_o;
  // pages of a power of two >= 16 (32) slots, none longer than 2^31 bytes, so that
  // 16 (32) keys lie in one page and offsets in a page in 32 bits
  bool whole16, whole32;
  bool dense;  // and a page's slots follow each other, 16 rows beginning at multiples of 16 bytes
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
struct __attribute__((packed, aligned(2))) Bytes8 {
  uint32_t w[2];
};
struct __attribute__((packed, aligned(2))) Bytes16 {
  uint32_t w[4];
};

// a value that all lanes share, known to the compiler as one
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

struct Range {
  int sink_steps;   // steps at positions 0, step, ..
  int begin;        // position of the first step after them
  int steps;        // all steps
  int end;          // no visible key at or past it
};

// The steps that the queries at positions p0 .. p1 (p1 >= p0) can see keys in.
__device__ __forceinline__ Range visible_range(const AttendArgs& a, long long p0, long long p1) {
  Range r;
  const long long table = (long long)a.seqs.max_pages * a.seqs.page_size;
  r.end = (int)max(0ll, min(min(p1 + 1, table), (long long)INT32_MAX - 128));
  const long long first = a.window > 0 ? max(0ll, p0 - a.window + 1) : 0;
  r.begin = (int)min(first, (long long)r.end) & -(1 << a.step_shift);
  r.sink_steps = (min(a.sinks, r.begin) + (1 << a.step_shift) - 1) >> a.step_shift;
  r.steps = r.sink_steps + ((r.end - r.begin + (1 << a.step_shift) - 1) >> a.step_shift);
  return r;
}

template <int kStep>
__device__ __forceinline__ int step_position(const Range& r, int step) {
  return step < r.sink_steps ? step * kStep : r.begin + (step - r.sink_steps) * kStep;
}

// The keys of a step at `pos` that a query at `qpos` sees, key i as bit i;
// `present`: the keys that are there.
__device__ __forceinline__ unsigned long long first_bits(int n) {
  return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
}
__device__ __forceinline__ unsigned long long seen_bits(const AttendArgs& a, unsigned long long present, int pos,
                                                        int qpos) {
  present &= first_bits(qpos - pos + 1);
  if (a.window > 0) present &= ~first_bits(qpos - a.window - pos + 1) | first_bits(a.sinks - pos);
  return present;
}

// A tile of query rows: its sequence, rows and keys.
struct TileRows {
  int seq, row0, rows, token0;  // token0: the sequence's first new token
  long long pos0;               // and its position
  Range range;
  int each;    // steps a split takes
  int before;  // tiles of the sequences before
};

__device__ __forceinline__ int wave_scan(int v) {  // inclusive
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += dpp<kDppBcast15, 0xA>(v);
  return v + dpp<kDppBcast31, 0xC>(v);
}
__device__ __forceinline__ int wave_scan_max(int v) {  // inclusive, of values >= 0
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
  v = max(v, dpp<kDppBcast15, 0xA>(v));
  return max(v, dpp<kDppBcast31, 0xC>(v));
}
__device__ __forceinline__ int wave_max_count(int v) {  // of values >= 0
  v = max(v, dpp<kDppXor1>(v));
  v = max(v, dpp<kDppXor2>(v));
  v = max(v, dpp<kDppHalfMirror>(v));
  v = max(v, dpp<kDppMirror>(v));
  v = max(v, dpp<kDppBcast15, 0xA>(v));
  v = max(v, dpp<kDppBcast31, 0xC>(v));
  return __builtin_amdgcn_readlane(v, 63);
}

// Where a tile of the call lies: tile number `tile` in the sequences' order, or
// with `row` >= 0 the tile of that new token's row (token, head in its group).
// Also the steps a split takes: the longest sequence's over the most splits, the
// same for every tile, so that shorter sequences make fewer splits of the same work.
// (The most splits are the host's; a call with as many tiles as run at once has one, and
// lasts as long as its longest sequence.)  The whole wave calls it; 64 sequences are looked at at once, so a call's
// starts and lengths cost one trip to memory.  A start below one before it counts as
// that one, so no row is in two sequences and a call has no more tiles than the host
// planned for.
__device__ __forceinline__ bool locate(const AttendArgs& a, int tile, int token, int head, TileRows& t) {
  const int lane = threadIdx.x & (kWave - 1);
  int longest = 0, before = 0, found = -1, first = 0, n = 0, in = 0, reached = 0;
  long long len = 0;
  for (int i = 0; i < a.seqs.n_seqs; i += kWave) {
    int f = 0, end = 0, length = 0;
    if (i + lane < a.seqs.n_seqs) {
      f = max(0, min(a.seqs.starts[i + lane], a.seqs.n_tokens));
      end = max(0, min(a.seqs.starts[i + lane + 1], a.seqs.n_tokens));
      length = a.seqs.lengths[i + lane];
    }
    f = max(reached, wave_scan_max(f));
    end = max(f, end);  // past the last sequence: no rows
    reached = __builtin_amdgcn_readlane(end, kWave - 1);
    const int count = end - f;
    int steps = 0;
    if (count > 0) steps = visible_range(a, (long long)length - count, (long long)length - 1).steps;
    longest = max(longest, wave_max_count(steps));
    const int tiles = (int)(((unsigned)(count * a.share) + (unsigned)a.tile - 1) / (unsigned)a.tile);
    const int sum = wave_scan(tiles), all = __builtin_amdgcn_readlane(sum, kWave - 1);
    if (found < 0) {
      const unsigned long long hit = token < 0 ? __ballot(before + sum > tile)
                                               : __ballot(count > 0 && token >= f && token < f + count);
      if (hit) {
        const int at = __builtin_ctzll(hit);
        found = i + at;
        first = __builtin_amdgcn_readlane(f, at);
        n = __builtin_amdgcn_readlane(count, at);
        len = __builtin_amdgcn_readlane(length, at);
        before += __builtin_amdgcn_readlane(sum - tiles, at);
        in = tile - before;
      } else {
        before += all;
      }
    }
  }
  if (found < 0) return false;
  if (token >= 0) in = ((token - first) * a.share + head) / a.tile;
  t.seq = found;
  t.token0 = first;
  t.row0 = in * a.tile;
  t.rows = min(a.tile, n * a.share - t.row0);
  t.pos0 = len - n;
  t.before = before;
  t.each = max(a.least, (longest + a.splits - 1) / a.splits);
  if (in < 0 || t.rows <= 0) return false;
  t.range = visible_range(a, t.pos0 + t.row0 / a.share, t.pos0 + (t.row0 + t.rows - 1) / a.share);
  return true;
}

// ------------------------------------------------------ lanes and numbers
// largest / sum of a value over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float quarters_max(float x) {
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
  s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float quarters_sum(float x) {
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// A row's weights are powers of two of its scores over a reference that lies kUp below
// the largest score, so that the 16 bits they are rounded to reach far down: weights of
// 2^-26 of the largest keep 11 bits, those below 2^-37 are lost.  (With the largest score
// itself as the reference that was 2^-14 and 2^-25: beside a key that takes nearly all the
// weight and has small values, outputs whose weights were e^-15 of it were 0.3 to 1.4 %
// off.)  The reference moves when a score is kMost above it, 2^15 as a weight: three past
// kUp, so that sums are not rescaled at nearly every step.  From 2^22 on, where kUp is no
// longer exact beside a score, the reference is the score.
constexpr float kUp = 12.f, kMost = 15.f;
__device__ __forceinline__ float reference(float top) { return fabsf(top) < 0x1p22f ? top - kUp : top; }

// exp2 of an argument <= kMost (results below 2^-126 are zero)
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Four code bytes as 16-bit integers, exactly: byte u as 0x6400 | u is 1024 + u.
// kZero: the value of code 0 (128 for signed bytes with their sign bit turned).
template <int kZero>
__device__ __forceinline__ void codes4(uint32_t bytes, f16x2& lo, f16x2& hi) {
  const f16x2 zero = {(_Float16)(1024 + kZero), (_Float16)(1024 + kZero)};
  lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, bytes, 0x04010400u)) - zero;
  hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, bytes, 0x04030402u)) - zero;
}

// any value of a row of the cache, for paths that are rarely taken
template <int T>
__device__ __forceinline__ float value_of(const uint8_t* row, int i) {
  const uint8_t* rec = row + (i / 32) * KvRecord<T>::kBytes;
  const int e = i & 31;
  if constexpr (T == kKvF16) return fp16_to_fp32(ld_u16(rec + 2 * e));
  const float d = fp16_to_fp32(ld_u16(rec));
  if constexpr (T == kKvQ8_0) return d * (float)(int8_t)rec[2 + e];
  return d * (float)((int)(rec[2 + (e & 15)] >> (e & 16 ? 4 : 0) & 15) - 8);
}

__device__ __forceinline__ bool half_not_finite(uint32_t h) { return (h & 0x7c00u) == 0x7c00u; }

// Whether a record's values may be past 16 bits, by its step: infinite, NaN, or from
// 65536 / 128 (8 for 4-bit codes) on.  kv_write makes such records of finite values.
template <int T>
__device__ __forceinline__ bool past_half(uint32_t step) {
  return !(__builtin_fabsf16(__builtin_bit_cast(_Float16, (uint16_t)step)) < (_Float16)(T == kKvQ8_0 ? 512.f : 8192.f));
}

// the many-row kernel's keys a step
__host__ __device__ constexpr int many_step(int d) { return d > 192 ? 32 : 64; }

// launches of the kernels, of a.items or (a launch has fewer than 2^32 threads: past
// that the runtime starts the rest of the division, without an error) in parts
constexpr int kMostItems = 1 << 23;
void attend_few(int type, int d, AttendArgs a, hipStream_t st);   // tile 16, step 32
void attend_many(int type, int d, AttendArgs a, hipStream_t st);  // tile 128, step many_step

}  // namespace weft
