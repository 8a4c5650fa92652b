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
  int tile;        // rows a tile
  int step;        // keys a step, 32 or 64
  int splits;      // the most splits of a tile's steps
  int least;       // the fewest steps a split is made for
  float scale;     // its magnitude times log2 e, > 0; the queries take its sign (0: they are zeros)
  float sign;
  bool half_q, half_o;
  // pages of a power of two >= 16 (32) slots, none longer than 2^31 bytes, so that
  // 16 (32) keys lie in one page and offsets in a page in 32 bits
  bool whole16, whole32;
};

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

// a value that all lanes share, known to the compiler as such
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long long uniform(long long x) {
  return (long long)(((unsigned long long)(uint32_t)uniform((int)(x >> 32)) << 32) | (uint32_t)uniform((int)x));
}

// the new tokens of a sequence, whatever its starts hold
__device__ __forceinline__ int seq_tokens(const KvSeqs& s, int seq, int& first) {
  first = max(0, min(s.starts[seq], s.n_tokens));
  return max(0, max(0, min(s.starts[seq + 1], s.n_tokens)) - first);
}

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
  r.begin = (int)min(first, (long long)r.end) & -a.step;
  r.sink_steps = (min(a.sinks, r.begin) + a.step - 1) / a.step;
  r.steps = r.sink_steps + (r.end - r.begin + a.step - 1) / a.step;
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

// Steps a split takes, the same for every tile of the call, so that a batch of
// uneven sequences makes splits of even work: the longest sequence's steps over
// the most splits.  The whole wave calls it.
__device__ __forceinline__ int split_steps(const AttendArgs& a) {
  const int lane = threadIdx.x & (kWave - 1);
  int longest = 0;
  for (int i = 0; i < a.seqs.n_seqs; i += kWave) {
    int steps = 0;
    if (i + lane < a.seqs.n_seqs) {
      int first;
      const int n = seq_tokens(a.seqs, i + lane, first);
      const long long len = a.seqs.lengths[i + lane];
      if (n > 0) steps = visible_range(a, len - n, len - 1).steps;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) steps = max(steps, __shfl_xor(steps, o, kWave));
    longest = max(longest, steps);
  }
  return uniform(max(a.least, (longest + a.splits - 1) / a.splits));
}

// Tile t of the call's tiles in the sequences' order -> its sequence (-1: there
// is none) and its tile in it; tile_of the other way round: the tiles of the
// sequences before `seq`.  The whole wave calls both.
__device__ __forceinline__ int seq_tiles(const AttendArgs& a, int seq) {
  int first;
  return seq < a.seqs.n_seqs ? (seq_tokens(a.seqs, seq, first) * a.share + a.tile - 1) / a.tile : 0;
}

__device__ __forceinline__ int find_tile(const AttendArgs& a, int t, int& tile) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int i = 0; i < a.seqs.n_seqs; i += kWave) {
    const int n = seq_tiles(a, i + lane);
    int sum = n;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int up = __shfl_up(sum, o, kWave);
      if (lane >= o) sum += up;
    }
    const int all = __builtin_amdgcn_readlane(sum, kWave - 1);
    if (t < all) {
      const int at = __popcll(__ballot(sum <= t));
      tile = uniform(t - __shfl(sum - n, at, kWave));
      return uniform(i + at);
    }
    t -= all;
  }
  return -1;
}

__device__ __forceinline__ int tiles_before(const AttendArgs& a, int seq) {
  const int lane = threadIdx.x & (kWave - 1);
  int n = 0;
  for (int i = 0; i < seq; i += kWave) n += i + lane < seq ? seq_tiles(a, i + lane) : 0;
  return wave_sum(n);
}

// One tile's rows: its first, how many, their first token and its position.
struct TileRows {
  int seq, row0, rows, token0;
  long long pos0;  // of the sequence's first new token
  Range range;
};

__device__ __forceinline__ bool tile_rows(const AttendArgs& a, int seq, int tile, TileRows& t) {
  int first;
  const int n = uniform(seq_tokens(a.seqs, seq, first));
  t.seq = seq;
  t.token0 = uniform(first);
  t.row0 = tile * a.tile;
  t.rows = min(a.tile, n * a.share - t.row0);
  t.pos0 = (long long)uniform(a.seqs.lengths[seq]) - n;
  if (tile < 0 || t.rows <= 0) return false;
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

// A row's maximum moves only when a score is more than 2^kLag times its weight's
// scale: weights up to 2^kLag keep their 11 bits in 16, and the sums are not
// rescaled at nearly every step.
constexpr float kLag = 8.f;

// exp2 of an argument <= kLag (results below 2^-126 are zero)
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

// the many-row kernel's keys a step
__host__ __device__ constexpr int many_step(int d) { return d > 192 ? 32 : 64; }

// launches of the kernels
void attend_few(int type, int d, const AttendArgs& a, int items, hipStream_t st);   // tile 16, step 32
void attend_many(int type, int d, const AttendArgs& a, int items, hipStream_t st);  // tile 128, step many_step

}  // namespace weft
