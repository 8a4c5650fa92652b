// What a step answers with, from its rows of logits in one pass:
//   d_i = (x_i - max x) scale,  S = sum e^d_i
//   log p_i = d_i - log S                       of given tokens and of the largest logits
//   H = log S - (sum e^d_i d_i) / S             the entropy; its terms have one sign
//
// A row is cut into ranges when there are few rows, a workgroup each, and a second launch
// joins them.  A lane holds 32 values of a chunk in registers, so a wave knows its chunk's
// maximum before it takes the exponentials: one exponential a value, and sums that are
// rescaled only when the maximum grows.
//
// The largest logits: each wave keeps the 64 best of its values sorted, one a lane, as
// 64-bit keys of the value and the inverted index, so that of equal values the first wins.
// Only few values are looked at: in the first chunk, with w waves and n asked for, each wave takes the
// p-th largest of its lanes' maxima (p = ceil(n / w)) and all the ceil(n / p)-th largest of
// those, which n values at least reach.  Where the row's end leaves too few waves with values, a wave
// counts its own values instead of lanes (98770 logits, five alternatives: 31 us without a bound for the
// range that has the last 466, 12 with it).  Later ones have to beat the list's n-th.  What
// passes goes to LDS and from there into the wave's list by rank: a key's place is the number of larger
// ones.  The waves' lists, and in the join those of the ranges, meet by rank too.
//
// Long batches are bound by memory: 4096 rows of 50021 16-bit logits take 81 us (5.1 TB/s).  Few
// rows are bound by chains of latency: 48 x 131072 to 20 alternatives 11.7 us (2.1 TB/s) and
// 4.4 for the join, 1 x 32000 to five 8.8, where a list costs about 3.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "runtime.h"
#include "weft_common.h"
#include "weft_hip.h"

namespace weft {
namespace {

constexpr int kMost = WEFT_GGML_MOST_ALTERNATIVES;  // one a lane
constexpr int kHold = 32;                           // values a lane holds of a chunk
constexpr int kThreads = 256, kMostThreads = 1024;  // of the join, and of a range at most
static_assert(kMost == kWave, "a list is one key a lane");

typedef unsigned long long Key;

struct LogProbsArgs {
  const uint8_t* x;
  const int32_t* tokens;
  float* token_lp;
  float* entropy;
  int32_t* top_ids;
  float* top_lp;
  long long x_row, tokens_row, token_lp_row, entropy_row, top_ids_row, top_lp_row;  // x in bytes, others in elements
  uint8_t* work;
  long long row0;
  float half, scale;  // d = (half x - half max) scale: differences past the largest number come with small scales
  int v, given, top;
  int splits, chunks, chunks_each;
};

struct Stats {
  float m, s, t;  // maximum, sum of e^d, sum of e^d d
};
// half x - half m: rounded once, and finite for halves
__device__ __forceinline__ float below(const LogProbsArgs& a, float x, float m) { return fmaf(x, a.half, -(m * a.half)); }

// below 2^-126 zero: the largest term is 1
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }

// Two parts' sums over their common maximum.  A part of nothing has the lowest maximum and
// sums of zero; the bound on d keeps 0 x infinity out of t.
__device__ __forceinline__ Stats join(const LogProbsArgs& args, Stats a, Stats b) {
  const float m = fmaxf(a.m, b.m);
  const float da = fmaxf(below(args, a.m, m) * args.scale, -1e4f), db = fmaxf(below(args, b.m, m) * args.scale, -1e4f);
  const float ea = exp_of(da), eb = exp_of(db);
  return {m, a.s * ea + b.s * eb, (a.t + da * a.s) * ea + (b.t + db * b.s) * eb};
}
__device__ __forceinline__ Stats join_wave(const LogProbsArgs& args, Stats a) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1)
    a = join(args, a, {__shfl_xor(a.m, o, kWave), __shfl_xor(a.s, o, kWave), __shfl_xor(a.t, o, kWave)});
  return a;
}

// floats in the order of their values, -0 as 0
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ Key key_of(float x, int i) { return (Key)ordered(x) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float value_of(Key k) { return from_ordered((uint32_t)(k >> 32)); }
__device__ __forceinline__ int index_of(Key k) { return (int)~(uint32_t)k; }

__device__ __forceinline__ Key lane_key(Key k, int lane) {
  return (Key)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, lane);
}

// The 64 largest keys of what a wave has seen (0: none), sorted, one a lane, and keys on their
// way there: `pending`, in LDS.
struct Best {
  Key* pending;
  int n_pending;
  Key list;
  bool sorted;  // keys have gone into the list
  __device__ __forceinline__ explicit Best(Key* at) : pending(at), n_pending(0), list(0), sorted(false) {}

  // the lanes' keys that are `in`, behind those on their way
  __device__ __forceinline__ void add(bool in, Key k, int lane) {
    const unsigned long long who = __ballot(in);
    if (in) pending[n_pending + __popcll(who & ((1ull << lane) - 1))] = k;
    n_pending += __popcll(who);
  }
  // the last n (at most 64) keys on their way into the list
  __device__ __forceinline__ void take(int n, int lane) {
    n_pending -= n;
    Key* p = pending + n_pending;
    __builtin_amdgcn_wave_barrier();  // the wave's own writes
    const Key mine = lane < n ? p[lane] : 0;
    __builtin_amdgcn_wave_barrier();
    int down = lane, rank = 0;  // where this lane's list entry, and its new key, go
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const Key k = lane_key(mine, j);
      const unsigned long long above = __ballot(list > k);
      down += k > list ? 1 : 0;
      rank += k > mine ? 1 : 0;
      if (lane == j) rank += __popcll(above);
    }
    // 64 entries and n keys have places 0 to 63 + n
    if (down < kWave) p[down] = list;
    if (lane < n && rank < kWave) p[rank] = mine;
    __builtin_amdgcn_wave_barrier();
    list = p[lane];
    __builtin_amdgcn_wave_barrier();
    sorted = true;
  }
  // a key a lane, in any order, among them the `top` largest
  __device__ __forceinline__ Key rest(int lane, int top) {
    if (sorted && n_pending > 0) take(n_pending, lane);
    if (sorted) return lane < top ? list : 0;
    __builtin_amdgcn_wave_barrier();
    return lane < n_pending ? pending[lane] : 0;
  }
};

// What a wave leaves for the others, beside its list.
struct Left {
  Stats st;
  float bound;  // of the first chunk
  int count;    // of keys
  int unused[3];
};
static_assert(sizeof(Left) == 32, "keys behind it are aligned");

// The keys of a workgroup (one a lane at most, 0: none) go to `all` (64 a wave), one after the other, and a
// thread gets one of them back with its place among them: the first waves, so that most rank none.
// n: how many there are; no thread past it has a place.
struct Placed {
  Key k;
  int place, n;
};
__device__ __forceinline__ Placed place_of(Key* all, Left* left, Key k, int lane, int wave, int waves) {
  const bool in = k != 0;
  const unsigned long long who = __ballot(in);
  if (lane == 0) left[wave].count = __popcll(who);
  __syncthreads();
  int at = __popcll(who & ((1ull << lane) - 1)), n = 0;
  for (int w = 0; w < waves; ++w) {
    at += w < wave ? left[w].count : 0;
    n += left[w].count;
  }
  if (in) all[at] = k;
  __syncthreads();
  const int tid = wave * kWave + lane;
  Placed p = {0, 0, n};
  if (tid >= n) return p;
  p.k = all[tid];
#pragma unroll 8
  for (int i = 0; i < n; ++i) p.place += all[i] > p.k ? 1 : 0;
  return p;
}

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
template <bool kHalf>
__device__ __forceinline__ float logit(const uint8_t* row, int i) {
  if constexpr (kHalf)
    return (float)reinterpret_cast<const _Float16*>(row)[i];
  else
    return reinterpret_cast<const float*>(row)[i];
}

// Values i .. of a row, 16-byte aligned there; a wave's lanes lie one after the other from `first` on
// (its lane 0's i).  Minus infinity before the row's begin (i modulo 2^32) and past its end.  The branches
// are the wave's and nothing is converted here, so that its loads do not wait for each other (each
// waited for the one before: 1024 rows of 131072 with 20 alternatives 127 us, now 104).
template <bool kHalf>
using Loaded = std::conditional_t<kHalf, half8, float4v>;
template <bool kHalf>
__device__ __forceinline__ Loaded<kHalf> load(const uint8_t* row, uint32_t i, uint32_t first, uint32_t v) {
  using T = std::conditional_t<kHalf, _Float16, float>;
  constexpr int N = 16 / sizeof(T);
  const T* p = reinterpret_cast<const T*>(row);
  Loaded<kHalf> x;
  if (first < v && v - first >= N * kWave) {
    x = *reinterpret_cast<const Loaded<kHalf>*>(p + i);
  } else if (first < v || (int32_t)first < 0) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool in = i + e < v;
      const T q = p[in ? i + e : 0];
      x[e] = in ? q : (T)-INFINITY;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = (T)-INFINITY;
  }
  return x;
}

struct Row {
  Stats st;
  float log_s;
  bool none;  // every logit is minus infinity
};
__device__ __forceinline__ Row row_of(const Stats& st) { return {st, logf(st.s), st.s == 0.f}; }

// and an alternative at its place; a key of zero: fewer numbers than alternatives
__device__ __forceinline__ void answer_top(const LogProbsArgs& a, long long row, const Row& r, Key k, int place) {
  a.top_ids[row * a.top_ids_row + place] = k ? index_of(k) : -1;
  a.top_lp[row * a.top_lp_row + place] =
      k ? (r.none ? -INFINITY : below(a, value_of(k), r.st.m) * a.scale - r.log_s) : r.st.s + NAN;
}

__device__ __forceinline__ Stats* work_stats(const LogProbsArgs& a, long long row) {
  return reinterpret_cast<Stats*>(a.work + row * a.splits * (16 + 8ll * a.top) + 8ll * a.splits * a.top);
}
__device__ __forceinline__ Key* work_keys(const LogProbsArgs& a, long long row) {
  return reinterpret_cast<Key*>(a.work + row * a.splits * (16 + 8ll * a.top));
}

// The keys on their way of a wave: those of four values a lane, fewer than 64 before them,
// and room for the list's 64 beside the last 64.
constexpr int kGroup = 4, kPending = kWave * (kGroup + 2);

// The largest number, in steps of 16 bits of the ordered value, that `n` lanes' values reach.
__device__ __forceinline__ float reached_by(float x, int n) {
  const uint32_t o = ordered(x);
  uint32_t bound = 0;
  for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
    if (__popcll(__ballot(o >= (bound | bit))) >= n) bound |= bit;
  return bound > ordered(-INFINITY) ? from_ordered(bound) : -INFINITY;
}

// The same of all values of the wave's first loads (of N values a lane): near the n-th largest.
template <int N>
__device__ __forceinline__ float reached_by_values(const float (&x)[kHold], int loads, int n) {
  uint32_t bound = 0;
  for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1) {
    const float b = from_ordered(bound | bit);  // no number past the infinities: nothing reaches it
    int count = 0;
#pragma unroll
    for (int j = 0; j < kHold / N; ++j) {
      if (j >= loads) continue;
#pragma unroll
      for (int e = 0; e < N; ++e) count += __popcll(__ballot(x[j * N + e] >= b));
    }
    if (count >= n) bound |= bit;
    if (count == n) break;
  }
  return bound > ordered(-INFINITY) ? from_ordered(bound) : -INFINITY;
}

// The given token of this thread (the first of them: others are read at the end), on its way before
// the rest, and its logit, asked for when the rest is on its way.
template <bool kHalf>
struct Given {
  int id;
  float x;
  __device__ __forceinline__ Given(const LogProbsArgs& a, long long row, bool wanted) : id(-1), x(0.f) {
    if (wanted && (int)threadIdx.x < a.given) id = a.tokens[row * a.tokens_row + threadIdx.x];
  }
  __device__ __forceinline__ void fetch(const LogProbsArgs& a, long long row) {
    if ((uint32_t)id < (uint32_t)a.v) x = logit<kHalf>(a.x + row * a.x_row, id);
  }
};

// A row's answers, by the threads of a workgroup
template <bool kHalf>
__device__ __forceinline__ void answer(const LogProbsArgs& a, long long row, const Row& r, const Given<kHalf>& first) {
  for (int i = threadIdx.x; i < a.given; i += blockDim.x) {
    Given<kHalf> g = first;
    if (i != (int)threadIdx.x) {
      g.id = a.tokens[row * a.tokens_row + i];
      g.fetch(a, row);
    }
    if ((uint32_t)g.id >= (uint32_t)a.v) continue;
    a.token_lp[row * a.token_lp_row + i] = r.none ? -INFINITY : below(a, g.x, r.st.m) * a.scale - r.log_s;
  }
  if (a.entropy != nullptr && threadIdx.x == 0) a.entropy[row * a.entropy_row] = r.none ? 0.f : r.log_s - r.st.t / r.st.s;
}

template <bool kHalf, bool kTop>
__global__ void __launch_bounds__(kMostThreads) log_probs_kernel(LogProbsArgs a) {
  constexpr int N = kHalf ? 8 : 4;  // values a load
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, threads = blockDim.x, waves = threads / kWave;
  Left* left = reinterpret_cast<Left*>(lds);
  Key* all = reinterpret_cast<Key*>(left + waves);
  Key* pending = all + waves * kWave;  // kPending a wave
  const long long row = a.row0 + (long long)(blockIdx.x / (unsigned)a.splits);
  const int split = (int)(blockIdx.x % (unsigned)a.splits);
  const uint8_t* x_row = a.x + row * a.x_row;
  const int c0 = split * a.chunks_each, c1 = min(a.chunks, c0 + a.chunks_each);
  // loads are 16-byte aligned: the first begins before a row that is not
  const int before = (int)(reinterpret_cast<uintptr_t>(x_row) & 15) / (kHalf ? 2 : 4);
  Given<kHalf> given(a, row, a.splits == 1);
  const float log2_scale = fminf(a.scale * 1.44269504088896341f, 3.402823466e38f);  // 0 x infinity is no number

  Stats st = {-3.402823466e38f, 0.f, 0.f};
  Best best(pending + wave * kPending);
  float limit = -INFINITY;  // what a candidate has at least
  auto raise = [&] {
    const Key last = lane_key(best.list, a.top - 1);
    // indexes that follow are larger: an equal value does not enter, and nothing beside infinities
    if (last) limit = value_of(last) == INFINITY ? NAN : fmaxf(limit, nextafterf(value_of(last), INFINITY));
  };

  for (int c = c0; c < c1; ++c) {
    const uint32_t first = __builtin_amdgcn_readfirstlane((uint32_t)c * threads * kHold + N * kWave * wave - before);
    const uint32_t at = first + N * lane;
    Loaded<kHalf> q[kHold / N];
#pragma unroll
    for (int j = 0; j < kHold / N; ++j)
      q[j] = load<kHalf>(x_row, at + (uint32_t)(j * N * threads), first + (uint32_t)(j * N * threads), (uint32_t)a.v);
    if (c == c0) given.fetch(a, row);
    float x[kHold];
#pragma unroll
    for (int i = 0; i < kHold; ++i) x[i] = (float)q[i / N][i % N];
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kHold; ++i) most = fmaxf(most, x[i]);
    if (kTop && c == c0) {
      const int p = (a.top + waves - 1) / waves;
      const float bound = reached_by(most, p);
      if (lane == 0) left[wave].bound = bound;
    }
    const float m = fmaxf(st.m, wave_max(most));
    const float d0 = fmaxf(below(a, st.m, m) * a.scale, -1e4f), e0 = exp_of(d0);
    st = {m, st.s * e0, (st.t + d0 * st.s) * e0};
    const float m_half = m * a.half;
    float t = 0.f;  // sum of e^d d / ln 2, which no scale takes past the largest number
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const float d2 = fmaf(x[i], a.half, -m_half) * log2_scale, e = __builtin_amdgcn_exp2f(d2);
      st.s += e;
      t = fmaf(e, fmaxf(d2, -3.402823466e38f), t);  // minus infinity counts nothing; NaN stays in e
    }
    st.t = fmaf(t, 0.693147180559945309f, st.t);
    if constexpr (kTop) {
      if (c == c0) {
        __syncthreads();  // all waves have a first chunk
        const int p = (a.top + waves - 1) / waves;
        limit = reached_by(lane < waves ? left[lane].bound : -INFINITY, (a.top + p - 1) / p);
        // the row's end may leave too few waves with values
        if (waves > 1 && limit == -INFINITY) {
          int loads = 0;
#pragma unroll
          for (int j = 0; j < kHold / N; ++j) loads = (int)(first + (uint32_t)(j * N * threads)) < a.v ? j + 1 : loads;
          limit = reached_by_values<N>(x, loads, a.top);
        }
      }
      bool taken = false;
#pragma unroll
      for (int j = 0; j < kHold / kGroup; ++j) {
        // indexes grow from load to load, not within one
        if (taken && j % (N / kGroup) == 0) {
          raise();
          taken = false;
        }
        // value e of the group is e + kGroup (j % (N / kGroup)) of load j / (N / kGroup)
        const uint32_t i0 = at + (uint32_t)(j / (N / kGroup) * N * threads + kGroup * (j % (N / kGroup)));
        const float* g = x + j * kGroup;
        if (__ballot(fmaxf(fmaxf(g[0], g[1]), fmaxf(g[2], g[3])) >= limit) == 0) continue;
#pragma unroll
        for (int e = 0; e < kGroup; ++e) best.add(g[e] >= limit && i0 + e < (uint32_t)a.v, key_of(g[e], (int)(i0 + e)), lane);
        const bool full = best.n_pending >= kWave;
        while (best.n_pending >= kWave) best.take(kWave, lane);
        taken |= full;
      }
      if (taken) raise();
    }
  }
  const Key mine = kTop ? best.rest(lane, a.top) : 0;

  st.s = wave_sum_f(st.s);
  st.t = wave_sum_f(st.t);
  if (lane == 0) left[wave].st = st;
  Placed key = {0, 0, 0};
  if constexpr (kTop)
    key = place_of(all, left, mine, lane, wave, waves);
  else
    __syncthreads();
  st = left[0].st;
  for (int w = 1; w < waves; ++w) st = join(a, st, left[w].st);
  // places past the numbers have none
  const int place = !kTop ? a.top : tid < key.n ? key.place : tid;
  if (a.splits == 1) {
    const Row r = row_of(st);
    answer<kHalf>(a, row, r, given);
    if (place < a.top) answer_top(a, row, r, key.k, place);
    return;
  }
  if (tid == 0) work_stats(a, row - a.row0)[split] = st;
  if (place < a.top) work_keys(a, row - a.row0)[(long long)split * a.top + place] = key.k;
}

// The ranges' sums and lists, a list a lane for the bound: p-th entries as above.
template <bool kHalf>
__global__ void __launch_bounds__(kThreads) log_probs_join_kernel(LogProbsArgs a) {
  constexpr int kWaves = kThreads / kWave;
  __shared__ Key pending[kWaves][kPending];
  __shared__ Key all[kThreads];
  __shared__ Left left[kWaves];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const long long row = blockIdx.x;
  const Stats* parts = work_stats(a, row);
  const Key* keys = work_keys(a, row);
  Given<kHalf> given(a, a.row0 + row, true);
  Stats st = {-3.402823466e38f, 0.f, 0.f};
  if (lane < a.splits) st = parts[lane];
  Best best(pending[wave]);
  if (a.top == 0) {
    given.fetch(a, a.row0 + row);
  } else {
    const int p = (a.top + a.splits - 2) / (a.splits - 1);  // the last range may be short: without it
    const Key entry = lane < a.splits ? keys[(long long)lane * a.top + p - 1] : 0;
    given.fetch(a, a.row0 + row);
    const float limit = reached_by(entry ? value_of(entry) : -INFINITY, (a.top + p - 1) / p);
    const int n = a.splits * a.top;
    for (int i = wave * kWave; i < n; i += kThreads) {
      const Key k = i + lane < n ? keys[i + lane] : 0;
      if (best.n_pending >= kWave) best.take(kWave, lane);
      best.add(k != 0 && value_of(k) >= limit, k, lane);
    }
    // at most 64 are left
    if (best.n_pending > kWave) best.take(kWave, lane);
  }
  st = join_wave(a, st);
  const Row r = row_of(st);
  answer<kHalf>(a, a.row0 + row, r, given);
  if (a.top == 0) return;
  const Placed key = place_of(all, left, best.rest(lane, a.top), lane, wave, kWaves);
  const int place = (int)threadIdx.x < key.n ? key.place : (int)threadIdx.x;
  if (place < a.top) answer_top(a, a.row0 + row, r, key.k, place);
}

// How a call is cut (us): workgroups of one wave for short rows, but for many alternatives, for which its
// lanes' maxima are a poor bound (300 rows of 2048 to 64: 20.8, of four waves 8.2; 3000 of 2000 to 20 11.3 and 20.5), of 16 for few rows that fit one chunk
// (256 rows of 32000: 13.2, in ranges of four waves 15.8), else of four in ranges until there are 1024
// of them (48 rows of 131072: 17.0, of 16 waves 18.0; one row 12.8 and 15.1); 64 ranges a row at
// most, a list a lane of the join.  A row that begins `late` values behind an aligned place may have a chunk more
// and is cut as that many are: with the aligned row's ranges, of two chunks each, half of them would be
// empty.  The work buffer's size is for either, of the shape alone.
struct Plan {
  int threads, chunks, splits;
  size_t row_bytes;  // of the work buffer
  int64_t rows;      // a launch
};
int64_t chunks_of(int64_t v, int threads) { return (v + (int64_t)threads * kHold - 1) / (threads * kHold); }
Plan plan_of(int64_t v, int64_t rows, int64_t top, int64_t late) {
  Plan p{};
  v += late;
  p.threads = v <= kWave * kHold && top <= 32 ? kWave : v <= kMostThreads * kHold && v > kThreads * kHold && rows <= 512 ? kMostThreads : kThreads;
  const int64_t chunks = chunks_of(v, p.threads);
  p.chunks = (int)chunks;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>({1024 / std::max<int64_t>(rows, 1), chunks, kWave}));
  const int64_t each = (chunks + want - 1) / want;
  p.splits = (int)((chunks + each - 1) / each);
  p.row_bytes = p.splits > 1 ? (size_t)p.splits * (16 + 8 * (size_t)top) : 0;
  // a launch has fewer than 2^32 threads
  p.rows = std::max<int64_t>(1, ((int64_t)1 << 31) / kMostThreads / p.splits);
  return p;
}
// values that a row begins behind an aligned place, at most
int64_t most_late(const weft_ggml_tensor* x) { return x->type == WEFT_GGML_TYPE_F16 ? 7 : 3; }
size_t work_size(const weft_ggml_tensor* x, int64_t top) {
  const int64_t v = x->ne[0], rows = x->ne[1];
  return (size_t)rows * std::max(plan_of(v, rows, top, 0).row_bytes, plan_of(v, rows, top, most_late(x)).row_bytes);
}

hipError_t fail(hipError_t e) {
  set_error(e);
  return e;
}

bool logits_ok(const weft_ggml_tensor* x) {
  const size_t unit = x->type == WEFT_GGML_TYPE_F16 ? 2 : 4;
  return x->ne[0] > 0 && x->ne[0] <= INT32_MAX && x->ne[1] >= 0 && x->ne[1] <= INT32_MAX && x->ne[2] == 1 && x->ne[3] == 1 &&
         x->nb[0] == unit && x->nb[1] % unit == 0 && x->nb[1] < ((size_t)1 << 40) && aligned(x->data, unit);
}
// a matrix of n 4-byte elements and that many rows
bool matrix(const weft_ggml_tensor* t, int64_t n, int64_t rows) {
  return t->ne[0] == n && t->ne[1] == rows && t->ne[2] == 1 && t->ne[3] == 1 && t->nb[0] == 4 && t->nb[1] % 4 == 0 &&
         t->nb[1] < ((size_t)1 << 40) && aligned(t->data, 4) && (t->data != nullptr || n == 0 || rows == 0);
}

hipError_t log_probs(const weft_ggml_tensor* x, const weft_ggml_tensor* tokens, const weft_ggml_tensor* token_lp,
                     const weft_ggml_tensor* entropy, const weft_ggml_tensor* top_ids, const weft_ggml_tensor* top_lp,
                     float scale, void* wdata, size_t wsize) {
  if (x == nullptr || (tokens == nullptr) != (token_lp == nullptr) || (top_ids == nullptr) != (top_lp == nullptr))
    return fail(hipErrorInvalidValue);
  if (x->type != WEFT_GGML_TYPE_F32 && x->type != WEFT_GGML_TYPE_F16) return fail(hipErrorNotSupported);
  for (const weft_ggml_tensor* t : {token_lp, entropy, top_lp})
    if (t != nullptr && t->type != WEFT_GGML_TYPE_F32) return fail(hipErrorNotSupported);
  for (const weft_ggml_tensor* t : {tokens, top_ids})
    if (t != nullptr && t->type != WEFT_GGML_TYPE_I32) return fail(hipErrorNotSupported);
  if (!logits_ok(x) || !(scale > 0.f) || !std::isfinite(scale)) return fail(hipErrorInvalidValue);
  const int64_t v = x->ne[0], rows = x->ne[1];
  const int64_t given = tokens != nullptr ? tokens->ne[0] : 0, top = top_ids != nullptr ? top_ids->ne[0] : 0;
  if (given < 0 || given > INT32_MAX || top < 0 || top > kMost || top > v) return fail(hipErrorInvalidValue);
  if ((tokens != nullptr && (!matrix(tokens, given, rows) || !matrix(token_lp, given, rows))) ||
      (top_ids != nullptr && (!matrix(top_ids, top, rows) || !matrix(top_lp, top, rows))) ||
      (entropy != nullptr && !matrix(entropy, rows, 1)))
    return fail(hipErrorInvalidValue);
  if (rows == 0 || (given == 0 && top == 0 && entropy == nullptr)) return hipSuccess;
  if (x->data == nullptr) return fail(hipErrorInvalidValue);
  const size_t size = work_size(x, top);
  if (wsize < size || (size > 0 && (wdata == nullptr || !aligned(wdata, 16)))) return fail(hipErrorInvalidValue);
  const bool even = aligned(x->data, 16) && (rows == 1 || x->nb[1] % 16 == 0);
  const Plan p = plan_of(v, rows, top, even ? 0 : most_late(x));

  LogProbsArgs a{};
  a.x = static_cast<const uint8_t*>(x->data);
  a.x_row = (long long)x->nb[1];
  if (given > 0) {
    a.tokens = static_cast<const int32_t*>(tokens->data), a.tokens_row = (long long)(tokens->nb[1] / 4);
    a.token_lp = static_cast<float*>(token_lp->data), a.token_lp_row = (long long)(token_lp->nb[1] / 4);
  }
  if (entropy != nullptr) a.entropy = static_cast<float*>(entropy->data), a.entropy_row = 1;
  if (top > 0) {
    a.top_ids = static_cast<int32_t*>(top_ids->data), a.top_ids_row = (long long)(top_ids->nb[1] / 4);
    a.top_lp = static_cast<float*>(top_lp->data), a.top_lp_row = (long long)(top_lp->nb[1] / 4);
  }
  a.half = scale < 1.f ? 0.5f : 1.f;
  a.scale = scale / a.half;
  a.v = (int)v;
  a.given = (int)given;
  a.top = (int)top;
  a.splits = p.splits;
  a.chunks = p.chunks;
  a.chunks_each = (a.chunks + p.splits - 1) / p.splits;
  const hipStream_t st = current_stream();
  const bool half = x->type == WEFT_GGML_TYPE_F16;
  for (int64_t r = 0; r < rows; r += p.rows) {
    const unsigned n = (unsigned)std::min(rows - r, p.rows);
    a.row0 = r;
    a.work = static_cast<uint8_t*>(wdata) + (p.row_bytes > 0 ? p.row_bytes * (size_t)r : 0);
    const dim3 grid(n * (unsigned)p.splits);
    const size_t waves = (size_t)(p.threads / kWave);
    const size_t lds = waves * (sizeof(Left) + (top > 0 ? (kWave + kPending) * sizeof(Key) : 0));
    if (half && top > 0)
      log_probs_kernel<true, true><<<grid, p.threads, lds, st>>>(a);
    else if (half)
      log_probs_kernel<true, false><<<grid, p.threads, lds, st>>>(a);
    else if (top > 0)
      log_probs_kernel<false, true><<<grid, p.threads, lds, st>>>(a);
    else
      log_probs_kernel<false, false><<<grid, p.threads, lds, st>>>(a);
    check_launch("log_probs_kernel");
    if (p.splits == 1) continue;
    if (half)
      log_probs_join_kernel<true><<<dim3(n), kThreads, 0, st>>>(a);
    else
      log_probs_join_kernel<false><<<dim3(n), kThreads, 0, st>>>(a);
    check_launch("log_probs_join_kernel");
  }
  return pending_error();
}

}  // namespace
}  // namespace weft

extern "C" size_t weft_ggml_log_probs_work_size(const weft_ggml_tensor* logits, int64_t n_top) {
  if (logits == nullptr || logits->ne[0] <= 0 || logits->ne[0] > INT32_MAX || logits->ne[1] <= 0 ||
      logits->ne[1] > INT32_MAX || n_top < 0 || n_top > weft::kMost)
    return 0;
  return weft::work_size(logits, n_top);
}

extern "C" int weft_ggml_log_probs(const weft_ggml_tensor* logits, const weft_ggml_tensor* tokens,
                                   const weft_ggml_tensor* token_lp, const weft_ggml_tensor* entropy,
                                   const weft_ggml_tensor* top_ids, const weft_ggml_tensor* top_lp, float scale,
                                   void* wdata, size_t wsize) {
  return (int)weft::log_probs(logits, tokens, token_lp, entropy, top_ids, top_lp, scale, wdata, wsize);
}
