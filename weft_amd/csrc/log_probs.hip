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
// In its first chunk the n-th largest of the lanes' own maxima bounds the n-th largest value
// from below (n lanes have a value that large); later chunks are compared with the list's
// n-th.  What passes goes to LDS and is sorted into the list 64 at a time.
#include <algorithm>
#include <cmath>

#include "runtime.h"
#include "weft_common.h"
#include "weft_hip.h"

namespace weft {
namespace {

constexpr int kMost = WEFT_GGML_MOST_ALTERNATIVES;  // one a lane
constexpr int kHold = 32;                           // values a lane holds of a chunk
constexpr int kThreads = 256;
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
  float scale;
  int v, given, top;
  int splits, chunks, chunks_each;
};

struct Stats {
  float m, s, t;  // maximum, sum of e^d, sum of e^d d
};

// below 2^-126 zero: the largest term is 1
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }

// Two parts' sums over their common maximum.  A part of nothing has the lowest maximum and
// sums of zero; the bound on d keeps 0 x infinity out of t.
__device__ __forceinline__ Stats join(Stats a, Stats b, float scale) {
  const float m = fmaxf(a.m, b.m);
  const float da = fmaxf((a.m - m) * scale, -1e4f), db = fmaxf((b.m - m) * scale, -1e4f);
  const float ea = exp_of(da), eb = exp_of(db);
  return {m, a.s * ea + b.s * eb, (a.t + da * a.s) * ea + (b.t + db * b.s) * eb};
}
__device__ __forceinline__ Stats join_wave(Stats a, float scale) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1)
    a = join(a, {__shfl_xor(a.m, o, kWave), __shfl_xor(a.s, o, kWave), __shfl_xor(a.t, o, kWave)}, scale);
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

// one step of a bitonic network: the larger of lanes l and l ^ o to the lower lane if `down`
__device__ __forceinline__ Key exchange(Key k, int o, bool down, int lane) {
  const Key other = __shfl_xor(k, o, kWave);
  const bool larger = ((lane & o) == 0) == down;
  return (k > other) == larger ? k : other;
}
// 64 keys, the largest in lane 0
__device__ __forceinline__ Key sort64(Key k, int lane) {
#pragma unroll
  for (int n = 2; n <= kWave; n <<= 1)
#pragma unroll
    for (int o = n / 2; o > 0; o >>= 1) k = exchange(k, o, (lane & n) == 0, lane);
  return k;
}
// the 64 largest of two sorted lists, sorted
__device__ __forceinline__ Key merge64(Key a, Key b, int lane) {
  const Key r = __shfl(b, kWave - 1 - lane, kWave);
  Key k = a > r ? a : r;
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) k = exchange(k, o, true, lane);
  return k;
}

struct __attribute__((packed, aligned(4))) Floats4 {
  float f[4];
};
struct __attribute__((packed, aligned(2))) Halves8 {
  _Float16 h[8];
};
// values i .. of a row, minus infinity past its end
template <bool kHalf, int N>
__device__ __forceinline__ void load(const uint8_t* row, long long i, int v, float* x) {
  if (i + N <= v) {
    if constexpr (kHalf) {
      const Halves8 q = *reinterpret_cast<const Halves8*>(row + 2 * i);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = (float)q.h[e];
    } else {
      const Floats4 q = *reinterpret_cast<const Floats4*>(row + 4 * i);
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] = q.f[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (i + e >= v)
        x[e] = -INFINITY;
      else if constexpr (kHalf)
        x[e] = (float)reinterpret_cast<const _Float16*>(row)[i + e];
      else
        x[e] = reinterpret_cast<const float*>(row)[i + e];
    }
  }
}

template <bool kHalf>
__device__ __forceinline__ float logit(const uint8_t* row, int i) {
  if constexpr (kHalf)
    return (float)reinterpret_cast<const _Float16*>(row)[i];
  else
    return reinterpret_cast<const float*>(row)[i];
}

// A row's answers, by one wave with the row's sums and list.
template <bool kHalf>
__device__ __forceinline__ void answer(const LogProbsArgs& a, long long row, const Stats& st, Key list, int lane) {
  const uint8_t* x = a.x + row * a.x_row;
  const bool none = st.s == 0.f;  // every logit is minus infinity
  const float log_s = logf(st.s);
  for (int i = lane; i < a.given; i += kWave) {
    const int id = a.tokens[row * a.tokens_row + i];
    if ((uint32_t)id >= (uint32_t)a.v) continue;
    a.token_lp[row * a.token_lp_row + i] = none ? -INFINITY : (logit<kHalf>(x, id) - st.m) * a.scale - log_s;
  }
  if (a.entropy != nullptr && lane == 0) a.entropy[row * a.entropy_row] = none ? 0.f : log_s - st.t / st.s;
  if (lane < a.top) {
    // a key of zero: fewer numbers than alternatives
    a.top_ids[row * a.top_ids_row + lane] = list ? index_of(list) : -1;
    a.top_lp[row * a.top_lp_row + lane] =
        list ? (none ? -INFINITY : (value_of(list) - st.m) * a.scale - log_s) : st.s + NAN;
  }
}

__device__ __forceinline__ Stats* work_stats(const LogProbsArgs& a, long long row) {
  return reinterpret_cast<Stats*>(a.work + row * a.splits * (16 + 8ll * a.top) + 8ll * a.splits * a.top);
}
__device__ __forceinline__ Key* work_keys(const LogProbsArgs& a, long long row) {
  return reinterpret_cast<Key*>(a.work + row * a.splits * (16 + 8ll * a.top));
}

// The candidates of a wave: those of one group of loads, and fewer than 64 before them.
template <int N>
constexpr int pending_keys() {
  return kWave * (N + 1);
}

template <bool kHalf, bool kTop>
__global__ void __launch_bounds__(kThreads) log_probs_kernel(LogProbsArgs a) {
  constexpr int N = kHalf ? 8 : 4;  // values a load
  constexpr int kPending = pending_keys<N>();
  __shared__ Key pending[kTop ? kThreads / kWave : 1][kTop ? kPending : 1];
  __shared__ Stats stats[kThreads / kWave];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, threads = blockDim.x;
  const long long row = a.row0 + (long long)(blockIdx.x / (unsigned)a.splits);
  const int split = (int)(blockIdx.x % (unsigned)a.splits);
  const uint8_t* x_row = a.x + row * a.x_row;
  const int c1 = min(a.chunks, (split + 1) * a.chunks_each);

  Stats st = {-3.402823466e38f, 0.f, 0.f};
  Key list = 0;
  int n_pending = 0;
  float limit = -INFINITY;  // what a candidate has at least
  auto take = [&](int n) {  // n pending keys into the list
    __builtin_amdgcn_wave_barrier();  // the wave's own writes
    const Key k = lane < n ? pending[wave][n_pending - n + lane] : 0;
    __builtin_amdgcn_wave_barrier();
    n_pending -= n;
    list = merge64(list, sort64(k, lane), lane);
    const Key last = __shfl(list, a.top - 1, kWave);
    if (last) {
      // indexes that follow are larger: an equal value does not enter
      limit = fmaxf(limit, nextafterf(value_of(last), INFINITY));
      if (value_of(last) == INFINITY) limit = NAN;
    }
  };

  for (int c = split * a.chunks_each; c < c1; ++c) {
    const long long at = (long long)c * threads * kHold + (long long)N * tid;
    float x[kHold];
#pragma unroll
    for (int j = 0; j < kHold / N; ++j) load<kHalf, N>(x_row, at + (long long)j * N * threads, a.v, x + j * N);
    float mine = -INFINITY;
#pragma unroll
    for (int i = 0; i < kHold; ++i) mine = fmaxf(mine, x[i]);
    const float m = fmaxf(st.m, wave_max(mine));
    const float d0 = fmaxf((st.m - m) * a.scale, -1e4f), e0 = exp_of(d0);
    st = {m, st.s * e0, (st.t + d0 * st.s) * e0};
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      const float d = (x[i] - m) * a.scale, e = exp_of(d);
      st.s += e;
      st.t = fmaf(e, fmaxf(d, -1e4f), st.t);  // minus infinity counts nothing; NaN stays in e
    }
    if constexpr (kTop) {
      if (c == split * a.chunks_each) {
        const uint32_t o = ordered(mine);
        uint32_t bound = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
          const int n = __popcll(__ballot(o >= (bound | bit)));
          if (n >= a.top) bound |= bit;
          if (n == a.top) break;
        }
        limit = from_ordered(max(bound, ordered(-INFINITY)));
      }
#pragma unroll
      for (int j = 0; j < kHold / N; ++j) {
        const long long i0 = at + (long long)j * N * threads;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const bool in = x[j * N + e] >= limit && i0 + e < a.v;
          const unsigned long long who = __ballot(in);
          if (who == 0) continue;
          if (in) pending[wave][n_pending + __popcll(who & ((1ull << lane) - 1))] = key_of(x[j * N + e], (int)(i0 + e));
          n_pending += __popcll(who);
        }
        while (n_pending >= kWave) take(kWave);
      }
    }
  }
  if constexpr (kTop)
    if (n_pending > 0) take(n_pending);

  st.s = wave_sum_f(st.s);
  st.t = wave_sum_f(st.t);
  if (lane == 0) stats[wave] = st;
  if constexpr (kTop) pending[wave][lane] = list;
  __syncthreads();
  if (wave > 0) return;
  for (int w = 1; w < threads / kWave; ++w) {
    st = join(st, stats[w], a.scale);
    if constexpr (kTop) list = merge64(list, pending[w][lane], lane);
  }
  if (a.splits == 1) {
    answer<kHalf>(a, row, st, list, lane);
    return;
  }
  if (lane == 0) work_stats(a, row - a.row0)[split] = st;
  if (lane < a.top) work_keys(a, row - a.row0)[(long long)split * a.top + lane] = list;
}

template <bool kHalf>
__global__ void __launch_bounds__(kThreads) log_probs_join_kernel(LogProbsArgs a) {
  __shared__ Key lists[kThreads / kWave][kWave];
  __shared__ Stats stats[kThreads / kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const long long row = blockIdx.x;
  const Stats* parts = work_stats(a, row);
  const Key* keys = work_keys(a, row);
  Stats st = {-3.402823466e38f, 0.f, 0.f};
  for (int s = threadIdx.x; s < a.splits; s += kThreads) st = join(st, parts[s], a.scale);
  st = join_wave(st, a.scale);
  Key list = 0;
  if (a.top > 0)
    for (int s = wave; s < a.splits; s += kThreads / kWave)
      list = merge64(list, lane < a.top ? keys[(long long)s * a.top + lane] : 0, lane);
  if (lane == 0) stats[wave] = st;
  lists[wave][lane] = list;
  __syncthreads();
  if (wave > 0) return;
  for (int w = 1; w < kThreads / kWave; ++w) {
    st = join(st, stats[w], a.scale);
    if (a.top > 0) list = merge64(list, lists[w][lane], lane);
  }
  answer<kHalf>(a, a.row0 + row, st, list, lane);
}

// How a call is cut: workgroups of one wave for short rows; ranges until there are 1024
// workgroups, 256 ranges a row at most.
struct Plan {
  int threads, chunks, chunks_each, splits;
  size_t row_bytes;  // of the work buffer
  int64_t rows;      // a launch
};
Plan plan_of(int64_t v, int64_t rows, int64_t top) {
  Plan p{};
  p.threads = v <= kWave * kHold ? kWave : kThreads;
  const int64_t chunk = (int64_t)p.threads * kHold;
  p.chunks = (int)((v + chunk - 1) / chunk);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>({1024 / std::max<int64_t>(rows, 1), p.chunks, 256}));
  p.chunks_each = (int)((p.chunks + want - 1) / want);
  p.splits = (p.chunks + p.chunks_each - 1) / p.chunks_each;
  p.row_bytes = p.splits > 1 ? (size_t)p.splits * (16 + 8 * (size_t)top) : 0;
  // a launch has fewer than 2^32 threads
  p.rows = std::max<int64_t>(1, ((int64_t)1 << 31) / kThreads / p.splits);
  return p;
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
  const Plan p = plan_of(v, rows, top);
  if (wsize < p.row_bytes * (size_t)rows || (p.row_bytes > 0 && (wdata == nullptr || !aligned(wdata, 16))))
    return fail(hipErrorInvalidValue);

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
  a.scale = scale;
  a.v = (int)v;
  a.given = (int)given;
  a.top = (int)top;
  a.splits = p.splits;
  a.chunks = p.chunks;
  a.chunks_each = p.chunks_each;
  const hipStream_t st = current_stream();
  const bool half = x->type == WEFT_GGML_TYPE_F16;
  for (int64_t r = 0; r < rows; r += p.rows) {
    const unsigned n = (unsigned)std::min(rows - r, p.rows);
    a.row0 = r;
    a.work = static_cast<uint8_t*>(wdata) + (p.row_bytes > 0 ? p.row_bytes * (size_t)r : 0);
    const dim3 grid(n * (unsigned)p.splits);
    if (half && top > 0)
      log_probs_kernel<true, true><<<grid, p.threads, 0, st>>>(a);
    else if (half)
      log_probs_kernel<true, false><<<grid, p.threads, 0, st>>>(a);
    else if (top > 0)
      log_probs_kernel<false, true><<<grid, p.threads, 0, st>>>(a);
    else
      log_probs_kernel<false, false><<<grid, p.threads, 0, st>>>(a);
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
  return weft::plan_of(logits->ne[0], logits->ne[1], n_top).row_bytes * (size_t)logits->ne[1];
}

extern "C" int weft_ggml_log_probs(const weft_ggml_tensor* logits, const weft_ggml_tensor* tokens,
                                   const weft_ggml_tensor* token_lp, const weft_ggml_tensor* entropy,
                                   const weft_ggml_tensor* top_ids, const weft_ggml_tensor* top_lp, float scale,
                                   void* wdata, size_t wsize) {
  return (int)weft::log_probs(logits, tokens, token_lp, entropy, top_ids, top_lp, scale, wdata, wsize);
}
