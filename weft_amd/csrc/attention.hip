// Attention of new tokens over the paged cache (kv_cache.h).
//
// For a query of head h (kv head h / share) at position p of its sequence,
//   o = sum_j softmax_j(scale q . k_j) v_j
// over the keys j <= p that lie in a page of the pool and, with a window, have
// j > p - window or j < sinks.  A query that sees no key gets zeros.
//
// attention_few.hip has tiles of 16 query rows, attention_many.hip of 128; this
// file checks calls, chooses tiles and splits, and joins the splits (a token's 32 splits
// in 4.4 us, 96 in 7.5, 48 tokens' in 6.8; 8 us for 512 tokens of 64 heads in two
// splits, 25 MB).
#include <algorithm>
#include <cmath>

#include "attention.h"
#include "runtime.h"

namespace weft {
namespace {

// The splits of a (token, head) row, each with its reference, sum and weighted
// values: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
constexpr int kJoinThreads = 256, kMaxSplits = 256;

__device__ __forceinline__ void store_row4(const AttendArgs& a, int t, int head, int e, f32x4 x, float all) {
  x *= all == 0.f ? 0.f : 1.f / all;  // a row that saw nothing: zeros
  uint8_t* dst = a.o + (long long)t * a.o_token + (long long)head * a.o_head;
  if (a.half_o) {
    const f16x4 h = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
    *reinterpret_cast<Bytes8*>(dst + 2 * e) = __builtin_bit_cast(Bytes8, h);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<float*>(dst)[e + i] = x[i];
  }
}

// where a row's partial results begin, and how many splits it has (0: none to join)
__device__ __forceinline__ int row_splits(const AttendArgs& a, int d, int token, int head, const float*& part,
                                          long long& stride) {
  const int kvh = head / a.share;
  TileRows t;
  if (!locate(a, 0, token, head - kvh * a.share, t)) return 0;
  const int n = (t.range.steps + t.each - 1) / t.each;
  const int row = (token - t.token0) * a.share + head - kvh * a.share;
  stride = (long long)a.tile * (d + 2);
  part = a.part + ((long long)(t.before + row / a.tile) * a.kv_heads + kvh) * a.splits * stride + (row % a.tile) * (d + 2);
  return n > 1 ? n : 0;  // one: written by its only split
}

// Few rows, many splits: a workgroup a row, groups of lanes taking every
// so-many-th split, four values a lane.
template <int D>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(AttendArgs a) {
  constexpr int kLanes = D <= 128 ? 32 : 64;  // of which D / 4 work
  constexpr int kGroups = kJoinThreads / kLanes;
  __shared__ float weight[kMaxSplits];
  __shared__ float wave_top[kJoinThreads / kWave], wave_sums[kJoinThreads / kWave];
  __shared__ f32x4 sums[kGroups][kLanes];
  const int t = (int)blockIdx.x, head = (int)blockIdx.y, tid = threadIdx.x;
  const float* part;
  long long stride;
  const int n = row_splits(a, D, t, head, part, stride);
  if (n == 0) return;
  float m = -INFINITY, l = 0.f;
  if (tid < n) m = part[tid * stride + D], l = part[tid * stride + D + 1];
  const float wt = wave_max(m);
  if (tid % kWave == 0) wave_top[tid / kWave] = wt;
  __syncthreads();
  float top = wave_top[0];
#pragma unroll
  for (int i = 1; i < kJoinThreads / kWave; ++i) top = fmaxf(top, wave_top[i]);
  const float w = top == -INFINITY ? 0.f : exp2_fast(m - top);
  weight[tid] = w;
  // a split that saw nothing adds nothing; one that met a NaN passes it on
  const float ws = wave_sum(tid < n ? w * l : 0.f);
  if (tid % kWave == 0) wave_sums[tid / kWave] = ws;
  __syncthreads();
  float all = 0.f;
#pragma unroll
  for (int i = 0; i < kJoinThreads / kWave; ++i) all += wave_sums[i];
  const int lane = tid % kLanes, group = tid / kLanes;
  f32x4 x = {};
  if (4 * lane < D)
    for (int i = group; i < n; i += kGroups) {
      const float* p = part + i * stride + 4 * lane;
      const f32x4 v = {p[0], p[1], p[2], p[3]};
      x += weight[i] * v;
    }
  sums[group][lane] = x;
  __syncthreads();
  if (group != 0 || 4 * lane >= D) return;
#pragma unroll
  for (int i = 1; i < kGroups; ++i) x += sums[i][lane];
  store_row4(a, t, head, 4 * lane, x, all);
}

// Many rows, few splits: a group of lanes a row, several heads of a token a
// workgroup.  Splits go four at a time, so that most rows wait for memory once.
constexpr int join_lanes(int d) { return d <= 64 ? 16 : d <= 128 ? 32 : 64; }  // of which d / 4 work
template <int D>
__global__ void __launch_bounds__(kJoinThreads) attend_join_rows_kernel(AttendArgs a) {
  constexpr int kLanes = join_lanes(D), kGroups = kJoinThreads / kLanes, kAhead = 4;
  const int t = (int)blockIdx.x, tid = threadIdx.x, lane = tid % kLanes;
  const int heads = a.kv_heads * a.share, head = (int)blockIdx.y * kGroups + tid / kLanes;
  const float* part;
  long long stride;
  const int n = row_splits(a, D, t, min(head, heads - 1), part, stride);
  if (n == 0 || head >= heads || 4 * lane >= D) return;
  float top = -INFINITY, all = 0.f;
  f32x4 x = {};
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    float m[kAhead], l[kAhead];
    f32x4 v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float* p = part + min(i0 + i, n - 1) * stride;
      m[i] = p[D], l[i] = p[D + 1];
      v[i] = f32x4{p[4 * lane], p[4 * lane + 1], p[4 * lane + 2], p[4 * lane + 3]};
    }
    float now = top;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) now = fmaxf(now, m[i]);
    const float f = now == -INFINITY ? 0.f : exp2_fast(top - now);
    top = now;
    x *= f;
    all *= f;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i >= n) break;
      const float w = top == -INFINITY ? 0.f : exp2_fast(m[i] - top);
      x += w * v[i];
      all += w * l[i];
    }
  }
  store_row4(a, t, head, 4 * lane, x, all);
}

template <int D>
void launch_join(const AttendArgs& a, bool rows, hipStream_t st) {
  const unsigned tokens = (unsigned)a.seqs.n_tokens, heads = (unsigned)(a.kv_heads * a.share);
  if (rows) {
    constexpr unsigned kGroups = kJoinThreads / join_lanes(D);
    attend_join_rows_kernel<D><<<dim3(tokens, (heads + kGroups - 1) / kGroups), kJoinThreads, 0, st>>>(a);
  } else {
    attend_join_kernel<D><<<dim3(tokens, heads), kJoinThreads, 0, st>>>(a);
  }
}

void join(int d, const AttendArgs& a, bool rows, hipStream_t st) {
  switch (d) {
    case 64: launch_join<64>(a, rows, st); break;
    case 96: launch_join<96>(a, rows, st); break;
    case 128: launch_join<128>(a, rows, st); break;
    case 192: launch_join<192>(a, rows, st); break;
    default: launch_join<256>(a, rows, st); break;
  }
  check_launch(rows ? "attend_join_rows_kernel" : "attend_join_kernel");
}

// Tiles and splits of a call, from what the host knows of it.
struct Plan {
  bool many;
  int tile, step, tiles, splits, least;
  size_t work;
};

Plan plan_of(const weft_ggml_tensor* q, const KvView& w) {
  Plan p;
  const int64_t tokens = q->ne[2], share = q->ne[1] / w.heads, seqs = w.seqs.n_seqs;
  const int64_t rows = tokens * share;
  // 32 rows a sequence on average: below, a tile of 16 rows reads the cache at its
  // full rate; above, 128 rows share a step's conversion (us in tiles of 16 and of 128,
  // Q8_0, 32 heads over 8 of 128, 16 / 32 / 64 / 128 rows: one sequence of 8192 keys
  // 21, 20, 30, 41 and 29, 29, 32, 41; 16 of up to 2048 31, 38, 50, 80 and 31, 32, 34, 44)
  p.many = rows > 32 * seqs;
  p.tile = p.many ? 128 : 16;
  p.step = p.many ? many_step(w.d) : 32;
  p.tiles = (int)std::min(tokens * ((share + p.tile - 1) / p.tile), rows / p.tile + std::min(tokens, seqs));
  p.least = 4;
  // as many workgroups as run at once, unless there are that many tiles: more of
  // them cost 10 % (131072 keys, Q8_0: 70 us at three a CU, 80 at six), as their
  // first steps and joins add up.  us at 1, 2, 3 and 4 a CU: a token over 65536 keys
  // Q8_0, heads of 64 37 29 29 29, of 128 49 41 41 44, of 256 81 88 102 103, F16 of 128
  // 48 49 52 52; tokens of 32 sequences of up to 4096 keys, in that order, 56 43 39 37,
  // 79 62 59 62, 132 144 153 156, 77 80 83 86; 300 tokens over 16384 keys, heads of 128
  // 103 100 92 97, of 256 355 278 289 286
  const int64_t resident = w.d > 128 ? 1 : p.many || w.type == kKvF16 ? 2 : 3;
  const int64_t items = (int64_t)p.tiles * w.heads, want = resident * (int64_t)cu_count();
  const int64_t steps = ((int64_t)w.seqs.max_pages * w.seqs.page_size + p.step - 1) / p.step;
  // two steps a wave cost less than a second launch that joins (one token, 256 keys:
  // 9.5 us in one split, 11.6 in two; 512 keys: 14.0 and 11.6)
  const int64_t most = !p.many && steps <= 2 * p.least ? 1 : (steps + p.least - 1) / p.least;
  p.splits = (int)std::max<int64_t>(1, std::min({(want + items - 1) / items, most, (int64_t)kMaxSplits}));
  p.work = p.splits == 1 ? 0 : (size_t)items * p.splits * p.tile * (w.d + 2) * sizeof(float);
  return p;
}

hipError_t fail(hipError_t e) {
  set_error(e);
  return e;
}

bool head_size_ok(int64_t d) { return d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

// the checks that need no pointers
hipError_t shapes(const weft_ggml_tensor* q, const KvView& w) {
  if (q == nullptr) return hipErrorInvalidValue;
  if ((q->type != WEFT_GGML_TYPE_F32 && q->type != WEFT_GGML_TYPE_F16) || !head_size_ok(w.d)) return hipErrorNotSupported;
  const size_t e = q->type == WEFT_GGML_TYPE_F32 ? 4 : 2;
  if (q->ne[0] != w.d || q->ne[1] <= 0 || q->ne[1] > 65535 || q->ne[1] % w.heads || q->ne[2] < 0 ||
      q->ne[2] > INT32_MAX / q->ne[1] || q->ne[3] != 1 || q->nb[0] != e || q->nb[1] % e || q->nb[2] % e ||
      !aligned(q->data, e))
    return hipErrorInvalidValue;
  return hipSuccess;
}

hipError_t attention(const weft_ggml_tensor* q, const weft_ggml_tensor* kc, const weft_ggml_tensor* vc,
                     const weft_ggml_kv_batch* batch, const weft_ggml_tensor* dst, float scale, int64_t window,
                     int64_t sinks, void* work, size_t work_size) {
  KvView w;
  hipError_t e = kv_view(kc, vc, batch, &w);
  if (e == hipSuccess) e = shapes(q, w);
  if (e == hipSuccess && dst == nullptr) e = hipErrorInvalidValue;
  if (e == hipSuccess && dst->type != WEFT_GGML_TYPE_F32 && dst->type != WEFT_GGML_TYPE_F16) e = hipErrorNotSupported;
  if (e != hipSuccess) return fail(e);
  const size_t oe = dst->type == WEFT_GGML_TYPE_F32 ? 4 : 2;
  if (dst->ne[0] != q->ne[0] || dst->ne[1] != q->ne[1] || dst->ne[2] != q->ne[2] || dst->ne[3] != 1 ||
      dst->nb[0] != oe || dst->nb[1] % oe || dst->nb[2] % oe || !aligned(dst->data, oe) || window < 0 || sinks < 0 ||
      !(scale - scale == 0.f))
    return fail(hipErrorInvalidValue);
  if (q->ne[2] == 0 || w.seqs.n_seqs == 0) return hipSuccess;
  if (q->data == nullptr || dst->data == nullptr) return fail(hipErrorInvalidValue);
  const Plan p = plan_of(q, w);
  if (p.work > 0 && (work == nullptr || !aligned(work, 16) || work_size < p.work)) return fail(hipErrorInvalidValue);
  if (w.seqs.n_pages == 0) w.seqs.max_pages = 0;
  AttendArgs a{};
  a.seqs = w.seqs;
  a.seqs.n_tokens = (int)q->ne[2];
  a.part = p.splits > 1 ? static_cast<float*>(work) : nullptr;
  a.items = p.tiles * w.heads;
  a.tile = p.tile;
  a.step_shift = p.step == 64 ? 6 : 5;
  a.splits = p.splits;
  a.least = p.least;
  a.kv_heads = w.heads;
  // a page's slots span less than 2^31 bytes, and so do two pages' starts
  const auto near = [&](const KvPool& c) {
    return c.slot >= 0 && c.page >= 0 && c.page < (long long)1 << 31 &&
           c.slot < ((long long)1 << 31) / w.seqs.page_size;
  };
  const bool fits = near(w.k) && near(w.v) && w.seqs.page_shift >= 0;
  a.whole16 = fits && w.seqs.page_size >= 16;
  a.whole32 = fits && w.seqs.page_size >= 32;
  const auto packed = [&](const KvPool& c) {
    return c.slot == (long long)kv_row_bytes(w.type, w.d) && c.head % 16 == 0 && c.page % 16 == 0 && aligned(c.data, 16);
  };
  a.dense = a.whole16 && packed(w.k) && packed(w.v);
  a.k = w.k;
  a.v = w.v;
  a.q = static_cast<const uint8_t*>(q->data);
  a.o = static_cast<uint8_t*>(dst->data);
  a.q_head = (long long)q->nb[1];
  a.q_token = (long long)q->nb[2];
  a.o_head = (long long)dst->nb[1];
  a.o_token = (long long)dst->nb[2];
  a.share = (int)(q->ne[1] / w.heads);
  a.window = (int)std::min<int64_t>(window, INT32_MAX);
  a.sinks = (int)std::min<int64_t>(sinks, INT32_MAX);
  a.scale = scale == 0.f ? 1.f : std::fabs(scale) * 1.44269504f;  // weights are powers of two
  a.sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
  a.half_q = q->type == WEFT_GGML_TYPE_F16;
  a.half_o = dst->type == WEFT_GGML_TYPE_F16;
  const hipStream_t st = current_stream();
  (p.many ? attend_many : attend_few)(w.type, w.d, a, st);
  if (p.splits > 1) join(w.d, a, p.many, st);
  return pending_error();
}

}  // namespace
}  // namespace weft

static __attribute__((aligned(16))) char w_stand_in[16];

extern "C" {

size_t weft_ggml_attention_work_size(const weft_ggml_tensor* q, const weft_ggml_tensor* k_cache,
                                     const weft_ggml_tensor* v_cache, const weft_ggml_kv_batch* batch) {
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || batch == nullptr) return 0;
  // the shapes alone count: buffers may be allocated later
  weft_ggml_tensor k = *k_cache, v = *v_cache;
  weft_ggml_kv_batch b = *batch;
  for (weft_ggml_tensor* t : {&k, &v, &b.pages, &b.starts, &b.lengths})
    if (t->data == nullptr) t->data = w_stand_in;
  weft::KvView w;
  if (weft::kv_view(&k, &v, &b, &w) != hipSuccess || weft::shapes(q, w) != hipSuccess) return 0;
  return q->ne[2] == 0 || w.seqs.n_seqs == 0 ? 0 : weft::plan_of(q, w).work;
}

int weft_ggml_attention(const weft_ggml_tensor* q, const weft_ggml_tensor* k_cache, const weft_ggml_tensor* v_cache,
                        const weft_ggml_kv_batch* batch, const weft_ggml_tensor* dst, float scale, int64_t window,
                        int64_t sinks, void* wdata, size_t wsize) {
  return (int)weft::attention(q, k_cache, v_cache, batch, dst, scale, window, sinks, wdata, wsize);
}

}  // extern "C"
