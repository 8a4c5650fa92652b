// Attention of new tokens over the paged cache (kv_cache.h).
//
// For a query of head h (kv head h / share) at position p of its sequence,
//   o = sum_j softmax_j(scale q . k_j) v_j
// over the keys j <= p that lie in a page of the pool and, with a window, have
// j > p - window or j < sinks.  A query that sees no key gets zeros.
//
// One wave a (token, head): 64 keys a step, a key a lane for the scores, then a
// value a lane for the sum, with the running maximum and sum in 32 bits.
#include <algorithm>

#include "kv_cache.h"
#include "runtime.h"

namespace weft {
namespace {

struct AttendArgs {
  KvSeqs seqs;
  KvPool k, v;
  const uint8_t* q;
  uint8_t* o;
  long long q_head, q_token, o_head, o_token;  // byte strides
  int heads, share, d, window, sinks;
  float scale;
  bool half_q, half_o;
};

template <int T>
__device__ __forceinline__ float value_of(const uint8_t* row, int i) {
  const uint8_t* rec = row + (i / 32) * KvRecord<T>::kBytes;
  const int e = i & 31;
  if constexpr (T == kKvF16) return fp16_to_fp32(ld_u16(rec + 2 * e));
  const float d = fp16_to_fp32(ld_u16(rec));
  if constexpr (T == kKvQ8_0) return d * (float)(int8_t)rec[2 + e];
  return d * (float)((int)(rec[2 + (e & 15)] >> (e & 16 ? 4 : 0) & 15) - 8);
}

template <int T>
__global__ void __launch_bounds__(kWave) attend_simple_kernel(AttendArgs a) {
  __shared__ float qs[256];
  __shared__ float ps[kWave];
  __shared__ int pg[kWave], sl[kWave];
  const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y, kvh = h / a.share;
  const int seq = kv_sequence_of(a.seqs, t);
  if (seq < 0) return;
  const long long pos = kv_position(a.seqs, seq, t);
  const uint8_t* qrow = a.q + t * a.q_token + h * a.q_head;
  for (int i = lane; i < a.d; i += kWave)
    qs[i] = a.scale * (a.half_q ? fp16_to_fp32(ld_u16(qrow + 2 * i)) : *reinterpret_cast<const float*>(qrow + 4 * i));
  const int last = (int)min(pos, (long long)INT32_MAX - 64);
  float m = -INFINITY, l = 0.f, acc[4] = {};
  // no key lies past the table, whatever a length says
  const int end = (int)min((long long)last + 1, min((long long)a.seqs.max_pages * a.seqs.page_size, (long long)INT32_MAX - 64));
  const int first = min(a.window > 0 ? max(0, last - a.window + 1) : 0, end);
  const int sinks = min(a.sinks, first);
  for (int base = 0; base < sinks + end - first; base += kWave) {
    __syncthreads();
    const int n = base + lane, j = n < sinks ? n : n - sinks + first;
    int page = -1, slot = 0;
    const bool there = j < end && kv_place(a.seqs, seq, j, page, slot);
    float s = -INFINITY;
    if (there) {
      const uint8_t* row = a.k.data + page * a.k.page + slot * a.k.slot + kvh * a.k.head;
      s = 0.f;
      for (int i = 0; i < a.d; ++i) s += qs[i] * value_of<T>(row, i);
    }
    const float m1 = fmaxf(m, wave_max(s));
    if (m1 == -INFINITY) continue;
    const float p = __expf(s - m1), f = __expf(m - m1);
    l = l * f + wave_sum(p);
    m = m1;
    ps[lane] = p;
    pg[lane] = there ? page : -1;
    sl[lane] = slot;
    __syncthreads();
    for (int i = 0; i < 4; ++i) acc[i] *= f;
    for (int c = 0; c < kWave; ++c) {
      if (pg[c] < 0) continue;
      const uint8_t* row = a.v.data + pg[c] * a.v.page + sl[c] * a.v.slot + kvh * a.v.head;
      for (int i = 0; i < 4; ++i)
        if (lane + kWave * i < a.d) acc[i] += ps[c] * value_of<T>(row, lane + kWave * i);
    }
  }
  uint8_t* orow = a.o + t * a.o_token + h * a.o_head;
  for (int i = 0; i < 4; ++i) {
    const int e = lane + kWave * i;
    if (e >= a.d) break;
    const float y = l == 0.f ? 0.f : acc[i] / l;  // l NaN: a visible key was
    if (a.half_o)
      *reinterpret_cast<_Float16*>(orow + 2 * e) = (_Float16)y;
    else
      *reinterpret_cast<float*>(orow + 4 * e) = y;
  }
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
  AttendArgs a{};
  a.seqs = w.seqs;
  a.seqs.n_tokens = (int)q->ne[2];
  a.k = w.k;
  a.v = w.v;
  a.q = static_cast<const uint8_t*>(q->data);
  a.o = static_cast<uint8_t*>(dst->data);
  a.q_head = (long long)q->nb[1];
  a.q_token = (long long)q->nb[2];
  a.o_head = (long long)dst->nb[1];
  a.o_token = (long long)dst->nb[2];
  a.heads = (int)q->ne[1];
  a.share = a.heads / w.heads;
  a.d = w.d;
  a.window = (int)std::min<int64_t>(window, INT32_MAX);
  a.sinks = (int)std::min<int64_t>(sinks, INT32_MAX);
  a.scale = scale;
  a.half_q = q->type == WEFT_GGML_TYPE_F16;
  a.half_o = dst->type == WEFT_GGML_TYPE_F16;
  const dim3 grid((unsigned)a.seqs.n_tokens, (unsigned)a.heads);
  const hipStream_t st = current_stream();
  switch (w.type) {
    case kKvF16: attend_simple_kernel<kKvF16><<<grid, kWave, 0, st>>>(a); break;
    case kKvQ8_0: attend_simple_kernel<kKvQ8_0><<<grid, kWave, 0, st>>>(a); break;
    default: attend_simple_kernel<kKvQ4_0><<<grid, kWave, 0, st>>>(a); break;
  }
  check_launch("attend_simple_kernel");
  return pending_error();
}

}  // namespace
}  // namespace weft

extern "C" {

size_t weft_ggml_attention_work_size(const weft_ggml_tensor* q, const weft_ggml_tensor* k_cache,
                                     const weft_ggml_tensor* v_cache, const weft_ggml_kv_batch* batch) {
  return 0;
}

int weft_ggml_attention(const weft_ggml_tensor* q, const weft_ggml_tensor* k_cache, const weft_ggml_tensor* v_cache,
                        const weft_ggml_kv_batch* batch, const weft_ggml_tensor* dst, float scale, int64_t window,
                        int64_t sinks, void* wdata, size_t wsize) {
  return (int)weft::attention(q, k_cache, v_cache, batch, dst, scale, window, sinks, wdata, wsize);
}

}  // extern "C"
