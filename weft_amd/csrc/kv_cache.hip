// Writing new tokens' keys and values into the paged cache, and reading
// sequences back from it (kv_cache.h has the cache's shape).
//
// Records are GGML's: F16 rounds to nearest even; Q8_0 is the activation
// quantizer's (d = amax / 127, codes rounded half away); Q4_0 takes the value
// of largest magnitude (the first, where several are) as -8 steps:
//   d = top / -8, code = min(15, trunc(x / d + 8.5)), value = d (code - 8),
// code j in the low and code j + 16 in the high half of byte j.
//
// Both directions are one pass bound by memory: a workgroup's threads take
// consecutive groups of four (write) or sixteen (read) values, keys and values
// in one launch.
#include <algorithm>

#include "kv_cache.h"
#include "runtime.h"

namespace weft {
namespace {

constexpr int kThreads = 256;

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) Bytes8 {
  uint32_t w[2];
};
struct __attribute__((packed, aligned(2))) Bytes16 {
  uint32_t w[4];
};
struct __attribute__((packed, aligned(4))) Floats4 {
  float f[4];
};

// the new rows: values of (token, head) at byte strides
struct Rows {
  uint8_t* data;
  long long head, token;
};

template <bool kHalfSrc>
__device__ __forceinline__ float4 load4(const uint8_t* p) {
  if constexpr (kHalfSrc) {
    const Bytes8 b = *reinterpret_cast<const Bytes8*>(p);
    const half4 h = __builtin_bit_cast(half4, b);
    return make_float4((float)h[0], (float)h[1], (float)h[2], (float)h[3]);
  } else {
    const Floats4 f = *reinterpret_cast<const Floats4*>(p);
    return make_float4(f.f[0], f.f[1], f.f[2], f.f[3]);
  }
}

// Four values a lane, a record in eight lanes: the lane's part of the record.
template <int T>
__device__ __forceinline__ void store_record(uint8_t* row, int block, int part, float4 x, bool live) {
  if constexpr (T == kKvF16) {
    const half4 h = {(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w};
    if (live) *reinterpret_cast<Bytes8*>(row + 64 * block + 8 * part) = __builtin_bit_cast(Bytes8, h);
  } else if constexpr (T == kKvQ8_0) {
    const Q8_0Lane r = q80_quantize_8lanes(x);
    if (!live) return;
    uint8_t* rec = row + kQ8_0Bytes * block;
    const uint32_t packed = (uint32_t)pack4_i8(r.q);
    uint16_t* q = reinterpret_cast<uint16_t*>(rec + 2 + 4 * part);
    q[0] = (uint16_t)packed;
    q[1] = (uint16_t)(packed >> 16);
    if (part == 0) *reinterpret_cast<uint16_t*>(rec) = (uint16_t)r.dh;
  } else {
#pragma clang fp contract(off)
    const float v[4] = {x.x, x.y, x.z, x.w};
    float top = 0.f, mine = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (fabsf(v[i]) > top) {
        top = fabsf(v[i]);
        mine = v[i];
      }
    const float all = group_max<8>(top);
    int first = top == all ? part : 8;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) first = min(first, __shfl_xor(first, o, kWave));
    const float value = __shfl(mine, first, 8);
    const float d = value / -8.f;
    const float id = d != 0.f ? __fdiv_rn(1.f, d) : 0.f;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = (int)(v[i] * id + 8.5f);
      codes |= (uint32_t)(max(0, min(15, q))) << (8 * i);
    }
    const uint32_t other = (uint32_t)__shfl_xor((int)codes, 4, kWave);
    if (!live) return;
    uint8_t* rec = row + kQ4_0Bytes * block;
    if (part < 4) {
      const uint32_t packed = codes | other << 4;
      uint16_t* q = reinterpret_cast<uint16_t*>(rec + 2 + 4 * part);
      q[0] = (uint16_t)packed;
      q[1] = (uint16_t)(packed >> 16);
    } else if (part == 4) {
      *reinterpret_cast<uint16_t*>(rec) = (uint16_t)fp32_to_fp16(d);
    }
  }
}

// blockIdx.x: token, blockIdx.y: keys or values.  A token's row is heads x d
// values; each 8 lanes own a record.
template <int T, bool kHalfSrc>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(KvSeqs seqs, KvPool k, KvPool v, Rows kx, Rows vx, int d,
                                                            int heads) {
  const int t = (int)blockIdx.x;
  const KvPool pool = blockIdx.y ? v : k;
  const Rows rows = blockIdx.y ? vx : kx;
  const int seq = kv_sequence_of(seqs, t);
  if (seq < 0) return;
  const long long pos = kv_position(seqs, seq, t);
  int page, slot;
  if (pos < 0 || pos > INT32_MAX || !kv_place(seqs, seq, (int)pos, page, slot)) return;
  uint8_t* at = pool.data + page * pool.page + slot * pool.slot;
  const uint8_t* src = rows.data + t * rows.token;
  const int per_head = d / 4, total = heads * per_head;
  // whole waves stay in the loop: a record's lanes exchange values
  for (int i0 = 0; i0 < total; i0 += kThreads) {
    const int i = i0 + (int)threadIdx.x;
    const bool live = i < total;
    const int h = live ? i / per_head : 0, c = live ? i - h * per_head : 0;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) x = load4<kHalfSrc>(src + h * rows.head + (long long)c * (kHalfSrc ? 8 : 16));
    store_record<T>(at + h * pool.head, c / 8, c & 7, x, live);
  }
}

// sixteen values of half a record
template <int T>
__device__ __forceinline__ void read16(const uint8_t* rec, int part, float (&x)[16]) {
  if constexpr (T == kKvF16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const half4 h = __builtin_bit_cast(half4, *reinterpret_cast<const Bytes8*>(rec + 32 * part + 8 * j));
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * j + i] = (float)h[i];
    }
  } else if constexpr (T == kKvQ8_0) {
    const float d = fp16_to_fp32(ld_u16(rec));
    const Bytes16 b = *reinterpret_cast<const Bytes16*>(rec + 2 + 16 * part);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = d * (float)(int8_t)(b.w[i / 4] >> (8 * (i & 3)));
  } else {
    const float d = fp16_to_fp32(ld_u16(rec));
    const Bytes16 b = *reinterpret_cast<const Bytes16*>(rec + 2);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = d * (float)((int)(b.w[i / 4] >> (8 * (i & 3) + 4 * part) & 15u) - 8);
  }
}

// blockIdx.x: 16 positions, blockIdx.y: sequence, blockIdx.z: keys or values;
// zeros where the sequence has no value.
constexpr int kReadTokens = 16;
template <int T, bool kHalfOut>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvSeqs seqs, KvPool k, KvPool v, Rows ko, Rows vo,
                                                           long long k_seq, long long v_seq, int d, int heads,
                                                           int n_pos) {
  const int seq = (int)blockIdx.y;
  const KvPool pool = blockIdx.z ? v : k;
  const Rows out = blockIdx.z ? vo : ko;
  uint8_t* dst = out.data + seq * (blockIdx.z ? v_seq : k_seq);
  const int length = seqs.lengths[seq];
  const int p0 = (int)blockIdx.x * kReadTokens;
  const int n = min(kReadTokens, n_pos - p0);
  const int per_head = d / 16, per_token = heads * per_head, total = n * per_token;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int j = i / per_token, r = i - j * per_token, h = r / per_head, c = r - h * per_head;
    const int pos = p0 + j;
    float x[16];
    int page, slot;
    if (pos < length && kv_place(seqs, seq, pos, page, slot)) {
      read16<T>(pool.data + page * pool.page + slot * pool.slot + h * pool.head + (c / 2) * KvRecord<T>::kBytes, c & 1,
                x);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = 0.f;
    }
    uint8_t* y = dst + pos * out.token + h * out.head + (long long)c * (kHalfOut ? 32 : 64);
    if constexpr (kHalfOut) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const half4 v4 = {(_Float16)x[4 * e], (_Float16)x[4 * e + 1], (_Float16)x[4 * e + 2], (_Float16)x[4 * e + 3]};
        reinterpret_cast<Bytes8*>(y)[e] = __builtin_bit_cast(Bytes8, v4);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<Floats4*>(y)[e] = Floats4{{x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]}};
    }
  }
}

constexpr int32_t kI32 = WEFT_GGML_TYPE_I32;

bool int_table(const weft_ggml_tensor& t) {
  return t.type == kI32 && t.nb[0] == 4 && aligned(t.data, 4) && t.ne[2] == 1 && t.ne[3] == 1 && t.ne[0] >= 0 &&
         t.ne[1] >= 0 && (t.data != nullptr || t.ne[0] == 0 || t.ne[1] == 0);
}

// rows of (d, heads, n, outer) values of F32 or F16 with element-aligned strides
hipError_t dense_rows(const weft_ggml_tensor* t, int64_t d, int64_t heads) {
  if (t == nullptr) return hipErrorInvalidValue;
  if (t->type != WEFT_GGML_TYPE_F32 && t->type != WEFT_GGML_TYPE_F16) return hipErrorNotSupported;
  const size_t e = t->type == WEFT_GGML_TYPE_F32 ? 4 : 2;
  if (t->ne[0] != d || t->ne[1] != heads || t->ne[2] < 0 || t->ne[3] < 0 || t->ne[2] > INT32_MAX || t->nb[0] != e ||
      t->nb[1] % e || t->nb[2] % e || t->nb[3] % e || !aligned(t->data, e))
    return hipErrorInvalidValue;
  return hipSuccess;
}

hipError_t fail(hipError_t e) {
  set_error(e);
  return e;
}

hipError_t kv_write(const weft_ggml_tensor* kx, const weft_ggml_tensor* vx, const weft_ggml_kv_batch* batch,
                    const weft_ggml_tensor* kc, const weft_ggml_tensor* vc) {
  KvView w;
  hipError_t e = kv_view(kc, vc, batch, &w);
  if (e == hipSuccess) e = dense_rows(kx, w.d, w.heads);
  if (e == hipSuccess) e = dense_rows(vx, w.d, w.heads);
  if (e != hipSuccess) return fail(e);
  if (kx->type != vx->type) return fail(hipErrorNotSupported);
  if (kx->ne[2] != vx->ne[2] || kx->ne[3] != 1 || vx->ne[3] != 1) return fail(hipErrorInvalidValue);
  if (kx->ne[2] == 0 || w.seqs.n_seqs == 0 || w.seqs.n_pages == 0) return hipSuccess;
  if (kx->data == nullptr || vx->data == nullptr) return fail(hipErrorInvalidValue);
  w.seqs.n_tokens = (int)kx->ne[2];
  const Rows kr{static_cast<uint8_t*>(kx->data), (long long)kx->nb[1], (long long)kx->nb[2]};
  const Rows vr{static_cast<uint8_t*>(vx->data), (long long)vx->nb[1], (long long)vx->nb[2]};
  const dim3 grid((unsigned)w.seqs.n_tokens, 2);
  const bool half = kx->type == WEFT_GGML_TYPE_F16;
  const hipStream_t st = current_stream();
#define WEFT_KV_WRITE(T)                                                                                         \
  (half ? kv_write_kernel<T, true><<<grid, kThreads, 0, st>>>(w.seqs, w.k, w.v, kr, vr, w.d, w.heads)            \
        : kv_write_kernel<T, false><<<grid, kThreads, 0, st>>>(w.seqs, w.k, w.v, kr, vr, w.d, w.heads))
  switch (w.type) {
    case kKvF16: WEFT_KV_WRITE(kKvF16); break;
    case kKvQ8_0: WEFT_KV_WRITE(kKvQ8_0); break;
    default: WEFT_KV_WRITE(kKvQ4_0); break;
  }
#undef WEFT_KV_WRITE
  check_launch("kv_write_kernel");
  return pending_error();
}

hipError_t kv_read(const weft_ggml_tensor* kc, const weft_ggml_tensor* vc, const weft_ggml_kv_batch* batch,
                   const weft_ggml_tensor* ko, const weft_ggml_tensor* vo) {
  KvView w;
  hipError_t e = kv_view(kc, vc, batch, &w);
  if (e == hipSuccess) e = dense_rows(ko, w.d, w.heads);
  if (e == hipSuccess) e = dense_rows(vo, w.d, w.heads);
  if (e != hipSuccess) return fail(e);
  if (ko->type != vo->type) return fail(hipErrorNotSupported);
  if (ko->ne[2] != vo->ne[2] || ko->ne[3] != w.seqs.n_seqs || vo->ne[3] != w.seqs.n_seqs || w.seqs.n_seqs > 65535)
    return fail(hipErrorInvalidValue);
  if (ko->ne[2] == 0 || w.seqs.n_seqs == 0) return hipSuccess;
  if (ko->data == nullptr || vo->data == nullptr) return fail(hipErrorInvalidValue);
  const Rows kr{static_cast<uint8_t*>(ko->data), (long long)ko->nb[1], (long long)ko->nb[2]};
  const Rows vr{static_cast<uint8_t*>(vo->data), (long long)vo->nb[1], (long long)vo->nb[2]};
  const int n_pos = (int)ko->ne[2];
  const dim3 grid((unsigned)((ko->ne[2] + kReadTokens - 1) / kReadTokens), (unsigned)w.seqs.n_seqs, 2);
  const bool half = ko->type == WEFT_GGML_TYPE_F16;
  const hipStream_t st = current_stream();
  const long long ks = (long long)ko->nb[3], vs = (long long)vo->nb[3];
#define WEFT_KV_READ(T)                                                                                              \
  (half ? kv_read_kernel<T, true><<<grid, kThreads, 0, st>>>(w.seqs, w.k, w.v, kr, vr, ks, vs, w.d, w.heads, n_pos)  \
        : kv_read_kernel<T, false><<<grid, kThreads, 0, st>>>(w.seqs, w.k, w.v, kr, vr, ks, vs, w.d, w.heads, n_pos))
  switch (w.type) {
    case kKvF16: WEFT_KV_READ(kKvF16); break;
    case kKvQ8_0: WEFT_KV_READ(kKvQ8_0); break;
    default: WEFT_KV_READ(kKvQ4_0); break;
  }
#undef WEFT_KV_READ
  check_launch("kv_read_kernel");
  return pending_error();
}

}  // namespace

int kv_type_of(int32_t t) {
  switch (t) {
    case WEFT_GGML_TYPE_F16: return kKvF16;
    case WEFT_GGML_TYPE_Q8_0: return kKvQ8_0;
    case WEFT_GGML_TYPE_Q4_0: return kKvQ4_0;
    default: return -1;
  }
}

size_t kv_row_bytes(int type, int64_t d) {
  const size_t rec = type == kKvF16 ? 64 : type == kKvQ8_0 ? kQ8_0Bytes : kQ4_0Bytes;
  return rec * (size_t)(d / 32);
}

hipError_t kv_view(const weft_ggml_tensor* kc, const weft_ggml_tensor* vc, const weft_ggml_kv_batch* b, KvView* out) {
  if (kc == nullptr || vc == nullptr || b == nullptr) return hipErrorInvalidValue;
  const int type = kv_type_of(kc->type);
  if (type < 0 || vc->type != kc->type) return hipErrorNotSupported;
  const size_t first = type == kKvF16 ? 2 : type == kKvQ8_0 ? kQ8_0Bytes : kQ4_0Bytes;
  for (const weft_ggml_tensor* t : {kc, vc}) {
    for (int i = 0; i < 4; ++i)
      if (t->ne[i] != kc->ne[i] || t->ne[i] < 0 || t->ne[i] > INT32_MAX) return hipErrorInvalidValue;
    if (t->nb[0] != first || t->nb[1] % 2 || t->nb[2] % 2 || t->nb[3] % 2 || !aligned(t->data, 2) ||
        (t->data == nullptr && t->ne[3] > 0))
      return hipErrorInvalidValue;
  }
  if (kc->ne[0] == 0 || kc->ne[0] % 32 || kc->ne[1] == 0 || kc->ne[2] == 0) return hipErrorInvalidValue;
  if (!int_table(b->pages) || !int_table(b->starts) || !int_table(b->lengths)) return hipErrorInvalidValue;
  const int64_t n = b->lengths.ne[0];
  if (n > INT32_MAX - 1 || b->lengths.ne[1] != 1 || b->starts.ne[0] != n + 1 || b->starts.ne[1] != 1 ||
      b->pages.ne[1] != n || b->pages.ne[0] > INT32_MAX || b->pages.nb[1] % 4)
    return hipErrorInvalidValue;
  KvSeqs& s = out->seqs;
  s.pages = static_cast<const int32_t*>(b->pages.data);
  s.starts = static_cast<const int32_t*>(b->starts.data);
  s.lengths = static_cast<const int32_t*>(b->lengths.data);
  s.pages_row = (long long)(b->pages.nb[1] / 4);
  s.n_seqs = (int)n;
  s.max_pages = (int)b->pages.ne[0];
  s.n_tokens = 0;
  s.page_size = (int)kc->ne[1];
  s.n_pages = (int)kc->ne[3];
  s.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (s.page_size == 1 << i) s.page_shift = i;
  out->k = KvPool{static_cast<uint8_t*>(kc->data), (long long)kc->nb[1], (long long)kc->nb[2], (long long)kc->nb[3]};
  out->v = KvPool{static_cast<uint8_t*>(vc->data), (long long)vc->nb[1], (long long)vc->nb[2], (long long)vc->nb[3]};
  out->type = type;
  out->d = (int)kc->ne[0];
  out->heads = (int)kc->ne[2];
  return hipSuccess;
}

}  // namespace weft

extern "C" {

int weft_ggml_kv_write(const weft_ggml_tensor* k, const weft_ggml_tensor* v, const weft_ggml_kv_batch* batch,
                       const weft_ggml_tensor* k_cache, const weft_ggml_tensor* v_cache) {
  return (int)weft::kv_write(k, v, batch, k_cache, v_cache);
}

int weft_ggml_kv_read(const weft_ggml_tensor* k_cache, const weft_ggml_tensor* v_cache,
                      const weft_ggml_kv_batch* batch, const weft_ggml_tensor* k, const weft_ggml_tensor* v) {
  return (int)weft::kv_read(k_cache, v_cache, batch, k, v);
}

}  // extern "C"
