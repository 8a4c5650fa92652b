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
// consecutive groups of four (write) or eight (read) values, keys and values
// in one launch.  Writing 5500 tokens of 8 heads of 128 F32 values as Q4_0 takes
// 18 us (2.9 TB/s), as Q8_0 18 (3.1), as F16 13.5 (5.0); reading 32 sequences of up to 16384 Q8_0 tokens into F16
// 545 us (5.3 TB/s, the zeros past their lengths with them); one token 3.3 us, and
// 131 tokens back 4.7 us: launches and the dependent loads of a row's place.
#include <limits.h>

#include <algorithm>

#include "kv_cache.h"
#include "runtime.h"

namespace weft {
namespace {

constexpr int kThreads = 256;
// A launch has fewer than 2^32 threads: past that the runtime starts the rest of the
// division, without an error.
constexpr int kMostBlocks = (int)(((int64_t)1 << 31) / kThreads);

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

// `waves` waves a token, blockIdx.y: keys or values.  A token's row is heads x d
// values, each 8 lanes own a record of it, and a lane has up to four groups of
// four values in flight; the first are on their way while the row's place is
// looked up (starts, length, page: three dependent loads, most of a small call).
template <int T, bool kHalfSrc>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(KvSeqs seqs, KvPool k, KvPool v, Rows kx, Rows vx, int d,
                                                            int heads, int waves, int t0) {
  constexpr int U = 4;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int t = t0 + (int)blockIdx.x * (kThreads / kWave / waves) + wave / waves;
  const int stride = waves * kWave, first = wave % waves * kWave;
  if ((unsigned)t >= (unsigned)seqs.n_tokens) return;
  const KvPool pool = blockIdx.y ? v : k;
  const Rows rows = blockIdx.y ? vx : kx;
  const uint8_t* src = rows.data + t * rows.token;
  const int per_head = d / 4, total = heads * per_head;
  float4 x[U];
  int h[U], c[U];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * stride >= total) break;
      const int i = min(i0 + u * stride + lane, total - 1);  // past the row: its last values, not stored
      h[u] = i / per_head;
      c[u] = i - h[u] * per_head;
      x[u] = load4<kHalfSrc>(src + h[u] * rows.head + (long long)c[u] * (kHalfSrc ? 8 : 16));
    }
  };
  load(first);
  const int seq = kv_sequence_of(seqs, t);
  if (seq < 0) return;
  const long long pos = kv_position(seqs, seq, t);
  int page, slot;
  if (pos < 0 || pos > INT32_MAX || !kv_place(seqs, seq, (int)pos, page, slot)) return;
  uint8_t* at = pool.data + page * pool.page + slot * pool.slot;
  for (int i0 = first; i0 < total; i0 += U * stride) {
    if (i0 > first) load(i0);
    // whole waves: a record's lanes exchange values
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * stride < total)
        store_record<T>(at + h[u] * pool.head, c[u] / 8, c[u] & 7, x[u], i0 + u * stride + lane < total);
  }
}

// Eight values (the part-th of a record's four groups) in 16 bits, bit for bit
// the 32-bit value rounded once, or in 32.
template <int T>
__device__ __forceinline__ Bytes16 load8(const uint8_t* rec, int part, uint32_t& step) {
  Bytes16 b{};
  if constexpr (T == kKvF16) {
    b = *reinterpret_cast<const Bytes16*>(rec + 16 * part);
  } else {
    step = ld_u16(rec);
    // Q4_0: parts 0 and 1 are the low, 2 and 3 the high halves of the bytes
    const Bytes8 w = *reinterpret_cast<const Bytes8*>(rec + 2 + 8 * (T == kKvQ8_0 ? part : part & 1));
    b.w[0] = w.w[0];
    b.w[1] = w.w[1];
  }
  return b;
}
template <int T>
__device__ __forceinline__ void values8(const Bytes16& b, int part, uint32_t step, float (&x)[8]) {
  if constexpr (T == kKvF16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fp16_to_fp32(b.w[i / 2] >> (16 * (i & 1)) & 0xffffu);
  } else {
    const float d = fp16_to_fp32(step);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = b.w[i / 4] >> (8 * (i & 3));
      x[i] = d * (float)(T == kKvQ8_0 ? (int)(int8_t)w : (int)(w >> (part & 2 ? 4 : 0) & 15u) - 8);
    }
  }
}

// blockIdx.x: kReadTokens positions, blockIdx.y: sequence, blockIdx.z: keys or
// values; zeros where the sequence has no value.  The positions' rows are looked
// up once; then a thread has four groups of eight values in flight, and a wave
// writes 1 KiB of F16 in one store, past the caches (us past them and through them, 134
// MB written: 29 and 29, 268 MB: 65 and 86, 2147 MB: 542 and 582; with a copy of it all
// right after: 79 and 82, 178 and 177, 1239 and 1282; with a reduction instead: 112 and
// 93, 225 and 234, 1582 and 1634: a reader of what the Infinity Cache would hold loses).
typedef _Float16 half8 __attribute__((ext_vector_type(8), aligned(2)));
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
constexpr int kReadTokens = 8;
template <int T, bool kHalfOut>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvSeqs seqs, KvPool k, KvPool v, Rows ko, Rows vo,
                                                           long long k_seq, long long v_seq, int d, int heads,
                                                           int n_pos, int p_first) {
  __shared__ long long place[kReadTokens];
  const int seq = (int)blockIdx.y;
  const KvPool pool = blockIdx.z ? v : k;
  const Rows out = blockIdx.z ? vo : ko;
  const int p0 = p_first + (int)blockIdx.x * kReadTokens;
  const int n = min(kReadTokens, n_pos - p0);
  if ((int)threadIdx.x < n) {
    const int pos = p0 + (int)threadIdx.x;
    int page, slot;
    place[threadIdx.x] = pos < seqs.lengths[seq] && kv_place(seqs, seq, pos, page, slot)
                             ? page * pool.page + slot * pool.slot
                             : LLONG_MIN;
  }
  __syncthreads();
  uint8_t* dst = out.data + seq * (blockIdx.z ? v_seq : k_seq) + p0 * out.token;
  const int per_head = d / 8, per_token = heads * per_head, total = n * per_token;
  constexpr int U = 4;
  for (int i0 = threadIdx.x; i0 < total; i0 += U * kThreads) {
    Bytes16 b[U];
    uint32_t step[U];
    uint8_t* to[U];
    int part[U];
    bool there[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kThreads;
      const int j = i / per_token, r = i - j * per_token, h = r / per_head, c = r - h * per_head;
      to[u] = i < total ? dst + j * out.token + h * out.head + (long long)c * (kHalfOut ? 16 : 32) : nullptr;
      const long long at = i < total ? place[j] : LLONG_MIN;
      there[u] = at != LLONG_MIN;
      part[u] = c & 3;
      if (there[u])
        b[u] = load8<T>(pool.data + at + h * pool.head + (c / 4) * KvRecord<T>::kBytes, c & 3, step[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (to[u] == nullptr) continue;
      float x[8] = {};
      if (there[u]) values8<T>(b[u], part[u], step[u], x);
      if constexpr (kHalfOut) {
        const half8 y = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3],
                         (_Float16)x[4], (_Float16)x[5], (_Float16)x[6], (_Float16)x[7]};
        __builtin_nontemporal_store(y, reinterpret_cast<half8*>(to[u]));
      } else {
        __builtin_nontemporal_store(float4u{x[0], x[1], x[2], x[3]}, reinterpret_cast<float4u*>(to[u]));
        __builtin_nontemporal_store(float4u{x[4], x[5], x[6], x[7]}, reinterpret_cast<float4u*>(to[u] + 16));
      }
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
  // few tokens: a workgroup each, one group a lane (8 x 128 values, one token:
  // 2.8 us against 4.6); more than are resident at once: a wave each (6,500 tokens of
  // Q4_0: 16.9 us against 19.4)
  const int waves = w.seqs.n_tokens <= 4 * cu_count() ? 4 : 1;
  const int each = kThreads / kWave / waves;  // tokens a workgroup
  const bool half = kx->type == WEFT_GGML_TYPE_F16;
  const hipStream_t st = current_stream();
#define WEFT_KV_WRITE(T)                                                                                             \
  (half ? kv_write_kernel<T, true><<<grid, kThreads, 0, st>>>(w.seqs, w.k, w.v, kr, vr, w.d, w.heads, waves, first)  \
        : kv_write_kernel<T, false><<<grid, kThreads, 0, st>>>(w.seqs, w.k, w.v, kr, vr, w.d, w.heads, waves, first))
  for (int64_t t0 = 0; t0 < w.seqs.n_tokens; t0 += (int64_t)kMostBlocks * each) {
    const int first = (int)t0;
    const dim3 grid((unsigned)std::min<int64_t>(kMostBlocks, (w.seqs.n_tokens - t0 + each - 1) / each), 2);
    switch (w.type) {
      case kKvF16: WEFT_KV_WRITE(kKvF16); break;
      case kKvQ8_0: WEFT_KV_WRITE(kKvQ8_0); break;
      default: WEFT_KV_WRITE(kKvQ4_0); break;
    }
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
  const bool half = ko->type == WEFT_GGML_TYPE_F16;
  const hipStream_t st = current_stream();
  const long long ks = (long long)ko->nb[3], vs = (long long)vo->nb[3];
#define WEFT_KV_READ(T)                                                                                            \
  (half ? kv_read_kernel<T, true><<<grid, kThreads, 0, st>>>(w.seqs, w.k, w.v, kr, vr, ks, vs, w.d, w.heads,       \
                                                             n_pos, first)                                         \
        : kv_read_kernel<T, false><<<grid, kThreads, 0, st>>>(w.seqs, w.k, w.v, kr, vr, ks, vs, w.d, w.heads,      \
                                                              n_pos, first))
  for (int64_t p0 = 0; p0 < n_pos; p0 += (int64_t)kMostBlocks * kReadTokens) {
    const int first = (int)p0;
    const dim3 grid((unsigned)std::min<int64_t>(kMostBlocks, (n_pos - p0 + kReadTokens - 1) / kReadTokens),
                    (unsigned)w.seqs.n_seqs, 2);
    switch (w.type) {
      case kKvF16: WEFT_KV_READ(kKvF16); break;
      case kKvQ8_0: WEFT_KV_READ(kKvQ8_0); break;
      default: WEFT_KV_READ(kKvQ4_0); break;
    }
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
  if (kc->ne[0] * kc->ne[2] > (int64_t)1 << 30) return hipErrorInvalidValue;  // a token's values are counted in 32 bits
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
