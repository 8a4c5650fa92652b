// The residual sum and its root-mean-square norm, written as the records the
// products read:
//   s = x + r,   y = s * (1 / sqrt(mean(s^2) + eps)) * w
// with y as F32, F16 or the Q8_0 / Q8_1 / Q8_K records of the activation
// quantizers (weft_common.h), so that a MUL_MAT takes it as an src1 that is
// already quantized.
//
// One workgroup a row, a lane owning groups of four consecutive values: a
// Q8_0 / Q8_1 record is eight lanes, a Q8_K record one wave, and the values stay
// in registers between the sum of squares and the records, so memory is read
// and written once (rows past 16384 values: the sum, or the inputs, are read again).
// The square sum is held in 32 bits: a lane sums its values, 16 at most in registers
// and one in 1024 of a longer row, then trees over the lanes and waves; the terms
// are not negative, so its error is at most 2^-24 for each of those additions.
//
// Bound by memory: 16384 rows of 8192 values with a residual and its sum, to Q8_K,
// take 307 us (5.7 TB/s); 509 rows of 11008 to Q8_0 17.4 us (4.2 TB/s); a row of
// 4096 3.5 us alone, two trips to memory.
#include <algorithm>

#include "runtime.h"
#include "weft_common.h"
#include "weft_hip.h"

namespace weft {
namespace {

enum NormOut { kOutF32 = 0, kOutF16 = 1, kOutQ8_0 = 2, kOutQ8_1 = 3, kOutQ8_K = 4 };

struct NormArgs {
  const float* x;
  const float* r;    // nullptr: no residual
  const float* w;    // nullptr: ones
  float* s;          // nullptr: the sum is not kept
  uint8_t* y;
  long long x_row, r_row, s_row, y_row;  // floats; y in bytes
  int k;
  float eps;
  bool wide;    // x, r, w and s in aligned groups of four
  bool wide_y;  // and y (F32)
};

__device__ __forceinline__ float4 load4(const float* p, int i, int k, bool wide) {
  if (wide) return *reinterpret_cast<const float4*>(p + i);  // k is a multiple of four here
  float4 v;
  v.x = i < k ? p[i] : 0.f;
  v.y = i + 1 < k ? p[i + 1] : 0.f;
  v.z = i + 2 < k ? p[i + 2] : 0.f;
  v.w = i + 3 < k ? p[i + 3] : 0.f;
  return v;
}

__device__ __forceinline__ void store4(float* p, int i, int k, bool wide, float4 v) {
  if (wide) {
    *reinterpret_cast<float4*>(p + i) = v;
    return;
  }
  if (i < k) p[i] = v.x;
  if (i + 1 < k) p[i + 1] = v.y;
  if (i + 2 < k) p[i + 2] = v.z;
  if (i + 3 < k) p[i + 3] = v.w;
}

// the sum's values i..i+3 of a row, stored where the caller keeps them
__device__ __forceinline__ float4 sum4(const NormArgs& a, long long row, int i) {
  float4 v = load4(a.x + row * a.x_row, i, a.k, a.wide);
  if (a.r != nullptr) {
    const float4 r = load4(a.r + row * a.r_row, i, a.k, a.wide);
    v = make_float4(v.x + r.x, v.y + r.y, v.z + r.z, v.w + r.w);
  }
  if (a.s != nullptr) store4(a.s + row * a.s_row, i, a.k, a.wide, v);
  return v;
}

// y's values i..i+3 as the output type has them; the whole wave calls it
// (records exchange values between lanes), live: i < k
template <int Out>
__device__ __forceinline__ void put4(const NormArgs& a, uint8_t* y, int i, float4 v, bool live) {
  const int lane = threadIdx.x & (kWave - 1);
  if constexpr (Out == kOutF32) {
    if (live) store4(reinterpret_cast<float*>(y), i, a.k, a.wide && a.wide_y, v);
  } else if constexpr (Out == kOutF16) {
    _Float16* h = reinterpret_cast<_Float16*>(y);
    const float f[4] = {v.x, v.y, v.z, v.w};
    if (live && i + 3 < a.k) {
      struct __attribute__((packed, aligned(2))) {
        _Float16 h[4];
      } q = {{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w}};
      __builtin_memcpy(h + i, &q, 8);
    } else if (live) {
      for (int e = 0; e < 4; ++e)
        if (i + e < a.k) h[i + e] = (_Float16)f[e];
    }
  } else if constexpr (Out == kOutQ8_K) {
    const Q8KLane q = q8k_quantize_wave(v, lane);
    if (!live) return;
    uint8_t* rec = y + (long long)(i / 256) * kQ8_KBytes;
    if (lane == 0) *reinterpret_cast<float*>(rec) = q.d;
    *reinterpret_cast<uint32_t*>(rec + 4 + 4 * lane) = (uint32_t)pack4_i8(q.q);
    // GGML leaves an all-zero record's bsums as they were; here they are zeros
    if ((lane & 3) == 0) reinterpret_cast<int16_t*>(rec + 260)[lane / 4] = (int16_t)(q.zero ? 0 : q.bsum16);
  } else {
    constexpr int kBytes = Out == kOutQ8_0 ? kQ8_0Bytes : kQ8_1Bytes;
    const Q8_0Lane q = q80_quantize_8lanes(v);
    uint32_t sh = 0;
    if constexpr (Out == kOutQ8_1) sh = q81_sum_half(q);
    if (!live) return;
    const int part = lane & 7;
    uint8_t* rec = y + (long long)(i / 32) * kBytes;
    const uint32_t packed = (uint32_t)pack4_i8(q.q);
    uint16_t* h = reinterpret_cast<uint16_t*>(rec + (kBytes - 32) + 4 * part);
    h[0] = (uint16_t)packed;
    h[1] = (uint16_t)(packed >> 16);
    if (part == 0) {
      reinterpret_cast<uint16_t*>(rec)[0] = (uint16_t)q.dh;
      if constexpr (Out == kOutQ8_1) reinterpret_cast<uint16_t*>(rec)[1] = (uint16_t)sh;
    }
  }
}

__device__ __forceinline__ float4 weight4(const NormArgs& a, int i) {
  if (a.w != nullptr && i < a.k) return load4(a.w, i, a.k, a.wide);
  return make_float4(1.f, 1.f, 1.f, 1.f);
}
__device__ __forceinline__ float4 scale4(float4 v, float f, float4 w) {
  return make_float4(v.x * f * w.x, v.y * f * w.y, v.z * f * w.z, v.w * f * w.w);
}

// V groups of four a lane in registers (k <= 4 V threads); V == 0: any k, the
// second pass reads the sums again (its own lane's, so no barrier orders them).
template <int Out, int V>
__global__ void __launch_bounds__(1024) add_rms_norm_kernel(NormArgs a) {
  __shared__ float part[16];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, n = blockDim.x;
  uint8_t* y = a.y + row * a.y_row;
  float4 v[V > 0 ? V : 1], w[V > 0 ? V : 1];
  float q = 0.f;
  if constexpr (V > 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = 4 * (j * n + tid);
      v[j] = i < a.k ? sum4(a, row, i) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // on their way beside the row, not after its sum
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = weight4(a, 4 * (j * n + tid));
#pragma unroll
    for (int j = 0; j < V; ++j) q += (v[j].x * v[j].x + v[j].y * v[j].y) + (v[j].z * v[j].z + v[j].w * v[j].w);
  } else {
    for (int i = 4 * tid; i < a.k; i += 4 * n) {
      const float4 s = sum4(a, row, i);
      q += (s.x * s.x + s.y * s.y) + (s.z * s.z + s.w * s.w);
    }
  }
  q = wave_sum_f(q);
  if (n > kWave) {
    if ((tid & (kWave - 1)) == 0) part[tid / kWave] = q;
    __syncthreads();
    q = 0.f;
    for (int i = 0; i < n / kWave; ++i) q += part[i];
  }
  const float f = 1.f / sqrtf(q / (float)a.k + a.eps);
  if constexpr (V > 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = 4 * (j * n + tid);
      const bool live = i < a.k;
      put4<Out>(a, y, i, scale4(v[j], f, w[j]), live);
    }
  } else {
    const NormArgs again = [&] {
      NormArgs b = a;
      if (a.s != nullptr) {  // the sums, which may lie over x
        b.x = a.s;
        b.x_row = a.s_row;
        b.r = nullptr;
        b.s = nullptr;
      }
      return b;
    }();
    for (int i0 = 0; i0 < a.k; i0 += 4 * n) {
      const int i = i0 + 4 * tid;
      const bool live = i < a.k;
      const float4 s = live ? sum4(again, row, i) : make_float4(0.f, 0.f, 0.f, 0.f);
      put4<Out>(a, y, i, scale4(s, f, weight4(a, i)), live);
    }
  }
}

// A launch has fewer than 2^32 threads; past that the runtime starts the rest of the
// division, without an error.
template <int Out>
void launch(NormArgs a, int64_t rows, hipStream_t st) {
  // threads: a lane's values stay in registers up to four groups of four
  const int groups = (a.k + 3) / 4;
  int threads = kWave;
  while (threads < 1024 && threads * 4 < groups) threads *= 2;
  const int v = (groups + threads - 1) / threads;
  const int64_t most = ((int64_t)1 << 31) / threads;
  for (; rows > 0; rows -= most) {
    const dim3 grid((unsigned)std::min(rows, most));
    if (v <= 1)
      add_rms_norm_kernel<Out, 1><<<grid, threads, 0, st>>>(a);
    else if (v <= 2)
      add_rms_norm_kernel<Out, 2><<<grid, threads, 0, st>>>(a);
    else if (v <= 4)
      add_rms_norm_kernel<Out, 4><<<grid, threads, 0, st>>>(a);
    else
      add_rms_norm_kernel<Out, 0><<<grid, threads, 0, st>>>(a);
    a.x += most * a.x_row;
    if (a.r != nullptr) a.r += most * a.r_row;
    if (a.s != nullptr) a.s += most * a.s_row;
    a.y += most * a.y_row;
  }
}

hipError_t fail(hipError_t e) {
  set_error(e);
  return e;
}

// an F32 matrix of k columns and that many rows
bool matrix(const weft_ggml_tensor* t, int64_t k, int64_t rows) {
  return t->ne[0] == k && t->ne[1] == rows && t->ne[2] == 1 && t->ne[3] == 1 && t->nb[0] == 4 && t->nb[1] % 4 == 0 &&
         t->data != nullptr && aligned(t->data, 4);
}

hipError_t add_rms_norm(const weft_ggml_tensor* x, const weft_ggml_tensor* r, const weft_ggml_tensor* w,
                        const weft_ggml_tensor* s, const weft_ggml_tensor* y, float eps) {
  if (x == nullptr || y == nullptr) return fail(hipErrorInvalidValue);
  for (const weft_ggml_tensor* t : {x, r, w, s})
    if (t != nullptr && t->type != WEFT_GGML_TYPE_F32) return fail(hipErrorNotSupported);
  int out;
  size_t first;
  int64_t block;
  switch (y->type) {
    case WEFT_GGML_TYPE_F32: out = kOutF32, first = 4, block = 1; break;
    case WEFT_GGML_TYPE_F16: out = kOutF16, first = 2, block = 1; break;
    case WEFT_GGML_TYPE_Q8_0: out = kOutQ8_0, first = kQ8_0Bytes, block = 32; break;
    case WEFT_GGML_TYPE_Q8_1: out = kOutQ8_1, first = kQ8_1Bytes, block = 32; break;
    case WEFT_GGML_TYPE_Q8_K: out = kOutQ8_K, first = kQ8_KBytes, block = 256; break;
    default: return fail(hipErrorNotSupported);
  }
  const int64_t k = x->ne[0], rows = x->ne[1];
  if (k < 0 || rows < 0 || k > INT32_MAX / 2 || rows > INT32_MAX || !(eps >= 0.f) || k % block) return fail(hipErrorInvalidValue);
  const size_t unit = out == kOutF32 || out == kOutQ8_K ? 4 : 2;
  if (y->ne[0] != k || y->ne[1] != rows || y->ne[2] != 1 || y->ne[3] != 1 || y->nb[0] != first || y->nb[1] % unit ||
      !aligned(y->data, unit))
    return fail(hipErrorInvalidValue);
  if (k == 0 || rows == 0) return hipSuccess;
  if (y->data == nullptr || !matrix(x, k, rows) || (r != nullptr && !matrix(r, k, rows)) ||
      (s != nullptr && !matrix(s, k, rows)) || (w != nullptr && !matrix(w, k, 1)))
    return fail(hipErrorInvalidValue);
  NormArgs a{};
  a.x = static_cast<const float*>(x->data);
  a.x_row = (long long)(x->nb[1] / 4);
  if (r != nullptr) a.r = static_cast<const float*>(r->data), a.r_row = (long long)(r->nb[1] / 4);
  if (w != nullptr) a.w = static_cast<const float*>(w->data);
  if (s != nullptr) a.s = static_cast<float*>(s->data), a.s_row = (long long)(s->nb[1] / 4);
  a.y = static_cast<uint8_t*>(y->data);
  a.y_row = (long long)y->nb[1];
  a.k = (int)k;
  a.eps = eps;
  a.wide = k % 4 == 0;
  for (const weft_ggml_tensor* t : {x, r, w, s})
    if (t != nullptr && (!aligned(t->data, 16) || (rows > 1 && t != w && t->nb[1] % 16))) a.wide = false;
  a.wide_y = aligned(y->data, 16) && (rows == 1 || y->nb[1] % 16 == 0);
  const hipStream_t st = current_stream();
  switch (out) {
    case kOutF32: launch<kOutF32>(a, rows, st); break;
    case kOutF16: launch<kOutF16>(a, rows, st); break;
    case kOutQ8_0: launch<kOutQ8_0>(a, rows, st); break;
    case kOutQ8_1: launch<kOutQ8_1>(a, rows, st); break;
    default: launch<kOutQ8_K>(a, rows, st); break;
  }
  check_launch("add_rms_norm_kernel");
  return pending_error();
}

}  // namespace
}  // namespace weft

extern "C" int weft_ggml_add_rms_norm(const weft_ggml_tensor* x, const weft_ggml_tensor* residual,
                                      const weft_ggml_tensor* weight, const weft_ggml_tensor* sum,
                                      const weft_ggml_tensor* dst, float eps) {
  return (int)weft::add_rms_norm(x, residual, weight, sum, dst, eps);
}
