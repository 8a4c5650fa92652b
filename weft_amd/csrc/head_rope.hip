// The norm of each query and key head and the rotation of its values by the token's
// position, in one pass between the products and the cache:
//   y = x / sqrt(mean(x^2) + eps) * w        (the mean over a head's D values)
//   (a, b) -> g (a cos t - b sin t, a sin t + b cos t),   t = p s base^(-2 i / n) / f_i
// for the pairs i < n / 2 of a head's first n values: (i, i + n / 2), or neighbours
// (2 i, 2 i + 1); the values from n on are only normed.
//
// A head is 8 to 64 lanes of eight values: four pairs, or eight values past the rotated ones.
// A lane has both values of its pairs, so the rotation moves nothing between lanes.  The
// angles depend on the token and the lane alone: a wave computes its own once for the
// heads of a token it walks, from the pairs' frequencies, computed once a workgroup.  They
// are kept in 64 bits as turns, t / 2 pi, of which the whole part is dropped before the sine
// and cosine are taken in 32: at position 10^6 a turn in 32 bits would be off by 0.06.
//
// Bound by memory: 16384 tokens of 64 + 8 heads of 128 16-bit values take 134 us (4.5 TB/s; with the
// frequencies computed in each wave 7 us more), one token 3.5 us, of which a launch is 2.4.  Tried:
// stores that pass the caches (5 us less, and whoever reads the result next loses more), two
// passes of loads on their way (nothing).
#include <algorithm>
#include <cmath>

#include "runtime.h"
#include "weft_common.h"
#include "weft_hip.h"

namespace weft {
namespace {

constexpr int kThreads = 256;
constexpr int kMostHead = 256;
// A launch has fewer than 2^32 threads: past that the runtime starts the rest of the
// division, without an error.
constexpr int64_t kMostGroups = ((int64_t)1 << 31) / kThreads;

struct Heads {
  const uint8_t* x;
  uint8_t* y;
  const float* weight;
  long long x_head, x_token, y_head, y_token;  // bytes
  int n;
};

struct RopeArgs {
  Heads q, k;
  const int32_t* positions;
  const float* factors;
  double turn;      // s / (2 pi)
  double log_step;  // -2 log2(base) / n
  float magnitude, eps, per_value;  // per_value: 1 / d
  int d, n_rot, pair_units, units;  // units of eight values: pairs first, then the rest
  int parts;                        // waves a token
  long long tokens;
  bool normed, neighbours;
};

struct __attribute__((packed, aligned(4))) Floats4 {
  float f[4];
};
struct __attribute__((packed, aligned(2))) Halves4 {
  _Float16 h[4];
};

// four values at p, of which `n` are there
template <bool kHalf>
__device__ __forceinline__ void load4(const uint8_t* row, int at, int n, float* x) {
  if (n >= 4) {
    if constexpr (kHalf) {
      const Halves4 v = *reinterpret_cast<const Halves4*>(row + 2 * at);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (float)v.h[e];
    } else {
      const Floats4 v = *reinterpret_cast<const Floats4*>(row + 4 * at);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = v.f[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (kHalf)
        x[e] = e < n ? (float)reinterpret_cast<const _Float16*>(row)[at + e] : 0.f;
      else
        x[e] = e < n ? reinterpret_cast<const float*>(row)[at + e] : 0.f;
    }
  }
}
template <bool kHalf>
__device__ __forceinline__ void store4(uint8_t* row, int at, int n, const float* x) {
  if (n >= 4) {
    if constexpr (kHalf)
      *reinterpret_cast<Halves4*>(row + 2 * at) = {{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]}};
    else
      *reinterpret_cast<Floats4*>(row + 4 * at) = {{x[0], x[1], x[2], x[3]}};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= n) continue;
      if constexpr (kHalf)
        reinterpret_cast<_Float16*>(row)[at + e] = (_Float16)x[e];
      else
        reinterpret_cast<float*>(row)[at + e] = x[e];
    }
  }
}

// the sum over aligned groups of G lanes, in each of them
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dppf<kDppXor1>(v);
  v += dppf<kDppXor2>(v);
  v += dppf<kDppHalfMirror>(v);
  if constexpr (G > 8) v += dppf<kDppMirror>(v);
  if constexpr (G > 16) v += __shfl_xor(v, 16, kWave);
  if constexpr (G > 32) v += __shfl_xor(v, 32, kWave);
  return v;
}
// 1 / sqrt(v) within two units of its last place; the instruction takes normal numbers, which v is
// unless eps is next to nothing
__device__ __forceinline__ float inverse_root(float v, float eps) {
  return eps >= 1e-30f ? __builtin_amdgcn_rsqf(v) : 1.f / sqrtf(v);
}

// G lanes a head
template <int G, bool kHalfIn, bool kHalfOut>
__global__ void __launch_bounds__(kThreads) head_norm_rope_kernel(RopeArgs a, long long first) {
  const int lane = threadIdx.x & (kWave - 1);
  const long long wave =
      first + (long long)blockIdx.x * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const long long token = wave / a.parts;
  const int unit = lane & (G - 1);
  // turns a position, of every pair: once a workgroup
  __shared__ double speed[kMostHead / 2];
  for (int i = threadIdx.x; i < a.n_rot / 2; i += kThreads) {
    const double v = a.turn * exp2(a.log_step * (double)i);
    speed[i] = a.factors != nullptr ? v / (double)a.factors[i] : v;
  }
  constexpr int kAtOnce = kWave / G;

  // where this lane's two groups of four lie in a head, and how many of each are there
  int at0, at1, n0, n1;
  const bool turned = unit < a.pair_units;
  if (unit >= a.units) {
    at0 = at1 = n0 = n1 = 0;
  } else if (!turned) {
    at0 = a.n_rot + 8 * (unit - a.pair_units);
    at1 = at0 + 4;
    n0 = min(4, a.d - at0);
    n1 = max(0, min(4, a.d - at1));
  } else if (a.neighbours) {
    at0 = 8 * unit;
    at1 = at0 + 4;
    n0 = min(4, a.n_rot - at0);
    n1 = max(0, min(4, a.n_rot - at1));
  } else {
    at0 = 4 * unit;
    at1 = at0 + a.n_rot / 2;
    n0 = n1 = min(4, a.n_rot / 2 - at0);
  }

  // passes of kAtOnce heads: those of the queries, then those of the keys
  const int q_passes = (a.q.n + kAtOnce - 1) / kAtOnce, passes = q_passes + (a.k.n + kAtOnce - 1) / kAtOnce;
  const int sub = lane / G;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  auto load = [&](int pass) {
    if (pass >= passes || token >= a.tokens) return;
    const bool is_k = pass >= q_passes;  // the wave's
    const Heads& s = is_k ? a.k : a.q;
    const int head = (is_k ? pass - q_passes : pass) * kAtOnce;
    if (head + sub >= s.n) return;
    const uint8_t* row = s.x + token * s.x_token + head * s.x_head + sub * s.x_head;
    load4<kHalfIn>(row, at0, n0, x);
    load4<kHalfIn>(row, at1, n1, x + 4);
  };
  int pass = (int)(wave - token * a.parts);
  load(pass);

  float wq[8], wk[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) wq[e] = wk[e] = 1.f;
  if (a.q.weight != nullptr) {
    load4<false>(reinterpret_cast<const uint8_t*>(a.q.weight), at0, n0, wq);
    load4<false>(reinterpret_cast<const uint8_t*>(a.q.weight), at1, n1, wq + 4);
  }
  if (a.k.weight != nullptr) {
    load4<false>(reinterpret_cast<const uint8_t*>(a.k.weight), at0, n0, wk);
    load4<false>(reinterpret_cast<const uint8_t*>(a.k.weight), at1, n1, wk + 4);
  }

  __syncthreads();
  if (token >= a.tokens) return;
  float c[4], s[4];
  if (turned) {
    const double p = (double)a.positions[token];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      double t = p * speed[min(4 * unit + e, a.n_rot / 2 - 1)];
      t -= rint(t);
      sincospif(2.f * (float)t, &s[e], &c[e]);  // half turns, -1 to 1
      c[e] *= a.magnitude;
      s[e] *= a.magnitude;
    }
  }

  for (; pass < passes; pass += a.parts) {
    const bool is_k = pass >= q_passes;
    const Heads& o = is_k ? a.k : a.q;
    const int head = (is_k ? pass - q_passes : pass) * kAtOnce;
    if (is_k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) wq[e] = wk[e];
    }
    float f = 1.f;
    if (a.normed) {
      float q = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) q = fmaf(x[e], x[e], q);
      q = lanes_sum<G>(q);
      f = inverse_root(q * a.per_value + a.eps, a.eps);
    }
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e] * f * wq[e];
    load(pass + a.parts);
    if (turned) {
      if (a.neighbours) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = y[2 * e], v = y[2 * e + 1];
          y[2 * e] = u * c[e] - v * s[e];
          y[2 * e + 1] = u * s[e] + v * c[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = y[e], v = y[e + 4];
          y[e] = u * c[e] - v * s[e];
          y[e + 4] = u * s[e] + v * c[e];
        }
      }
    }
    if (head + sub < o.n) {
      uint8_t* row = o.y + token * o.y_token + head * o.y_head + sub * o.y_head;
      store4<kHalfOut>(row, at0, n0, y);
      store4<kHalfOut>(row, at1, n1, y + 4);
    }
  }
}

template <int G, bool kHalfIn, bool kHalfOut>
void launch_g(const RopeArgs& a) {
  const int64_t waves = a.tokens * a.parts, most = kMostGroups * (kThreads / kWave);
  for (int64_t first = 0; first < waves; first += most) {
    const int64_t n = std::min(waves - first, most);
    head_norm_rope_kernel<G, kHalfIn, kHalfOut>
        <<<dim3((unsigned)((n + kThreads / kWave - 1) / (kThreads / kWave))), kThreads, 0, current_stream()>>>(a, first);
    check_launch("head_norm_rope_kernel");
  }
}
template <bool kHalfIn, bool kHalfOut>
void launch_io(const RopeArgs& a, int g) {
  switch (g) {
    case 8: launch_g<8, kHalfIn, kHalfOut>(a); break;
    case 16: launch_g<16, kHalfIn, kHalfOut>(a); break;
    case 32: launch_g<32, kHalfIn, kHalfOut>(a); break;
    default: launch_g<64, kHalfIn, kHalfOut>(a); break;
  }
}

hipError_t fail(hipError_t e) {
  set_error(e);
  return e;
}

bool heads_of(const weft_ggml_tensor* t, int64_t d, int64_t tokens, size_t unit) {
  return t->ne[0] == d && t->ne[2] == tokens && t->ne[1] > 0 && t->ne[1] <= (1 << 28) && t->ne[3] == 1 && t->nb[0] == unit &&
         t->nb[1] % unit == 0 && t->nb[2] % unit == 0 && t->nb[1] < ((size_t)1 << 40) && t->nb[2] < ((size_t)1 << 40) &&
         aligned(t->data, unit);
}
bool vector_of(const weft_ggml_tensor* t, int64_t n) {
  return t->ne[0] == n && t->ne[1] == 1 && t->ne[2] == 1 && t->ne[3] == 1 && t->nb[0] == 4 && t->data != nullptr &&
         aligned(t->data, 4);
}

hipError_t head_norm_rope(const weft_ggml_tensor* q, const weft_ggml_tensor* k, const weft_ggml_tensor* q_dst,
                          const weft_ggml_tensor* k_dst, const weft_ggml_tensor* positions, const weft_ggml_head_rope* r,
                          bool normed, float eps, const weft_ggml_tensor* q_weight, const weft_ggml_tensor* k_weight,
                          const weft_ggml_tensor* factors) {
  if (q == nullptr || q_dst == nullptr || r == nullptr || (k == nullptr) != (k_dst == nullptr))
    return fail(hipErrorInvalidValue);
  for (const weft_ggml_tensor* t : {q, k, q_dst, k_dst})
    if (t != nullptr && t->type != WEFT_GGML_TYPE_F32 && t->type != WEFT_GGML_TYPE_F16) return fail(hipErrorNotSupported);
  for (const weft_ggml_tensor* t : {q_weight, k_weight, factors})
    if (t != nullptr && t->type != WEFT_GGML_TYPE_F32) return fail(hipErrorNotSupported);
  if (positions != nullptr && positions->type != WEFT_GGML_TYPE_I32) return fail(hipErrorNotSupported);
  if (k != nullptr && (k->type != q->type || k_dst->type != q_dst->type)) return fail(hipErrorNotSupported);
  const int64_t d = q->ne[0], tokens = q->ne[2];
  if (d < 1 || tokens < 0 || tokens > INT32_MAX) return fail(hipErrorInvalidValue);
  if (d > kMostHead) return fail(hipErrorNotSupported);
  if (r->n_rot < 0 || r->n_rot > d || r->n_rot % 2) return fail(hipErrorInvalidValue);
  if (normed ? !(eps >= 0.f) : (q_weight != nullptr || k_weight != nullptr)) return fail(hipErrorInvalidValue);
  if (r->n_rot > 0 && (!(r->base > 0) || !std::isfinite(r->base) || !std::isfinite(r->scale) || !std::isfinite(r->magnitude)))
    return fail(hipErrorInvalidValue);
  const size_t in = q->type == WEFT_GGML_TYPE_F32 ? 4 : 2, out = q_dst->type == WEFT_GGML_TYPE_F32 ? 4 : 2;
  if (!heads_of(q, d, tokens, in) || !heads_of(q_dst, d, tokens, out) || q_dst->ne[1] != q->ne[1])
    return fail(hipErrorInvalidValue);
  if (k != nullptr && (!heads_of(k, d, tokens, in) || !heads_of(k_dst, d, tokens, out) || k_dst->ne[1] != k->ne[1]))
    return fail(hipErrorInvalidValue);
  if (tokens == 0) return hipSuccess;
  if ((q_weight != nullptr && !vector_of(q_weight, d)) || (k_weight != nullptr && (k == nullptr || !vector_of(k_weight, d))) ||
      (factors != nullptr && (r->n_rot == 0 || !vector_of(factors, r->n_rot / 2))) ||
      (r->n_rot > 0 && (positions == nullptr || !vector_of(positions, tokens))))
    return fail(hipErrorInvalidValue);
  for (const weft_ggml_tensor* t : {q, k, q_dst, k_dst})
    if (t != nullptr && t->data == nullptr) return fail(hipErrorInvalidValue);

  RopeArgs a{};
  const auto view = [](const weft_ggml_tensor* x, const weft_ggml_tensor* y, const weft_ggml_tensor* w) {
    Heads h{};
    h.x = static_cast<const uint8_t*>(x->data);
    h.y = static_cast<uint8_t*>(y->data);
    h.weight = w != nullptr ? static_cast<const float*>(w->data) : nullptr;
    h.x_head = (long long)x->nb[1], h.x_token = (long long)x->nb[2];
    h.y_head = (long long)y->nb[1], h.y_token = (long long)y->nb[2];
    h.n = (int)x->ne[1];
    return h;
  };
  a.q = view(q, q_dst, q_weight);
  if (k != nullptr) a.k = view(k, k_dst, k_weight);
  a.d = (int)d;
  a.n_rot = r->n_rot;
  a.tokens = tokens;
  a.normed = normed;
  a.neighbours = r->neighbours != 0;
  a.eps = eps;
  a.per_value = 1.f / (float)d;
  if (r->n_rot > 0) {
    a.positions = static_cast<const int32_t*>(positions->data);
    a.factors = factors != nullptr ? static_cast<const float*>(factors->data) : nullptr;
    a.turn = r->scale / (2.0 * 3.14159265358979323846);
    a.log_step = -2.0 * std::log2(r->base) / r->n_rot;
    a.magnitude = (float)r->magnitude;
  }
  a.pair_units = (r->n_rot / 2 + 3) / 4;
  a.units = a.pair_units + (int)((d - r->n_rot + 7) / 8);
  int g = 8;
  while (g < a.units) g *= 2;
  // A token's heads go to as many waves as there are passes over them, until a launch has 4096 waves,
  // and past that to as many as leave each five passes or more: 16384 tokens of 18 passes 140 us in one wave, 134 in
  // three of six, 145 in four of four and five; 8192 tokens 86 in one and 73; 2116 of 16 passes 36 and 22.5.
  const int at_once = kWave / g;
  const int passes = (a.q.n + at_once - 1) / at_once + (a.k.n + at_once - 1) / at_once;
  a.parts = (int)std::max<int64_t>(1, std::min<int64_t>(passes, std::max<int64_t>(4096 / tokens, passes / 5)));
  if (in == 2 && out == 2)
    launch_io<true, true>(a, g);
  else if (in == 2)
    launch_io<true, false>(a, g);
  else if (out == 2)
    launch_io<false, true>(a, g);
  else
    launch_io<false, false>(a, g);
  return pending_error();
}

}  // namespace
}  // namespace weft

extern "C" int weft_ggml_head_norm_rope(const weft_ggml_tensor* q, const weft_ggml_tensor* k,
                                        const weft_ggml_tensor* q_dst, const weft_ggml_tensor* k_dst,
                                        const weft_ggml_tensor* positions, const weft_ggml_head_rope* rope,
                                        int32_t normed, float eps, const weft_ggml_tensor* q_weight,
                                        const weft_ggml_tensor* k_weight, const weft_ggml_tensor* factors) {
  return (int)weft::head_norm_rope(q, k, q_dst, k_dst, positions, rope, normed != 0, eps, q_weight, k_weight, factors);
}
