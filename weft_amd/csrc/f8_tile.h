// What the product kernels of 8-bit floats share: operand types, loads into LDS, tiles.
#pragma once

#include "f8.h"

namespace weft {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr;

struct __attribute__((packed, aligned(1))) Bytes16 {
  uint32_t w[4];
};

__device__ __forceinline__ uint4 codes16(const uint8_t* at) {
  const Bytes16 r = *reinterpret_cast<const Bytes16*>(at);
  return {r.w[0], r.w[1], r.w[2], r.w[3]};
}
// The 16 codes of a row of k from `at` on, zeros behind its end; without branches of lanes, so that
// several of these do not wait for each other.  Rows of 16 and more: the 16 bytes that end with the row,
// moved down.
__device__ __forceinline__ uint4 codes16(const uint8_t* row, int at, int k) {
  if (k >= 16) {
    const int from = min(at, k - 16), s = at - from;
    const uint4 v = codes16(row + from);
    const uint64_t first = (uint64_t)v.y << 32 | v.x, last = (uint64_t)v.w << 32 | v.z;
    const uint64_t a = s & 8 ? last : first, b = s & 8 ? 0 : last;
    const int n = 8 * (s & 7);
    const uint64_t lo = s < 16 ? a >> n | b << 1 << (63 - n) : 0, hi = s < 16 ? b >> n : 0;
    return {(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint32_t c = row[min(at + e, k - 1)];
    w[e / 4] |= at + e < k ? c << (8 * (e & 3)) : 0;
  }
  return {w[0], w[1], w[2], w[3]};
}

// 16 (4) bytes per lane from global straight into LDS: lane l writes [lds + 16 l, +16)
// ([lds + 4 l, +4)).  The kernel waits itself; nothing else in it uses M0.
__device__ __forceinline__ void dma16(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void dma16(const uint8_t* at, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(at)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(const float* at, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               :
               : "s"(lds), "v"(at)
               : "memory", "m0");
}
// The wave's own loads but the last N have arrived and its LDS reads are done; then all waves'.
template <int N>
__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
}

// the e4m3 numbers of eight codes
__device__ __forceinline__ half8 halves(int lo, int hi) {
  const half2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  const half2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const half2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  const half2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Tile t of tiles_m x tiles_n.  Workgroup b runs on XCD b % 8, so consecutive tiles are given
// to one XCD; they are bands of eight token tiles, one weight tile after the other, so that
// an XCD's 32 workgroups read 8 + 4 tiles through its L2.
__device__ __forceinline__ void place(int b, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int tiles = tiles_m * tiles_n, each = tiles / 8, rest = tiles % 8, x = b % 8;
  int t = x * each + min(x, rest) + b / 8;
  const int band = t / (8 * tiles_n);
  t -= band * 8 * tiles_n;
  const int wide = min(8, tiles_m - 8 * band);
  tn = t / wide;
  tm = 8 * band + t - tn * wide;
}

// Four weights n .. n + 3 of a token's row y, those before `end`.
__device__ __forceinline__ void store_weights(uint8_t* y, int n, int end, bool half_out, v4f v) {
  if (half_out) {
    _Float16* q = reinterpret_cast<_Float16*>(y) + n;
    const half4 w = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    if (n + 3 < end && (reinterpret_cast<uintptr_t>(q) & 7u) == 0) {
      *reinterpret_cast<half4*>(q) = w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < end) q[e] = w[e];
    }
  } else {
    float* q = reinterpret_cast<float*>(y) + n;
    if (n + 3 < end && (reinterpret_cast<uintptr_t>(q) & 15u) == 0) {
      *reinterpret_cast<v4f*>(q) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < end) q[e] = v[e];
    }
  }
}

// A tile's output by way of LDS, so that a wave stores whole rows at once: straight from the
// registers a store has 16 or 32 bytes of each of 32 rows (8192 x 8192 outputs of 16 bits 41 us, so
// 29; 2048 x 11008 of 32 bits 16 us of 192).  Rows of TN outputs lie kTileRow bytes apart.
template <int TN, typename Out>
constexpr int kTileRow = TN * (int)sizeof(Out) + 8;
template <int TN, typename Out>
__device__ __forceinline__ void tile_put(uint8_t* lds, int token, int n, float a, float b, float c, float d) {
  struct __attribute__((packed, aligned(8))) Four {
    Out v[4];
  };
  *reinterpret_cast<Four*>(lds + token * kTileRow<TN, Out> + n * (int)sizeof(Out)) = {{(Out)a, (Out)b, (Out)c, (Out)d}};
}
template <int TN, int TM, int kThreads, typename Out>
__device__ __forceinline__ void tile_store(const uint8_t* lds, const F8Product& p, int n0, int m0) {
  constexpr int kEach = 8 / sizeof(Out), kUnits = TN / kEach;
  static_assert(kThreads % kUnits == 0, "whole rows");
  struct __attribute__((packed, aligned(8))) Unit {
    Out v[kEach];
  };
  const int unit = threadIdx.x % kUnits, n = n0 + unit * kEach;
  const bool whole = n + kEach <= p.n && (reinterpret_cast<uintptr_t>(p.y) & 7u) == 0 && (p.y_row & 7) == 0;
  for (int t = threadIdx.x / kUnits; t < min(TM, p.m - m0); t += kThreads / kUnits) {
    const Unit v = *reinterpret_cast<const Unit*>(lds + t * kTileRow<TN, Out> + 8 * unit);
    Out* y = reinterpret_cast<Out*>(p.y + (long long)(m0 + t) * p.y_row) + n;
    if (whole) {
      *reinterpret_cast<Unit*>(y) = v;
    } else {
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (n + e < p.n) y[e] = v.v[e];
    }
  }
}

}  // namespace weft
