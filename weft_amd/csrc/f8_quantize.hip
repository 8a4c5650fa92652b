// Quantizing rows, and blocks of weights, to 8-bit floats (f8.h has the formula).
//
// Both are one pass bound by memory.  Rows: 16 lanes a block of 128 values, eight a lane, so
// the block's maximum is four lane exchanges within a row of 16 and memory is read once.
// 2048 rows of 11008 16-bit values take 13.8 us (4.9 TB/s); up to some hundred rows the launch
// is what takes the time (509 rows 5.3, one of 4096 3.8).
// Weights: a workgroup a block of 128 x 128, its 64 values a thread in registers between the
// maximum and the codes.  11008 x 4096 32-bit values take 42 us (5.4 TB/s), 11008 x 4101, where every
// access is unaligned, 47 (4.8 TB/s), 4096 x 11008 16-bit ones 27 (5.0 TB/s).
#include <algorithm>

#include "f8.h"
#include "runtime.h"

namespace weft {
namespace {

constexpr int kThreads = 256;
// A launch has fewer than 2^32 threads: past that the runtime starts the rest of the
// division, without an error.
constexpr int64_t kMostGroups = ((int64_t)1 << 31) / kThreads;

struct __attribute__((packed, aligned(1))) Codes8 {
  uint2 w;
};
// eight codes of which those before `end` are stored
__device__ __forceinline__ void store_codes(uint8_t* row, int i, int end, uint2 codes) {
  if (i + 8 <= end) {
    reinterpret_cast<Codes8*>(row + i)->w = codes;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < end) row[i + e] = (uint8_t)((e < 4 ? codes.x : codes.y) >> (8 * (e & 3)));
  }
}

struct QuantizeArgs {
  const uint8_t* x;
  uint8_t* y;
  float* scales;
  long long x_row, y_row, s_row, s_block;
  long long groups;  // blocks of 128 values: rows x blocks of a row
  int k, wide, blocks;
  bool shared_lines;  // rows do not begin with a line, so neighbouring blocks share lines
};

// The place of a workgroup of weights in its launch.  Workgroups go to the XCDs in turn and each
// XCD has its own L2.  Where neighbouring blocks share lines of memory, kNear of them go to
// one XCD, so that most lines are written whole: 11008 x 4101 32-bit values 57.6 -> 46.8 us,
// 16-bit ones 43.7 -> 33.8; without shared lines it costs 1 to 4 % (11008 x 4096 42.0 -> 43.3).  The
// rows' kernel gains nothing from it: its workgroups are 16 blocks long.
constexpr uint32_t kNear = 16;
__device__ __forceinline__ uint32_t group_of(bool shared_lines) {
  const uint32_t b = blockIdx.x, window = b / (8 * kNear);
  if (!shared_lines || window == gridDim.x / (8 * kNear)) return b;
  return window * (8 * kNear) + b % 8 * kNear + b / 8 % kNear;
}

template <bool kHalf>
__global__ void __launch_bounds__(kThreads) f8_quantize_rows_kernel(QuantizeArgs a) {
  const int part = threadIdx.x & 15;
  const long long g = (long long)blockIdx.x * (kThreads / 16) + threadIdx.x / 16;
  if (g >= a.groups) return;
  const long long row = g / a.blocks;
  const int block = (int)(g - row * a.blocks);
  const int i = block * kF8Block + 8 * part;
  float x[8];
  f8_load8<kHalf>(a.x + row * a.x_row, i, a.k, x);
  float scale;
  const uint2 codes = f8_quantize_16lanes(x, scale);
  store_codes(a.y + row * a.y_row, i, a.wide, codes);
  if (part == 0) a.scales[row * a.s_row + block * a.s_block] = scale;
}

template <bool kHalf>
__global__ void __launch_bounds__(kThreads) f8_quantize_blocks_kernel(QuantizeArgs a, long long rows, long long first) {
  __shared__ float most[kThreads / kWave];
  const int part = threadIdx.x & 15, sub = threadIdx.x / 16;
  const long long g = first + group_of(a.shared_lines);
  const long long band = g / a.blocks;
  const int block = (int)(g - band * a.blocks);
  const int i = block * kF8Block + 8 * part;
  float x[8][8];
  float m = 0.f;
  // A whole block's loads have no branches of lanes between them, so they do not wait for each
  // other (4096 x 11008 16-bit values 34 us without this, 27 with it).
  if ((band + 1) * kF8Block <= rows && (block + 1) * kF8Block <= a.k) {
#pragma unroll
    for (int p = 0; p < 8; ++p)
      f8_load8<kHalf>(a.x + (band * kF8Block + 16 * p + sub) * a.x_row, i, i + 8, x[p]);
  } else {
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const long long row = band * kF8Block + 16 * p + sub;
      if (row < rows) {
        f8_load8<kHalf>(a.x + row * a.x_row, i, a.k, x[p]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[p][e] = 0.f;
      }
    }
  }
#pragma unroll
  for (int p = 0; p < 8; ++p)
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, f8_finite_abs(x[p][e]));
  m = wave_max_nonneg(m);
  if ((threadIdx.x & (kWave - 1)) == 0) most[threadIdx.x / kWave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
  const F8Scale s = f8_scale(m);
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const long long row = band * kF8Block + 16 * p + sub;
    if (row >= rows) continue;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = f8_scaled(x[p][e], s.factor);
    store_codes(a.y + row * a.y_row, i, a.wide, make_uint2(f8_pack4(y[0], y[1], y[2], y[3]), f8_pack4(y[4], y[5], y[6], y[7])));
  }
  if (threadIdx.x == 0) a.scales[band * a.s_row + block * a.s_block] = s.scale;
}

bool share_lines(const QuantizeArgs& a) {
  return reinterpret_cast<uintptr_t>(a.y) % kF8Block != 0 || a.y_row % kF8Block != 0;
}

void quantize_blocks(QuantizeArgs a, bool half, int64_t rows) {
  for (int64_t first = 0; first < a.groups; first += kMostGroups) {
    const dim3 grid((unsigned)std::min<int64_t>(a.groups - first, kMostGroups));
    if (half)
      f8_quantize_blocks_kernel<true><<<grid, kThreads, 0, current_stream()>>>(a, rows, first);
    else
      f8_quantize_blocks_kernel<false><<<grid, kThreads, 0, current_stream()>>>(a, rows, first);
    check_launch("f8_quantize_blocks_kernel");
  }
}

hipError_t fail(hipError_t e) {
  set_error(e);
  return e;
}

hipError_t quantize(const weft_ggml_tensor* x, const weft_ggml_tensor* codes, const weft_ggml_tensor* scales) {
  if (x == nullptr || codes == nullptr || scales == nullptr) return fail(hipErrorInvalidValue);
  if ((x->type != WEFT_GGML_TYPE_F32 && x->type != WEFT_GGML_TYPE_F16) || codes->type != WEFT_GGML_TYPE_F8_E4M3 ||
      scales->type != WEFT_GGML_TYPE_F32)
    return fail(hipErrorNotSupported);
  const bool half = x->type == WEFT_GGML_TYPE_F16;
  const size_t unit = half ? 2 : 4;
  const int64_t k = x->ne[0], rows = x->ne[1];
  if (k < 0 || rows < 0 || k > INT32_MAX / 2 || rows > INT32_MAX) return fail(hipErrorInvalidValue);
  const bool per_row = scales->ne[1] == rows;
  for (const weft_ggml_tensor* t : {x, codes, scales})
    if (t->ne[2] != 1 || t->ne[3] != 1) return fail(hipErrorInvalidValue);
  if (codes->ne[0] != k || codes->ne[1] != rows || scales->ne[0] != f8_blocks(k) ||
      (!per_row && scales->ne[1] != f8_blocks(rows)))
    return fail(hipErrorInvalidValue);
  if (x->nb[0] != unit || x->nb[1] % unit || !aligned(x->data, unit) || codes->nb[0] != 1 || scales->nb[0] % 4 ||
      scales->nb[1] % 4 || !aligned(scales->data, 4))
    return fail(hipErrorInvalidValue);
  if (k == 0 || rows == 0) return hipSuccess;
  if (x->data == nullptr || codes->data == nullptr || scales->data == nullptr) return fail(hipErrorInvalidValue);
  QuantizeArgs a{};
  a.x = static_cast<const uint8_t*>(x->data);
  a.y = static_cast<uint8_t*>(codes->data);
  a.scales = static_cast<float*>(scales->data);
  a.x_row = (long long)x->nb[1];
  a.y_row = (long long)codes->nb[1];
  a.s_row = (long long)(scales->nb[1] / 4);
  a.s_block = (long long)(scales->nb[0] / 4);
  a.k = (int)k;
  a.wide = (int)k;
  a.blocks = (int)f8_blocks(k);
  if (per_row) {
    f8_quantize_rows(a.x, half, a.x_row, a.y, a.y_row, a.wide, a.scales, a.s_row, a.s_block, rows, a.k);
  } else {
    a.groups = f8_blocks(rows) * a.blocks;
    a.shared_lines = share_lines(a);
    quantize_blocks(a, half, rows);
  }
  return pending_error();
}

}  // namespace

void f8_quantize_rows(const uint8_t* x, bool half, long long x_row, uint8_t* y, long long y_row, int wide,
                      float* scales, long long s_row, long long s_block, int64_t rows, int k) {
  QuantizeArgs a{x, y, scales, x_row, y_row, s_row, s_block, 0, k, wide, (int)f8_blocks(k)};
  // whole rows a launch; a row of 2^30 values is half of the most
  const int64_t most = std::max<int64_t>(1, kMostGroups * (kThreads / 16) / a.blocks);
  for (int64_t r = 0; r < rows; r += most) {
    a.groups = std::min(rows - r, most) * a.blocks;
    const dim3 grid((unsigned)((a.groups + kThreads / 16 - 1) / (kThreads / 16)));
    if (half)
      f8_quantize_rows_kernel<true><<<grid, kThreads, 0, current_stream()>>>(a);
    else
      f8_quantize_rows_kernel<false><<<grid, kThreads, 0, current_stream()>>>(a);
    check_launch("f8_quantize_rows_kernel");
    a.x += most * a.x_row;
    a.y += most * a.y_row;
    a.scales += most * a.s_row;
  }
}

}  // namespace weft

extern "C" int weft_ggml_quantize_f8(const weft_ggml_tensor* x, const weft_ggml_tensor* codes,
                                     const weft_ggml_tensor* scales) {
  return (int)weft::quantize(x, codes, scales);
}
