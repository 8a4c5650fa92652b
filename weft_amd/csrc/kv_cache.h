// The paged key / value cache: what its writer, its reader and the attention
// over it share.
//
// A pool holds pages of page_size slots, every slot one token's values of one
// kv head as records (F16, Q8_0 or Q4_0 rows of `d` values) at byte strides
// between slots, heads and pages.  Sequence s's token at position p lies in
// page pages[s][p / page_size], slot p % page_size.  The table, the starts and
// the lengths are read on the device, so a call needs no host copy of them; an
// entry that names no page of the pool (a page that was given back) makes its
// slots absent: nothing is written there, they read as zeros, and no query
// sees them.
#pragma once

#include "weft_common.h"
#include "weft_hip.h"

namespace weft {

enum KvType { kKvF16 = 0, kKvQ8_0 = 1, kKvQ4_0 = 2 };

template <int T>
struct KvRecord;  // bytes of 32 values
template <>
struct KvRecord<kKvF16> {
  static constexpr int kBytes = 64;
};
template <>
struct KvRecord<kKvQ8_0> {
  static constexpr int kBytes = kQ8_0Bytes;
};
template <>
struct KvRecord<kKvQ4_0> {
  static constexpr int kBytes = kQ4_0Bytes;
};

struct KvPool {
  uint8_t* data;
  long long slot, head, page;  // byte strides
};

struct KvSeqs {
  const int32_t* pages;    // [n_seqs][max_pages], rows pages_row entries apart
  const int32_t* starts;   // [n_seqs + 1]
  const int32_t* lengths;  // [n_seqs]
  long long pages_row;
  int n_seqs, max_pages, n_tokens;
  int page_size, page_shift, n_pages;  // page_shift: log2(page_size), or -1
};

// Page id and slot of position pos (>= 0) of a sequence; false where the
// position is past the table or its entry names no page.
__device__ __forceinline__ bool kv_place(const KvSeqs& s, int seq, int pos, int& page, int& slot) {
  int entry;
  if (s.page_shift >= 0) {
    entry = pos >> s.page_shift;
    slot = pos & (s.page_size - 1);
  } else {
    entry = (int)((uint32_t)pos / (uint32_t)s.page_size);
    slot = pos - entry * s.page_size;
  }
  page = -1;
  if (entry < s.max_pages) page = s.pages[(long long)seq * s.pages_row + entry];
  return (uint32_t)page < (uint32_t)s.n_pages;
}

// The sequence that new token t (wave-uniform) belongs to, -1 for none; the
// whole wave calls it, 64 starts a step.  Starts count as in the attention: one below
// one before it as that one, so t's is the first sequence that ends past it.
__device__ __forceinline__ int kv_sequence_of(const KvSeqs& s, int t) {
  const int lane = threadIdx.x & (kWave - 1);
  int n = 0;
  for (int i = 0; i < s.n_seqs; i += kWave) {
    const bool past = i + lane < s.n_seqs && s.starts[i + lane + 1] <= t;
    const unsigned long long left = ~__ballot(past);
    n += left ? __builtin_ctzll(left) : kWave;
    if (left) break;
  }
  if (n >= s.n_seqs || s.starts[0] > t) return -1;
  return n;
}

// Position of new token t of its sequence: its new tokens are its last ones, those
// past the call's rows left out.  Negative where a length is shorter than the new
// tokens; past the table where a length says so (kv_place refuses it).
__device__ __forceinline__ long long kv_position(const KvSeqs& s, int seq, int t) {
  return (long long)s.lengths[seq] - min(s.starts[seq + 1], s.n_tokens) + t;
}

// ---------------------------------------------------------------- host side
int kv_type_of(int32_t ggml_type);           // -1: no cache type
size_t kv_row_bytes(int kv_type, int64_t d);  // d a multiple of 32

// Checks a batch against a pair of pools (types, shapes, strides, alignment)
// and fills the kernels' views; hipSuccess, hipErrorInvalidValue or
// hipErrorNotSupported.  d and heads come from the pools.
struct KvView {
  KvSeqs seqs;
  KvPool k, v;
  int type;
  int d, heads;
};
hipError_t kv_view(const weft_ggml_tensor* k_cache, const weft_ggml_tensor* v_cache,
                   const weft_ggml_kv_batch* batch, KvView* out);

}  // namespace weft
