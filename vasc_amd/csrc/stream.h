// Shared by the streaming operators (rotary.hip, cache.hip, cache_attn.hip).
#pragma once

#include "../../include/vasc_stream.h"
#include "common.h"

namespace vasc {

typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kPage = 64;  // tokens of a cache page

__device__ __forceinline__ float to_f32(__bf16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float to_f32(_Float16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float to_f32(float x) { return x; }
// Round to nearest even (the hardware conversions).
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  return static_cast<T>(x);
}

// Place of token t of a page in vc's last dimension, ks and vs.
__device__ __forceinline__ int page_place(int t) { return ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3); }

// 2^(byte - 127); byte 255 gives infinity, which times a zero code is NaN.
__device__ __forceinline__ float pow2_byte(uint32_t byte) { return __uint_as_float(byte << 23); }

// Tokens of sequence b that its page table can hold.
__device__ __forceinline__ int64_t clamp_tokens(int64_t n, int64_t max_pages) {
  return n < 0 ? 0 : (n < max_pages * kPage ? n : max_pages * kPage);
}

// The pages that one unit of queries sees: logical pages [0, seen), of which those from `own` on hold the rows' own
// positions (causal) or are the last one. Tokens [t0, t1) of the sequence's n_q queries; length L.
struct UnitView {
  int64_t seen;  // pages
  int64_t own;   // first of the pages that are always among the last
};
__device__ __forceinline__ UnitView unit_view(int64_t L, int64_t n_q, int64_t t0, int64_t t1, int64_t max_pages, bool causal) {
  UnitView v;
  if (t1 <= t0) return {0, 0};
  const int64_t cut = clamp_tokens(L, max_pages);
  if (!causal) {
    v.seen = cdiv(cut, kPage);
    v.own = v.seen - 1;
  } else {
    const int64_t last = L - n_q + t1, first = L - n_q + t0;  // one past the last row's position; the first row's
    const int64_t keys = last < cut ? last : cut;
    v.seen = keys > 0 ? cdiv(keys, kPage) : 0;
    v.own = first > 0 ? first / kPage : 0;
  }
  return v;
}

}  // namespace vasc
