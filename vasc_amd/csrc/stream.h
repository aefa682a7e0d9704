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

// Place of token t of a page in vc's last dimension and in vs: a lane group's four tokens of each 16 lie together.
__device__ __forceinline__ int page_place(int t) { return ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3); }
// Its place in ks: a lane's four keys, one of each 16, are the bytes of a word.
__device__ __forceinline__ int key_place(int t) { return (t & 15) * 4 + (t >> 4); }

// Four floats -> four e4m3 codes, rounded to nearest even (|x| <= 448).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  return static_cast<uint32_t>(r);
}

__device__ __forceinline__ void unpack_e4m3(uint32_t w, float (&f)[4]) {
  const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const floatx2 b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
}

// Smallest e in [least, most] with top <= 448 * 2^e (`most` where none is).
__device__ __forceinline__ int power_of(float top, int least, int most) {
  const uint32_t u = __float_as_uint(top);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, least), most);
}

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
