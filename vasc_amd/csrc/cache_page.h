// Shared by the writing, reading and moving of cache pages (cache.hip, cache4.hip, pages.hip): a call's tokens, and the
// page of a workgroup.
#pragma once

#include "stream.h"

namespace vasc {
namespace {

struct CacheArgs {
  uint8_t *kc, *vc, *ks, *vs;
  uint16_t *mean;
  int64_t pages;
  const int32_t *table;
  int64_t table_stride, max_pages;
  uint8_t *vo;  // of the 4-bit cache
};

struct RowArgs {
  const void *k, *v;  // read: the outputs
  int64_t ksb, ksh, kst, vsb, vsh, vst;
  const int32_t *start, *count;
  int64_t B, H, T;
  int span;  // pages that T tokens can touch
};

// 16 bytes of a tensor that is read once; kPast: past the caches.
template <bool kPast>
__device__ __forceinline__ u32x4 load16(const u32x4 *from) {
  if constexpr (kPast) return __builtin_nontemporal_load(from);
  else return *from;
}

// The rows to be written into a cache are read past the caches (kPast), in half types whatever their number. Measured, 16 heads
// of 64, in us with plain loads and so: two products that make the rows and the write after them, 1041 tokens 11.8 and 11.8,
// 4164 22.3 and 21.1, 16656 44.7 and 45.1, 33312 84.4 and 82.9; 32 frames that are in no cache 73 and 70 with the read back.
// A lane's eight floats are two loads, each of half of every 32 bytes, which fetch a line twice: float32 rows go past the
// caches from 256 MB on, where these have lost them anyway: 34 MB 27 and 30, 68 MB 40.5 and 48, 136 MB 75 and 81, 273 MB 155
// and 153.5, 546 MB 317 and 310; rows that are in no cache, with 100 us for emptying these, 123 and 115, 148 and 133, 194 and
// 166, 260 and 236 from 68 MB on.
bool floats_past(const RowArgs &r, int64_t D) { return r.B * r.H * r.T * D * 8 >= int64_t(1) << 28; }

// Eight consecutive elements as floats.
template <bool kPast, typename T>
__device__ __forceinline__ void load8(const T *src, float (&x)[8]) {
  struct alignas(16) Eight { T v[8]; };
  const u32x4 *from = reinterpret_cast<const u32x4 *>(src);
  const u32x4 a = load16<kPast>(from);
  Eight e;
  if constexpr (sizeof(T) == 2) {
    e = __builtin_bit_cast(Eight, a);
  } else {
    typedef uint32_t words __attribute__((ext_vector_type(8)));
    const u32x4 b = load16<kPast>(from + 1);
    e = __builtin_bit_cast(Eight, words{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(e.v[i]);
}

// Rows that are read back are mostly used at once, and go past the caches (kPast) only where these would hardly hold them:
// where the two outputs have 128 MB, half the cache behind HBM, which the codes and what is made of the rows want as well.
// Measured (8 bits, 16 heads of 64), in us with plain stores and past the caches, the read and the sum k + v after it: one token
// 5.8 and 6.4, 1041 tokens 8.8 and 9.4, 4164 15.6 and 16.0 (8 heads of 128: 16.6 and 16.3). Larger outputs, again and again
// and after a fill of 100 us that empties the caches: 68 MB 34 and 36, 136 and 148; 98 MB 46 and 50, 155 and 170; 136 MB 71
// and 65, 176 and 199; 205 MB 104 and 113, 217 and 233; 273 MB 161 and 155, 275 and 275. The read by itself: 98 MB 25 and 24,
// 136 MB 33 and 32.5, 273 MB 87 and 62 (4 bits: 75 and 53). Float32 rows never do: their two stores a lane have half of every
// 32 bytes each, which only the caches join (the read by itself 136 MB 30 and 59, 546 MB 169 and 226, with the sum 321 and 299;
// 4 bits 151 and 229, 305 and 339).
bool halves_past(const RowArgs &r, int64_t D) { return r.B * r.H * r.T * D * 4 >= int64_t(1) << 27; }

template <bool kPast, typename T>
__device__ __forceinline__ void store8(T *dst, const float (&x)[8]) {
  typedef uint32_t words __attribute__((ext_vector_type(sizeof(T) == 4 ? 8 : 4)));
  struct alignas(sizeof(words)) Eight { T v[8]; };
  Eight e;
#pragma unroll
  for (int i = 0; i < 8; ++i) e.v[i] = from_f32<T>(x[i]);
  const words w = __builtin_bit_cast(words, e);
  static_assert(!kPast || sizeof(T) == 2, "float32 rows stay in the caches");
  u32x4 *to = reinterpret_cast<u32x4 *>(dst);
  const u32x4 a = {w[0], w[1], w[2], w[3]};
  if constexpr (kPast) __builtin_nontemporal_store(a, to);
  else *to = a;
  if constexpr (sizeof(T) == 4) to[1] = u32x4{w[4], w[5], w[6], w[7]};
}

struct PageWork {
  int64_t b, h, j;   // sequence, head, logical page
  int64_t pid;       // physical page, or -1
  int64_t s;         // position of the call's first token
  int lo, hi;        // slots of the page that the call's tokens cover
};

// The page of this workgroup: false where the call has no token in it.
__device__ __forceinline__ bool page_work(const CacheArgs &c, const RowArgs &r, int64_t tokens, PageWork &w) {
  const uint32_t id = blockIdx.x, span = r.span, ph = id / span;
  const int64_t jj = id - ph * span;
  w.b = ph / static_cast<uint32_t>(r.H);
  w.h = ph - static_cast<uint32_t>(w.b) * static_cast<uint32_t>(r.H);
  w.s = r.start[w.b];
  if (w.s < 0) return false;
  w.j = w.s / kPage + jj;
  const int64_t lo = w.s - w.j * kPage, hi = w.s + tokens - w.j * kPage;
  w.lo = static_cast<int>(lo > 0 ? lo : 0);
  w.hi = static_cast<int>(hi < kPage ? hi : kPage);
  if (w.hi <= w.lo) return false;
  w.pid = -1;
  if (w.j < c.max_pages) {
    const int64_t pid = c.table[w.b * c.table_stride + w.j];
    if (pid >= 0 && pid < c.pages) w.pid = pid;
  }
  return true;
}

__device__ __forceinline__ int64_t new_tokens(const RowArgs &r, int64_t b) {
  if (!r.count) return r.T;
  const int64_t n = r.count[b];
  return n < 0 ? 0 : (n < r.T ? n : r.T);
}

// The page of this workgroup of a read of r.T tokens of sequence b; live: whether it holds anything (else its rows are zero).
__device__ __forceinline__ bool read_work(const CacheArgs &c, const RowArgs &r, int64_t b, PageWork &w, bool &live) {
  live = r.start[b] >= 0;
  if (!page_work(c, r, r.T, w)) {
    if (live) return false;
    // a negative start reads nothing: its rows are zero, 64 to a workgroup
    w.s = 0;
    w.j = blockIdx.x % r.span;
    w.h = (blockIdx.x / r.span) % r.H;
    w.b = b;
    w.lo = 0;
    const int64_t hi = r.T - w.j * kPage;
    w.hi = static_cast<int>(hi < kPage ? hi : kPage);
    w.pid = -1;
    if (w.hi <= 0) return false;
  }
  live = live && w.pid >= 0;
  return true;
}

int check_cache(const void *kc, const void *vc, const void *ks, const void *vs, int64_t pages, const int32_t *table,
                int64_t table_stride, int64_t max_pages, int64_t D) {
  VASC_REQUIRE(kc && vc && ks && vs && table, "the cache and the page table are required");
  VASC_REQUIRE(pages > 0 && max_pages > 0, "pages and max_pages must be positive");
  VASC_REQUIRE(max_pages < (int64_t(1) << 24), "max_pages %lld too large", (long long)max_pages);
  VASC_REQUIRE(table_stride >= max_pages || table_stride == 0, "table_stride %lld below max_pages", (long long)table_stride);
  VASC_SUPPORTED(D == 64 || D == 128, "D %lld not built (64, 128)", (long long)D);
  for (const void *x : {kc, vc, ks, vs})
    VASC_REQUIRE((reinterpret_cast<uintptr_t>(x) & 15) == 0, "the cache must be 16-byte aligned");
  return VASC_OK;
}

int check_rows(const char *name, const void *x, int64_t sb, int64_t sh, int64_t st) {
  VASC_REQUIRE(x, "%s is NULL", name);
  VASC_REQUIRE((reinterpret_cast<uintptr_t>(x) & 15) == 0 && sb % 8 == 0 && sh % 8 == 0 && st % 8 == 0,
               "%s needs 16-byte aligned rows and strides that are multiples of 8", name);
  return VASC_OK;
}

// Sizes and type of the tokens; fills r.span.
int check_tokens(RowArgs &r, int32_t dtype) {
  VASC_REQUIRE(r.B > 0 && r.H > 0 && r.T > 0, "empty tensor");
  VASC_SUPPORTED(dtype >= 0 && dtype <= 2, "dtype %d not built", dtype);
  VASC_REQUIRE(r.T < (int64_t(1) << 30), "too many tokens");
  r.span = static_cast<int>((r.T + 2 * kPage - 2) / kPage);
  VASC_REQUIRE(r.H < (1 << 16) && r.B < (int64_t(1) << 24) && r.B * r.H * r.span < (int64_t(1) << 31), "too many tokens");
  return VASC_OK;
}

}  // namespace
}  // namespace vasc
