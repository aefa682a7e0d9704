// The 4-bit block cache: writing tokens into it and reading them back.
//
// A row of k or v is held in groups of 32 features, e2m1 codes times a power of two, 17/32 bytes a value and a bit more
// (value rows: a byte for the row's largest group, half a byte a group for what it lies below that, so that attention takes
// the row's power into the softmax and the rest into the widened values). The power is the smallest with max <= 7 * 2^e: 7
// is as far from 6 as a value of that binade may be from its neighbour, so nothing is lost against 6 * 2^e, and a fifth of
// the groups has steps half as wide.
//
// Bound by HBM, as the 8-bit cache (cache.hip), whose division of work it has: one workgroup owns one (page, head) of a
// call, partly covered words are merged with plain loads and stores, and the page's key mean is summed anew from its codes
// in an order that the slots fix.
// Measured (bf16): 32 frames of 1041 tokens, 16 heads of 64, written in 38 us (4.5 TB/s; a large copy reaches 5.1), read back
// in 26 us (6.5 TB/s, partly from the cache behind HBM); one token of 64 sequences, 8 heads of 128, in 7.1 us: the latency of
// table, codes, barrier and merge.
#include "cache_page.h"

namespace vasc {
namespace {

// Eight consecutive elements of a row as they come. Half types stay packed: magnitudes are compared as integers, and the
// conversion takes pairs and the power, so that a value costs two instructions, not ten (the kernel's bound had been those:
// 128 frames of 16 heads of 64 at 89% of what the vector pipes issue).
template <typename T>
struct Eight {
  typedef uint32_t words __attribute__((ext_vector_type(sizeof(T) == 4 ? 8 : 4)));
  words w;

  template <bool kPast>
  __device__ __forceinline__ void load(const T *src) {
    const u32x4 *from = reinterpret_cast<const u32x4 *>(src);
    const u32x4 a = load16<kPast>(from);
    if constexpr (sizeof(T) == 2) {
      w = a;
    } else {
      const u32x4 b = load16<kPast>(from + 1);
      w = words{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }

  // The bits of the largest magnitude, of an infinity or a NaN if there is one.
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 2) {
      typedef uint16_t pair __attribute__((ext_vector_type(2)));
      pair m = {0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = w[i] & 0x7fff7fffu;
        m = __builtin_elementwise_max(m, __builtin_bit_cast(pair, x));
      }
      return max(static_cast<uint32_t>(m[0]), static_cast<uint32_t>(m[1]));
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    }
  }
  static __device__ __forceinline__ bool finite(uint32_t top) {
    return top < (sizeof(T) == 4 ? 0x7f800000u : __is_same(T, __bf16) ? 0x7f80u : 0x7c00u);
  }
  static __device__ __forceinline__ float value(uint32_t top) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(top);
    else if constexpr (__is_same(T, __bf16)) return __uint_as_float(top << 16);
    else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(top)));
  }

  // Over 2^(byte - 127) as e2m1 codes: to nearest, ties to even, at most 6 (the conversion saturates).
  __device__ __forceinline__ uint32_t codes(int byte) const {
    const float power = pow2_byte(byte);
    uint32_t r = 0;
    if constexpr (sizeof(T) == 4) {
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[0]), __uint_as_float(w[1]), power, 0);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[2]), __uint_as_float(w[3]), power, 1);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[4]), __uint_as_float(w[5]), power, 2);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[6]), __uint_as_float(w[7]), power, 3);
    } else if constexpr (__is_same(T, __bf16)) {
      const uint32_t a = w[0], b = w[1], c = w[2], d = w[3];  // copies: a bit cast of an element itself reads element 0
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, a), power, 0);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, b), power, 1);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, c), power, 2);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, d), power, 3);
    } else {
      const uint32_t a = w[0], b = w[1], c = w[2], d = w[3];
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(halfx2, a), power, 0);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(halfx2, b), power, 1);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(halfx2, c), power, 2);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(halfx2, d), power, 3);
    }
    return r;
  }
};

// Max over the four neighbouring lanes of a group.
__device__ __forceinline__ uint32_t group4_max(uint32_t v) {
  v = max(v, xor_lane(v, 1));
  return max(v, xor_lane(v, 2));
}

// Max over the groups of a row, which agree within.
template <int D>
__device__ __forceinline__ int groups_max(int v) {
  v = max(v, xor_lane(v, 4));
  return D == 128 ? max(v, xor_lane(v, 8)) : v;
}

template <typename T, int D, bool kPast>
__global__ __launch_bounds__(256) void cache4_write_kernel(const CacheArgs c, const RowArgs r) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes, kG = D / 32;
  constexpr int kS = kLanes + 1;         // words of a value row in LDS: four rows on, four banks on
  constexpr int kGroups = 256 / kLanes;  // row groups of the mean, eight columns a thread
  __shared__ uint32_t kt[kPage][kLanes];
  __shared__ uint32_t vt[kPage][kS];
  __shared__ uint8_t ke[kPage][kG], vn[kPage][kG];
  __shared__ double part[kGroups][D];
  const int tid = threadIdx.x;
  PageWork w;
  const int64_t b = blockIdx.x / (static_cast<uint32_t>(r.span) * static_cast<uint32_t>(r.H));
  if (!page_work(c, r, new_tokens(r, b), w) || w.pid < 0) return;
  const int64_t ph = w.pid * r.H + w.h;
  uint8_t *kc = c.kc + ph * (kPage * D / 2), *vc = c.vc + ph * (kPage * D / 2);
  uint8_t *ks = c.ks + ph * (kPage * kG), *vs = c.vs + ph * kPage, *vo = c.vo + ph * (kG * 32);
  const int word = tid % kLanes, col = word * 8, gr = col / 32;
  const T *kin = static_cast<const T *>(r.k) + w.b * r.ksb + w.h * r.ksh;
  const T *vin = static_cast<const T *>(r.v) + w.b * r.vsb + w.h * r.vsh;
#pragma unroll
  for (int pass = 0; pass < kPage / kRows; ++pass) {
    const int row = pass * kRows + tid / kLanes;
    if (row < w.lo) {  // held before: its part of the mean
      kt[row][word] = *reinterpret_cast<const uint32_t *>(kc + key4_at<D>(row, col));
      if ((col & 31) == 0) ke[row][gr] = ks[gr * kPage + key_place(row)];
    } else if (row < w.hi) {
      const int64_t t = w.j * kPage + row - w.s;
      Eight<T> x, y;
      x.template load<kPast>(kin + t * r.kst + col);
      y.template load<kPast>(vin + t * r.vst + col);
      const uint32_t ktop = group4_max(x.top()), vtop = group4_max(y.top());
      int kb = power_of<2>(Eight<T>::value(ktop), -60, 60) + 127, vb = power_of<2>(Eight<T>::value(vtop), -60, 60) + 127;
      int row_b = groups_max<D>(vb);
      vb = max(vb, row_b - 14);
      uint32_t kw = 0, vw = 0;
      if (groups_max<D>(Eight<T>::finite(max(ktop, vtop)) ? 0 : 1) == 0) {
        kw = x.codes(kb);
        vw = y.codes(vb);
      } else {
        kb = 255;
        vb = row_b = 127;
      }
      kt[row][word] = kw;
      *reinterpret_cast<uint32_t *>(kc + key4_at<D>(row, col)) = kw;
      vt[row][word] = vw;
      if ((col & 31) == 0) {
        ke[row][gr] = static_cast<uint8_t>(kb);
        ks[gr * kPage + key_place(row)] = static_cast<uint8_t>(kb);
        vn[row][gr] = static_cast<uint8_t>(15 - (row_b - vb));
        if (col == 0) vs[page_place(row)] = static_cast<uint8_t>(row_b);
      }
    }
  }
  __syncthreads();
  // values, transposed: 16 bytes hold a lane group's 16 tokens of two features
  if (tid < 64 * kG) {
    const int g = tid & 3, f = (tid >> 6) * 32 + ((tid >> 2) & 15);
    uint32_t out[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        out[half * 2 + (i >> 3)] |= (vt[token4_of(g, i)][(f >> 3) + half * 2] >> (4 * (f & 7)) & 15u) << (4 * (i & 7));
    u32x4 *at = reinterpret_cast<u32x4 *>(vc + value4_at(f, g));
    u32x4 x = {out[0], out[1], out[2], out[3]};
    if (w.lo > 0 || w.hi < kPage) {  // what the call does not cover stays (and was not in vt)
      uint32_t cover[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (token4_of(g, i) >= w.lo && token4_of(g, i) < w.hi) cover[i >> 3] |= 15u << (4 * (i & 7));
      if (cover[0] | cover[1]) {
        const u32x4 old = *at;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (x[i] & cover[i & 1]) | (old[i] & ~cover[i & 1]);
        *at = x;
      }
    } else {
      *at = x;
    }
  }
  if (tid < 8 * kG) {  // the offsets: a word holds eight tokens of a group
    const int half = tid & 1, grp = (tid >> 1) % kG, g = tid / (2 * kG);
    uint32_t cover = 0, out = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int t = token4_of(g, half * 8 + k);
      if (t < w.lo || t >= w.hi) continue;
      cover |= 15u << offset4_bit(k);
      out |= static_cast<uint32_t>(vn[t][grp]) << offset4_bit(k);
    }
    if (cover) {
      uint32_t *at = reinterpret_cast<uint32_t *>(vo + (g * kG + grp) * 8 + half * 4);
      if (cover != 0xffffffffu) out |= *at & ~cover;
      *at = out;
    }
  }
  // the page's key mean, in an order that the slots fix: a group of threads takes every kGroups-th row
  {
    const int grp = tid / kLanes;
    double s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int row = grp; row < w.hi; row += kGroups) {
      float f[8];
      unpack_e2m1(kt[row][word], f, pow2_byte(ke[row][gr]));
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += static_cast<double>(f[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[grp][col + i] = s[i];
  }
  __syncthreads();
  if (tid < D) {
    double s = 0;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) s += part[i][tid];
    c.mean[ph * D + tid] = f32_to_bf16(static_cast<float>(s / w.hi));
  }
}

template <typename T, int D, bool kPast>
__global__ __launch_bounds__(256) void cache4_read_kernel(const CacheArgs c, const RowArgs r) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes, kG = D / 32;
  constexpr int kS = 36;  // bytes of a feature in LDS: eight features on, eight banks on
  __shared__ __align__(16) uint8_t vt[D * kS];
  const int tid = threadIdx.x;
  PageWork w;
  const int64_t b = blockIdx.x / (static_cast<uint32_t>(r.span) * static_cast<uint32_t>(r.H));
  const int64_t n = new_tokens(r, b);
  bool live;
  if (!read_work(c, r, b, w, live)) return;
  const int64_t ph = w.pid * r.H + w.h;
  const uint8_t *kc = c.kc + ph * (kPage * D / 2), *vc = c.vc + ph * (kPage * D / 2);
  const uint8_t *ks = c.ks + ph * (kPage * kG), *vs = c.vs + ph * kPage, *vo = c.vo + ph * (kG * 32);
  // everything that is read is on its way before anything is waited for
  constexpr int kPasses = kPage / kRows;
  const int col = tid % kLanes * 8, gr = col / 32;
  uint32_t kw[kPasses], kb[kPasses], vb[kPasses], off[kPasses];
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    const int row = pass * kRows + tid / kLanes;
    const int place = page_place(row), i = place & 15;
    kw[pass] = kb[pass] = vb[pass] = off[pass] = 0;
    if (!live) continue;
    kw[pass] = *reinterpret_cast<const uint32_t *>(kc + key4_at<D>(row, col));
    kb[pass] = ks[gr * kPage + key_place(row)];
    vb[pass] = vs[place];
    off[pass] = *reinterpret_cast<const uint32_t *>(vo + ((place >> 4) * kG + gr) * 8 + (i >> 3) * 4) >> offset4_bit(i & 7) & 15u;
  }
  if (live && tid < 64 * kG) {
    const int g = tid & 3, f = (tid >> 6) * 32 + ((tid >> 2) & 15);
    const u32x4 x = *reinterpret_cast<const u32x4 *>(vc + value4_at(f, g));
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t *>(vt + (f + (i >> 1) * 16) * kS + g * 8 + (i & 1) * 4) = x[i];
  }
  __syncthreads();
  T *ko = const_cast<T *>(static_cast<const T *>(r.k)) + (w.b * r.H + w.h) * r.T * D;
  T *vout = const_cast<T *>(static_cast<const T *>(r.v)) + (w.b * r.H + w.h) * r.T * D;
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    const int row = pass * kRows + tid / kLanes;
    if (row < w.lo || row >= w.hi) continue;
    const int64_t t = w.j * kPage + row - w.s;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (live && t < n) {
      const int place = page_place(row), g = place >> 4, i = place & 15;
      // a slot that was never written has zeros throughout
      const float ke = pow2_byte(kb[pass]);
      const float ve = kb[pass] == 255 ? ke : pow2_byte(max(static_cast<int>(vb[pass] + off[pass]) - 15, 0));
      uint32_t vw = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) vw |= (vt[(col + e) * kS + g * 8 + (i >> 1)] >> (4 * (i & 1)) & 15u) << (4 * e);
      unpack_e2m1(kw[pass], x, ke);
      unpack_e2m1(vw, y, ve);
    }
    store8<kPast>(ko + t * D + col, x);
    store8<kPast>(vout + t * D + col, y);
  }
}

template <typename T, int D>
void launch_write4(const CacheArgs &c, const RowArgs &r, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(r.B * r.H * r.span));
  if constexpr (sizeof(T) == 4) {
    if (!floats_past(r, D)) {
      hipLaunchKernelGGL((cache4_write_kernel<T, D, false>), grid, dim3(256), 0, s, c, r);
      return;
    }
  }
  hipLaunchKernelGGL((cache4_write_kernel<T, D, true>), grid, dim3(256), 0, s, c, r);
}
template <typename T, int D>
void launch_read4(const CacheArgs &c, const RowArgs &r, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(r.B * r.H * r.span));
  if constexpr (sizeof(T) == 2) {
    if (halves_past(r, D)) {
      hipLaunchKernelGGL((cache4_read_kernel<T, D, true>), grid, dim3(256), 0, s, c, r);
      return;
    }
  }
  hipLaunchKernelGGL((cache4_read_kernel<T, D, false>), grid, dim3(256), 0, s, c, r);
}

}  // namespace
}  // namespace vasc

extern "C" int vasc_cache4_write(const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st, const void *v, int64_t v_sb,
                                 int64_t v_sh, int64_t v_st, int64_t B, int64_t H, int64_t T, int64_t D, int32_t dtype,
                                 const int32_t *page_table, int64_t table_stride, int64_t max_pages, const int32_t *start,
                                 const int32_t *count, uint8_t *kc, uint8_t *vc, uint8_t *ks, uint8_t *vs, uint8_t *vo,
                                 uint16_t *mean, int64_t pages, void *stream) {
  using namespace vasc;
  int rc;
  if ((rc = check_cache(kc, vc, ks, vs, pages, page_table, table_stride, max_pages, D))) return rc;
  if ((rc = check_rows("k", k, k_sb, k_sh, k_st))) return rc;
  if ((rc = check_rows("v", v, v_sb, v_sh, v_st))) return rc;
  VASC_REQUIRE(vo && (reinterpret_cast<uintptr_t>(vo) & 15) == 0, "vo must be given and 16-byte aligned");
  VASC_REQUIRE(mean && start, "mean and start are required");
  RowArgs r = {k, v, k_sb, k_sh, k_st, v_sb, v_sh, v_st, start, count, B, H, T, 0};
  if ((rc = check_tokens(r, dtype))) return rc;
  const CacheArgs c = {kc, vc, ks, vs, mean, pages, page_table, table_stride, max_pages, vo};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (D == 64)
    (dtype == 0 ? launch_write4<__bf16, 64> : dtype == 1 ? launch_write4<_Float16, 64> : launch_write4<float, 64>)(c, r, s);
  else
    (dtype == 0 ? launch_write4<__bf16, 128> : dtype == 1 ? launch_write4<_Float16, 128> : launch_write4<float, 128>)(c, r, s);
  return check_launch("vasc_cache4_write");
}

extern "C" int vasc_cache4_read(const uint8_t *kc, const uint8_t *vc, const uint8_t *ks, const uint8_t *vs,
                                const uint8_t *vo, int64_t pages, const int32_t *page_table, int64_t table_stride,
                                int64_t max_pages, const int32_t *start, const int32_t *count, int64_t B, int64_t H,
                                int64_t T, int64_t D, int32_t dtype, void *ko, void *vout, void *stream) {
  using namespace vasc;
  int rc;
  if ((rc = check_cache(kc, vc, ks, vs, pages, page_table, table_stride, max_pages, D))) return rc;
  if ((rc = check_rows("ko", ko, 0, 0, D))) return rc;
  if ((rc = check_rows("vo", vout, 0, 0, D))) return rc;
  VASC_REQUIRE(vo && (reinterpret_cast<uintptr_t>(vo) & 15) == 0, "the cache's vo must be given and 16-byte aligned");
  VASC_REQUIRE(start, "start is required");
  RowArgs r = {ko, vout, 0, 0, 0, 0, 0, 0, start, count, B, H, T, 0};
  if ((rc = check_tokens(r, dtype))) return rc;
  const CacheArgs c = {const_cast<uint8_t *>(kc), const_cast<uint8_t *>(vc), const_cast<uint8_t *>(ks),
                       const_cast<uint8_t *>(vs), nullptr, pages, page_table, table_stride, max_pages,
                       const_cast<uint8_t *>(vo)};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (D == 64)
    (dtype == 0 ? launch_read4<__bf16, 64> : dtype == 1 ? launch_read4<_Float16, 64> : launch_read4<float, 64>)(c, r, s);
  else
    (dtype == 0 ? launch_read4<__bf16, 128> : dtype == 1 ? launch_read4<_Float16, 128> : launch_read4<float, 128>)(c, r, s);
  return check_launch("vasc_cache4_read");
}
