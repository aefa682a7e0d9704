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
#include "cache_page.h"

namespace vasc {
namespace {

// Eight values over 2^(byte - 127) as e2m1 codes: to nearest, ties to even, at most 6.
__device__ __forceinline__ uint32_t quantise8_e2m1(const float (&x)[8], int byte) {
  const float inv = __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fminf(fmaxf(x[i] * inv, -6.f), 6.f);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.0f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.0f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.0f, 3);
}

// Max over the four neighbouring lanes of a group.
__device__ __forceinline__ float group4_max(float v) {
  v = fmaxf(v, dpp<kQuadXor1>(v));
  return fmaxf(v, dpp<kQuadXor2>(v));
}

// Max over the groups of a row, which agree within.
template <int D>
__device__ __forceinline__ int groups_max(int v) {
  v = max(v, xor_lane(v, 4));
  return D == 128 ? max(v, xor_lane(v, 8)) : v;
}

template <typename T, int D>
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
      float x[8], y[8];
      load8(kin + t * r.kst + col, x);
      load8(vin + t * r.vst + col, y);
      float kmax = 0.f, vmax = 0.f, bad = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        kmax = fmaxf(kmax, fabsf(x[i]));
        vmax = fmaxf(vmax, fabsf(y[i]));
        // all ones in the exponent: infinity or NaN (a maximum drops NaN)
        if ((__float_as_uint(x[i]) & 0x7f800000u) == 0x7f800000u || (__float_as_uint(y[i]) & 0x7f800000u) == 0x7f800000u)
          bad = 1.f;
      }
      int kb = power_of<2>(group4_max(kmax), -60, 60) + 127, vb = power_of<2>(group4_max(vmax), -60, 60) + 127;
      int row_b = groups_max<D>(vb);
      vb = max(vb, row_b - 14);
      uint32_t kw = 0, vw = 0;
      if (groups_max<D>(static_cast<int>(group4_max(bad))) == 0) {
        kw = quantise8_e2m1(x, kb);
        vw = quantise8_e2m1(y, vb);
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
    uint32_t cover[2] = {0, 0}, out[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int t = token4_of(g, i);
      if (t < w.lo || t >= w.hi) continue;
      cover[i >> 3] |= 15u << (4 * (i & 7));
#pragma unroll
      for (int half = 0; half < 2; ++half)
        out[half * 2 + (i >> 3)] |= (vt[t][(f >> 3) + half * 2] >> (4 * (f & 7)) & 15u) << (4 * (i & 7));
    }
    if (cover[0] | cover[1]) {
      u32x4 *at = reinterpret_cast<u32x4 *>(vc + value4_at(f, g));
      u32x4 x = {out[0], out[1], out[2], out[3]};
      if ((cover[0] & cover[1]) != 0xffffffffu) {
        const u32x4 old = *at;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] |= old[i] & ~cover[i & 1];
      }
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
      unpack_e2m1(kt[row][word], f);
      const float e = pow2_byte(ke[row][gr]);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += static_cast<double>(f[i] * e);
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

template <typename T, int D>
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
      unpack_e2m1(kw[pass], x);
      unpack_e2m1(vw, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] *= ke;
        y[e] *= ve;
      }
    }
    store8(ko + t * D + col, x);
    store8(vout + t * D + col, y);
  }
}

template <typename T, int D>
void launch_write4(const CacheArgs &c, const RowArgs &r, hipStream_t s) {
  hipLaunchKernelGGL((cache4_write_kernel<T, D>), dim3(static_cast<unsigned>(r.B * r.H * r.span)), dim3(256), 0, s, c, r);
}
template <typename T, int D>
void launch_read4(const CacheArgs &c, const RowArgs &r, hipStream_t s) {
  hipLaunchKernelGGL((cache4_read_kernel<T, D>), dim3(static_cast<unsigned>(r.B * r.H * r.span)), dim3(256), 0, s, c, r);
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
