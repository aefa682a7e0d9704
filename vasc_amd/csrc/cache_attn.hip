// Attention over listed pages of the 8-bit block cache.
//
// A unit's query rows (block_q tokens x G heads of one key head) are the
// columns of S^T = K Q^T, 16 to a tile. K's codes are read as they lie: a
// 16-key tile is the A operand of 16x16x32 products, lane l holding 16
// consecutive features of key l & 15, converted in registers (e4m3 is exact in
// bfloat16 and in half). S^T leaves each lane four consecutive keys of one
// query row, which is what the second product's B operand wants of P^T; the
// cache holds V transposed with the tokens in that same order, so V too goes
// from memory to the matrix pipe without a shuffle.
//
// Powers of two: a row's exponents scale S (keys) and enter the softmax's
// exponent (values), e = c S + ev, so that the weights of the second product
// are w = 2^(e - m) with m the running maximum of e, and its sum l takes them
// without the value's power: l = sum w 2^-ev. Weights are rounded to half (11
// bits; bfloat16's 8 would be the largest error of a float16 result). They are
// held as 2^(11 + e - m), so that those under half's range are below 2^-36 of
// the row's largest, and m is renewed only when it would be passed by 2^4.
#include "stream.h"

namespace vasc {
namespace {

constexpr float kHeadroom = 11.f, kSlack = 4.f;  // kHeadroom + kSlack < 16: half's largest exponent

struct AttnParams {
  const void *q;
  int64_t qsb, qsh, qst;
  void *o;
  int64_t osb, osh, ost;
  int64_t B, T;
  int H, G, U;
  const uint8_t *kc, *vc, *ks, *vs;
  int64_t pages;
  const int32_t *table;
  int64_t table_stride, max_pages;
  const int32_t *lengths, *n_q;
  int block_q, causal;
  const int32_t *index, *count;
  int64_t width;
  float scale;  // times log2(e)
  int rows;     // block_q * G
  int parts;    // workgroups that share a unit's pages
  int tiles;    // workgroups that share a unit's rows
  float *ws;
};

template <typename Q>
struct Mfma;
template <>
struct Mfma<__bf16> {
  typedef bf16x8 vec;
  static __device__ __forceinline__ floatx4 mul(vec a, vec b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t two(uint32_t w, bool hi) {
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
  }
};
template <>
struct Mfma<_Float16> {
  typedef halfx8 vec;
  static __device__ __forceinline__ floatx4 mul(vec a, vec b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t two(uint32_t w, bool hi) {
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                                           : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
  }
};

// Eight e4m3 codes as the eight 16-bit values of an operand.
template <typename Q>
__device__ __forceinline__ typename Mfma<Q>::vec widen(uint32_t a, uint32_t b) {
  const u32x4 w = {Mfma<Q>::two(a, false), Mfma<Q>::two(a, true), Mfma<Q>::two(b, false), Mfma<Q>::two(b, true)};
  return __builtin_bit_cast(typename Mfma<Q>::vec, w);
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const floatx2 f = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, halfx2));
}

// The four lanes l, l ^ 16, l ^ 32, l ^ 48 share a query row.
__device__ __forceinline__ float row4_max(float v) {
  v = fmaxf(v, xor_lane(v, 16));
  return fmaxf(v, xor_lane(v, 32));
}
__device__ __forceinline__ float row4_sum(float v) {
  v += xor_lane(v, 16);
  return v + xor_lane(v, 32);
}

// A workgroup of 4 waves: kRowWaves of them side by side over the rows, the others over the pages.
// Each wave holds kTiles tiles of 16 rows.
template <typename Q, int D, int kTiles, int kRowWaves>
__global__ __launch_bounds__(256, 2) void cache_attn_kernel(const AttnParams p) {
  constexpr int kPageWaves = 4 / kRowWaves;
  constexpr int kK = D / 64;    // 16-byte loads of a key per lane
  constexpr int kDT = D / 16;   // feature tiles of the output
  constexpr int kRows = kRowWaves * kTiles * 16;
  typedef typename Mfma<Q>::vec vec;
  __shared__ float lo[kPageWaves > 1 ? kPageWaves : 1][kPageWaves > 1 ? kRows : 1][kPageWaves > 1 ? D + 2 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const int rw = wave % kRowWaves, pw = wave / kRowWaves;
  // workgroup -> (sequence and key head, part, unit, row tile): the units of a part read the same pages
  int id = static_cast<int>(xcd_remap(blockIdx.x, gridDim.x));
  const int tile = id % p.tiles;
  id /= p.tiles;
  const int u = id % p.U;
  id /= p.U;
  const int part = id % p.parts;
  const int bh = id / p.parts;
  const int64_t b = bh / p.H;
  const int h = bh - static_cast<int>(b) * p.H;
  const int64_t L = p.lengths[b];
  int64_t nq = p.n_q ? p.n_q[b] : p.T;
  nq = nq < 0 ? 0 : (nq < p.T ? nq : p.T);
  const int64_t t0 = static_cast<int64_t>(u) * p.block_q;
  const int64_t t1 = t0 + p.block_q < nq ? t0 + p.block_q : nq;
  const UnitView view = unit_view(L, nq, t0, t1, p.max_pages, p.causal);
  const int64_t cut = clamp_tokens(L, p.max_pages);

  // the rows of this wave's tiles: query operand, and one past the last key that the row sees
  vec qf[kTiles][kK * 2];
  int64_t limit[kTiles];
  int64_t low = cut;  // keys below it are seen by every row of the wave that counts
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    const int r = ((tile * kRowWaves + rw) * kTiles + i) * 16 + col;
    const int tl = r / p.G, gh = r - tl * p.G;
    const int64_t t = t0 + tl;
    const bool live = r < p.rows && t < t1;
    limit[i] = live ? cut : 0;
    if (live && p.causal) {
      const int64_t own = L - nq + t + 1;
      limit[i] = own < cut ? (own > 0 ? own : 0) : cut;
    }
    if (live && limit[i] < low) low = limit[i];
    const Q *src = static_cast<const Q *>(p.q) + b * p.qsb + (static_cast<int64_t>(h) * p.G + gh) * p.qsh + t * p.qst + g * 16;
#pragma unroll
    for (int x = 0; x < kK; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y)
        qf[i][x * 2 + y] = live ? *reinterpret_cast<const vec *>(src + x * 64 + y * 8) : vec{};
  }
  // the lowest limit over the wave's rows: pages below it need no mask
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t other = __shfl_xor(static_cast<long long>(low), off);
    if (other < low) low = other;
  }

  floatx4 acc[kTiles][kDT];
  float m[kTiles], l[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    m[i] = -__builtin_inff();
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < kDT; ++d) acc[i][d] = floatx4{0, 0, 0, 0};
  }

  // this part's entries of the list (or of the pages in order)
  const int64_t unit_row = static_cast<int64_t>(bh) * p.U + u;
  int64_t entries = view.seen;
  const int32_t *list = nullptr;
  if (p.index) {
    list = p.index + unit_row * p.width;
    const int64_t n = p.count[unit_row];
    entries = view.seen == 0 ? 0 : (n < 0 ? 0 : (n < p.width ? n : p.width));
  }
  const int64_t share = cdiv(entries, p.parts);
  const int64_t e0 = part * share, e1 = e0 + share < entries ? e0 + share : entries;

  for (int64_t base = e0; base < e1; base += 64) {
    // lane i resolves entry base + i: logical page and physical page, or -1
    int64_t mine = base + lane;
    int page = -1, pid = -1;
    if (mine < e1) {
      page = list ? list[mine] : static_cast<int>(mine);
      if (list && mine > 0 && list[mine - 1] >= page) page = -1;
      if (page >= 0 && page < view.seen) {
        pid = p.table[b * p.table_stride + page];
        if (pid < 0 || pid >= p.pages) pid = -1;
      }
    }
    const int n = static_cast<int>(e1 - base < 64 ? e1 - base : 64);
    for (int i = pw; i < n; i += kPageWaves) {
      const int ppage = __builtin_amdgcn_readlane(pid, i);
      const int lpage = __builtin_amdgcn_readlane(page, i);
      if (ppage < 0) continue;
      const int64_t ph = static_cast<int64_t>(ppage) * p.H + h;
      const uint8_t *kp = p.kc + ph * (kPage * D) + col * D + g * 16;
      const uint8_t *vp = p.vc + ph * (kPage * D) + col * kPage + g * 16;
      u32x4 kr[4][kK], vr[kDT];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int x = 0; x < kK; ++x) kr[t][x] = *reinterpret_cast<const u32x4 *>(kp + t * 16 * D + x * 64);
      const u32x4 kb = *reinterpret_cast<const u32x4 *>(p.ks + ph * kPage + g * 16);
      const u32x4 vb = *reinterpret_cast<const u32x4 *>(p.vs + ph * kPage + g * 16);
#pragma unroll
      for (int d = 0; d < kDT; ++d) vr[d] = *reinterpret_cast<const u32x4 *>(vp + d * 16 * kPage);

      floatx4 s[kTiles][4];
#pragma unroll
      for (int i2 = 0; i2 < kTiles; ++i2)
#pragma unroll
        for (int t = 0; t < 4; ++t) s[i2][t] = floatx4{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int x = 0; x < kK; ++x) {
          const u32x4 w = kr[t][x];
          const vec a0 = widen<Q>(w[0], w[1]), a1 = widen<Q>(w[2], w[3]);
#pragma unroll
          for (int i2 = 0; i2 < kTiles; ++i2) {
            s[i2][t] = Mfma<Q>::mul(a0, qf[i2][x * 2], s[i2][t]);
            s[i2][t] = Mfma<Q>::mul(a1, qf[i2][x * 2 + 1], s[i2][t]);
          }
        }
      const int64_t key0 = static_cast<int64_t>(lpage) * kPage;
      const bool masked = key0 + kPage > low;
      halfx8 w[kTiles][2];
#pragma unroll
      for (int i2 = 0; i2 < kTiles; ++i2) {
        float e[16];
        float top = -__builtin_inff();
        const int lim = static_cast<int>(limit[i2] - key0 < kPage ? (limit[i2] > key0 ? limit[i2] - key0 : 0) : kPage);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t kw = kb[t], vw = vb[t];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float c = pow2_byte((kw >> (8 * j)) & 255u) * p.scale;
            const float ev = static_cast<float>((vw >> (8 * j)) & 255u) - 127.f;
            float x = fmaf(s[i2][t][j], c, ev);
            if (masked) x = t * 16 + g * 4 + j < lim ? x : -__builtin_inff();
            e[t * 4 + j] = x;
            top = fmaxf(top, x);
          }
        }
        top = row4_max(top);
        if (__ballot(top > m[i2] + kSlack)) {
          const float mn = fmaxf(m[i2], top);
          const float a = mn == m[i2] ? 1.f : __builtin_amdgcn_exp2f(m[i2] - mn);
          l[i2] *= a;
#pragma unroll
          for (int d = 0; d < kDT; ++d) acc[i2][d] *= a;
          m[i2] = mn;
        }
        const float ref = m[i2] == -__builtin_inff() ? 0.f : m[i2] - kHeadroom;
        uint32_t packed[8];
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint32_t vw = vb[t];
          float x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[j] = __builtin_amdgcn_exp2f(e[t * 4 + j] - ref);
            sum = fmaf(x[j], pow2_byte(254u - ((vw >> (8 * j)) & 255u)), sum);
          }
          packed[t * 2] = pack_half2(x[0], x[1]);
          packed[t * 2 + 1] = pack_half2(x[2], x[3]);
        }
        l[i2] += sum;
        w[i2][0] = __builtin_bit_cast(halfx8, u32x4{packed[0], packed[1], packed[2], packed[3]});
        w[i2][1] = __builtin_bit_cast(halfx8, u32x4{packed[4], packed[5], packed[6], packed[7]});
      }
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
        const u32x4 v = vr[d];
        const halfx8 a0 = widen<_Float16>(v[0], v[1]), a1 = widen<_Float16>(v[2], v[3]);
#pragma unroll
        for (int i2 = 0; i2 < kTiles; ++i2) {
          acc[i2][d] = Mfma<_Float16>::mul(a0, w[i2][0], acc[i2][d]);
          acc[i2][d] = Mfma<_Float16>::mul(a1, w[i2][1], acc[i2][d]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    l[i] = row4_sum(l[i]);
    if (limit[i] == 0) {  // no key, or no row: pages that all counting rows see were not masked for it
      m[i] = -__builtin_inff();
      l[i] = 0.f;
#pragma unroll
      for (int d = 0; d < kDT; ++d) acc[i][d] = floatx4{0, 0, 0, 0};
    }
  }

  // the page waves' parts, joined in LDS by the first of them
  if constexpr (kPageWaves > 1) {
    if (pw > 0) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        float *dst = lo[pw][(rw * kTiles + i) * 16 + col];
        if (g == 0) {
          dst[D] = m[i];
          dst[D + 1] = l[i];
        }
#pragma unroll
        for (int d = 0; d < kDT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) dst[d * 16 + g * 4 + j] = acc[i][d][j];
      }
    }
    __syncthreads();
    if (pw > 0) return;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      float mx = m[i];
#pragma unroll
      for (int x = 1; x < kPageWaves; ++x) mx = fmaxf(mx, lo[x][(rw * kTiles + i) * 16 + col][D]);
      const float a = m[i] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m[i] - mx);
      l[i] *= a;
#pragma unroll
      for (int d = 0; d < kDT; ++d) acc[i][d] *= a;
#pragma unroll
      for (int x = 1; x < kPageWaves; ++x) {
        const float *src = lo[x][(rw * kTiles + i) * 16 + col];
        const float mo = src[D];
        const float c = mo == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mo - mx);
        l[i] = fmaf(src[D + 1], c, l[i]);
#pragma unroll
        for (int d = 0; d < kDT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][d][j] = fmaf(src[d * 16 + g * 4 + j], c, acc[i][d][j]);
      }
      m[i] = mx;
    }
  }
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    const int r = ((tile * kRowWaves + rw) * kTiles + i) * 16 + col;
    if (r >= p.rows) continue;
    const int tl = r / p.G, gh = r - tl * p.G;
    const int64_t t = t0 + tl;
    if (t >= p.T) continue;
    if (p.parts == 1) {
      const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
      Q *dst = static_cast<Q *>(p.o) + b * p.osb + (static_cast<int64_t>(h) * p.G + gh) * p.osh + t * p.ost + g * 4;
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
        struct alignas(8) Four { Q v[4]; } out;
#pragma unroll
        for (int j = 0; j < 4; ++j) out.v[j] = from_f32<Q>(acc[i][d][j] * inv);
        *reinterpret_cast<Four *>(dst + d * 16) = out;
      }
    } else {
      // [unit row][part][D], behind them (m, l) alike
      const int64_t at = (unit_row * p.rows + r) * p.parts + part;
      float *dst = p.ws + at * D + g * 4;
#pragma unroll
      for (int d = 0; d < kDT; ++d) *reinterpret_cast<floatx4 *>(dst + d * 16) = acc[i][d];
      if (g == 0) {
        float *ml = p.ws + static_cast<int64_t>(p.B) * p.H * p.U * p.rows * p.parts * D + at * 2;
        ml[0] = m[i];
        ml[1] = l[i];
      }
    }
  }
}

// Joins the parts of each row: 16 or 32 lanes a row, four features each.
template <typename Q, int D>
__global__ __launch_bounds__(256) void cache_join_kernel(const AttnParams p) {
  constexpr int kLanes = D / 4;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  const int64_t all = p.B * p.H * p.U * static_cast<int64_t>(p.rows);
  if (row >= all) return;
  const int d = (threadIdx.x % kLanes) * 4;
  const int64_t unit = row / p.rows;
  const int r = static_cast<int>(row - unit * p.rows), tl = r / p.G, gh = r - tl * p.G;
  const int u = static_cast<int>(unit % p.U);
  const int64_t bh = unit / p.U, b = bh / p.H, h = bh - b * p.H;
  const int64_t t = static_cast<int64_t>(u) * p.block_q + tl;
  if (t >= p.T) return;
  const float *o = p.ws + row * p.parts * D + d;
  const float *ml = p.ws + all * p.parts * D + row * p.parts * 2;
  float mx = -__builtin_inff();
  for (int i = 0; i < p.parts; ++i) mx = fmaxf(mx, ml[i * 2]);
  floatx4 acc = {0, 0, 0, 0};
  float l = 0.f;
  for (int i = 0; i < p.parts; ++i) {
    const float c = ml[i * 2] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ml[i * 2] - mx);
    l = fmaf(ml[i * 2 + 1], c, l);
    acc += *reinterpret_cast<const floatx4 *>(o + static_cast<int64_t>(i) * D) * c;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  struct alignas(8) Four { Q v[4]; } out;
#pragma unroll
  for (int j = 0; j < 4; ++j) out.v[j] = from_f32<Q>(acc[j] * inv);
  *reinterpret_cast<Four *>(static_cast<Q *>(p.o) + b * p.osb + (h * p.G + gh) * p.osh + t * p.ost + d) = out;
}

struct Shape {
  int kind;   // 0: 16 rows, four page waves; 1: 32 rows likewise; 2: 64 rows, four row waves; 3: 128 rows
  int tiles, parts;
};

// Up to 32 rows a workgroup is bound by the cache's bytes, so its waves share the pages; beyond, by the products, so
// they share the rows. The pages are split over workgroups until about four of them run on each CU, with at least
// eight pages each (two for a page wave).
Shape attn_shape(int64_t units, int64_t rows, int64_t pages) {
  Shape s;
  s.kind = rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
  s.tiles = 1;
  int64_t parts = cdiv(1024, units);
  const int64_t most = cdiv(pages, 8);
  if (parts > most) parts = most;
  s.parts = static_cast<int>(parts < 1 ? 1 : parts > 256 ? 256 : parts);
  return s;
}

template <typename Q, int D>
int launch_attn(const AttnParams &p, const Shape &s, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.B * p.H * p.U * s.parts * s.tiles));
  switch (s.kind) {
    case 0: hipLaunchKernelGGL((cache_attn_kernel<Q, D, 1, 1>), grid, dim3(256), 0, st, p); break;
    case 1: hipLaunchKernelGGL((cache_attn_kernel<Q, D, 2, 1>), grid, dim3(256), 0, st, p); break;
    case 2: hipLaunchKernelGGL((cache_attn_kernel<Q, D, 1, 4>), grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL((cache_attn_kernel<Q, D, 2, 4>), grid, dim3(256), 0, st, p); break;
  }
  int rc = check_launch("vasc_cache_attn");
  if (rc || s.parts == 1) return rc;
  const int64_t rows = p.B * p.H * p.U * static_cast<int64_t>(p.rows);
  hipLaunchKernelGGL((cache_join_kernel<Q, D>), dim3(static_cast<unsigned>(cdiv(rows, 256 / (D / 4)))), dim3(256), 0, st, p);
  return check_launch("vasc_cache_attn");
}

bool attn_sizes(int64_t B, int64_t Hq, int64_t H, int64_t T, int64_t D, int64_t block_q, int64_t max_pages, int64_t width) {
  if (!(B > 0 && H > 0 && T > 0 && Hq > 0 && Hq % H == 0 && (D == 64 || D == 128))) return false;
  if (!(block_q >= 1 && block_q <= 128 && Hq / H <= 128 && block_q * (Hq / H) <= 128)) return false;
  if (!(max_pages > 0 && max_pages < (int64_t(1) << 24) && width >= 0 && width < (int64_t(1) << 24))) return false;
  if (!(B < (1 << 24) && H < (1 << 16) && T < (int64_t(1) << 30))) return false;
  return B * H < (int64_t(1) << 30) / cdiv(T, block_q);
}

int64_t workspace_bytes(int64_t units, int64_t rows, int64_t D, int parts) {
  return parts == 1 ? 0 : units * rows * parts * (D + 2) * 4;
}

}  // namespace
}  // namespace vasc

extern "C" int64_t vasc_cache_attn_workspace_size(int64_t B, int64_t Hq, int64_t H, int64_t T, int64_t D,
                                                  int64_t block_q, int64_t max_pages, int64_t width) {
  using namespace vasc;
  if (!attn_sizes(B, Hq, H, T, D, block_q, max_pages, width)) return -1;
  const int64_t units = B * H * cdiv(T, block_q), rows = block_q * (Hq / H);
  return workspace_bytes(units, rows, D, attn_shape(units, rows, width ? width : max_pages).parts);
}

extern "C" int vasc_cache_attn(const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st, void *o, int64_t o_sb,
                               int64_t o_sh, int64_t o_st, int64_t B, int64_t Hq, int64_t H, int64_t T, int64_t D,
                               int32_t dtype, const uint8_t *kc, const uint8_t *vc, const uint8_t *ks,
                               const uint8_t *vs, int64_t pages, const int32_t *page_table, int64_t table_stride,
                               int64_t max_pages, const int32_t *lengths, const int32_t *q_count, int64_t block_q,
                               const int32_t *index, int64_t width, const int32_t *count, int32_t causal, float scale,
                               void *workspace, int64_t workspace_bytes_given, void *stream) {
  using namespace vasc;
  VASC_SUPPORTED(D == 64 || D == 128, "D %lld not built (64, 128)", (long long)D);
  VASC_SUPPORTED(dtype == 0 || dtype == 1, "dtype %d not built", dtype);
  VASC_REQUIRE(q && o && kc && vc && ks && vs && page_table && lengths, "a required pointer is NULL");
  VASC_REQUIRE((index == nullptr) == (count == nullptr) && (index == nullptr) == (width == 0), "index, width and count go together");
  VASC_REQUIRE(attn_sizes(B, Hq, H, T, D, block_q, max_pages, width),
               "sizes B %lld Hq %lld H %lld T %lld block_q %lld: Hq a multiple of H, block_q * Hq / H from 1 to 128",
               (long long)B, (long long)Hq, (long long)H, (long long)T, (long long)block_q);
  VASC_REQUIRE(pages > 0 && pages < (int64_t(1) << 31), "pages outside [1, 2^31)");
  VASC_REQUIRE(table_stride >= max_pages || table_stride == 0, "table_stride below max_pages");
  for (const void *x : {q, static_cast<const void *>(kc), static_cast<const void *>(vc), static_cast<const void *>(ks),
                        static_cast<const void *>(vs)})
    VASC_REQUIRE((reinterpret_cast<uintptr_t>(x) & 15) == 0, "q and the cache must be 16-byte aligned");
  VASC_REQUIRE((reinterpret_cast<uintptr_t>(o) & 7) == 0, "o must be 8-byte aligned");
  for (int64_t st : {q_sb, q_sh, q_st}) VASC_REQUIRE(st % 8 == 0, "q's strides must be multiples of 8");
  for (int64_t st : {o_sb, o_sh, o_st}) VASC_REQUIRE(st % 4 == 0, "o's strides must be multiples of 4");
  AttnParams p = {};
  p.q = q; p.qsb = q_sb; p.qsh = q_sh; p.qst = q_st;
  p.o = o; p.osb = o_sb; p.osh = o_sh; p.ost = o_st;
  p.B = B; p.T = T;
  p.H = static_cast<int>(H);
  p.G = static_cast<int>(Hq / H);
  p.U = static_cast<int>(cdiv(T, block_q));
  p.kc = kc; p.vc = vc; p.ks = ks; p.vs = vs; p.pages = pages;
  p.table = page_table; p.table_stride = table_stride; p.max_pages = max_pages;
  p.lengths = lengths; p.n_q = q_count;
  p.block_q = static_cast<int>(block_q);
  p.causal = causal;
  p.index = index; p.width = width; p.count = count;
  p.scale = scale * 1.4426950408889634f;
  p.rows = p.block_q * p.G;
  const int64_t units = B * H * p.U;
  const Shape s = attn_shape(units, p.rows, width ? width : max_pages);
  p.parts = s.parts;
  p.tiles = s.tiles;
  VASC_REQUIRE(units < (int64_t(1) << 31) / (s.parts * s.tiles), "too many units");
  const int64_t need = workspace_bytes(units, p.rows, D, s.parts);
  VASC_REQUIRE(need == 0 || (workspace && workspace_bytes_given >= need), "workspace of %lld bytes, %lld needed",
               (long long)workspace_bytes_given, (long long)need);
  VASC_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "the workspace must be 16-byte aligned");
  p.ws = static_cast<float *>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (D == 64) return dtype == 0 ? launch_attn<__bf16, 64>(p, s, st) : launch_attn<_Float16, 64>(p, s, st);
  return dtype == 0 ? launch_attn<__bf16, 128>(p, s, st) : launch_attn<_Float16, 128>(p, s, st);
}
