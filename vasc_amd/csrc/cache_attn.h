// Shared by the attention over the 8-bit and the 4-bit block cache (cache_attn.hip, cache4_attn.hip): the units of work and
// their pages, the running softmax of a wave's row tiles, the join of parts, and how many parts there are.
#pragma once

#include <cmath>

#include "stream.h"

namespace vasc {
namespace {

constexpr float kHeadroom = 11.f, kSlack = 4.f;  // kHeadroom + kSlack < 16: half's largest exponent
constexpr uint32_t kSmall = 127 - 30;            // exponent bytes from 67 to below it are small; 0 is a slot that was never written

struct AttnParams {
  const void *q;
  int64_t qsb, qsh, qst;
  void *o;
  int64_t osb, osh, ost;
  int64_t B, T;
  int H, G, U;          // U: units of this launch, from u0 of the call's list_U on
  int u0, list_U;
  const uint8_t *kc, *vc, *ks, *vs, *vo;  // vo: of the 4-bit cache
  int64_t pages;
  const int32_t *table;
  int64_t table_stride, max_pages;
  const int32_t *lengths, *n_q;
  int block_q, causal;
  const int32_t *index, *count;
  int64_t width;
  float c;      // scale * log2(e)
  int rows;     // block_q * G
  int parts;    // workgroups that share a unit's pages
  float *ws;
};

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const floatx2 f = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, halfx2));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;  // three operands at once; a NaN gives way to a number, as with fmaxf
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// 2^d, d <= 0, as near * far: d may lie under -126 where a sum is scaled. far is 1 for d from -120 on.
__device__ __forceinline__ void two_powers(float d, float &near, float &far) {
  near = __builtin_amdgcn_exp2f(fmaxf(d, -120.f));
  far = __builtin_amdgcn_exp2f(fminf(d + 120.f, 0.f));
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

// What a workgroup works on: workgroup -> (sequence and key head, part, unit); the units of a part read the same pages.
struct Work {
  int64_t b, L, nq, t0, t1, unit_row;
  int h, u, part, cut;
  int entries;          // pages of the unit
  int e0, e1;           // this part's of them
  int seen;
  const int32_t *list;  // or NULL: the pages in order
};

__device__ __forceinline__ Work work_of(const AttnParams &p) {
  Work w;
  // The units of a part on one XCD, whose L2 then has their pages once; the parts in turn over the XCDs, which have the same
  // work so however uneven the sequences are. Measured, in us: eight sequences of 12000 to 33000 tokens, 59 with a range of the
  // parts to each XCD and 45 so (4 bits), 87 and 72 (8 bits). What does not fill all XCDs comes last.
  int id = blockIdx.x;
  const int even = static_cast<int>(gridDim.x) / p.U / 8 * 8 * p.U;
  if (id < even) {
    const int local = id >> 3;
    w.u = local % p.U;
    id = local / p.U * 8 + (id & 7);
  } else {
    w.u = id % p.U;  // `even` is a multiple of U
    id /= p.U;
  }
  w.part = id % p.parts;
  const int bh = id / p.parts;
  w.b = bh / p.H;
  w.h = bh - static_cast<int>(w.b) * p.H;
  w.L = p.lengths[w.b];
  w.nq = p.n_q ? p.n_q[w.b] : p.T;
  w.nq = w.nq < 0 ? 0 : (w.nq < p.T ? w.nq : p.T);
  w.t0 = static_cast<int64_t>(p.u0 + w.u) * p.block_q;
  w.t1 = w.t0 + p.block_q < w.nq ? w.t0 + p.block_q : w.nq;
  const UnitView view = unit_view(w.L, w.nq, w.t0, w.t1, p.max_pages, p.causal);
  w.cut = static_cast<int>(clamp_tokens(w.L, p.max_pages));  // below 2^30
  w.seen = static_cast<int>(view.seen);
  w.unit_row = static_cast<int64_t>(bh) * p.U + w.u;
  w.entries = w.seen;
  w.list = nullptr;
  if (p.index) {
    const int64_t row = static_cast<int64_t>(bh) * p.list_U + p.u0 + w.u;
    w.list = p.index + row * p.width;
    const int64_t n = p.count[row];
    w.entries = w.seen == 0 ? 0 : static_cast<int>(n < 0 ? 0 : (n < p.width ? n : p.width));
  }
  const int share = (w.entries + p.parts - 1) / p.parts;
  w.e0 = min(w.part * share, w.entries);
  w.e1 = min(w.e0 + share, w.entries);
  return w;
}

// Entry `at` of the unit: its logical page (-1: none) and physical page (0 where there is none: it is read, and not seen).
__device__ __forceinline__ void resolve(const AttnParams &p, const Work &w, int at, int &page, int &pid) {
  page = -1;
  pid = 0;
  if (at >= w.e1) return;
  page = w.list ? w.list[at] : at;
  if (w.list && at > 0 && w.list[at - 1] >= page) page = -1;
  if (page >= w.seen) page = -1;
  if (page < 0) {
    page = -1;
    return;
  }
  pid = p.table[w.b * p.table_stride + page];
  if (pid < 0 || pid >= p.pages) {
    pid = 0;
    page = -1;
  }
}

// One past the last key that unit row r sees; 0 for no row.
__device__ __forceinline__ int row_limit(const AttnParams &p, const Work &w, int r, int64_t &t, int &gh) {
  const int tl = r / p.G;
  gh = r - tl * p.G;
  t = w.t0 + tl;
  if (r >= p.rows || t >= w.t1) return 0;
  if (!p.causal) return w.cut;
  const int64_t own = w.L - w.nq + t + 1;
  return static_cast<int>(own < w.cut ? (own > 0 ? own : 0) : w.cut);
}

// This lane's query operands of a row: [part][product]; zeros where there is no row. Product y takes the lane's features
// kRun g + 8 y on of every 4 kRun (kRun: as many consecutive features as a lane holds of a key). An infinite query has no softmax, whatever
// the sign of its logits, which a running maximum would not see where all of them are minus infinity: it goes as NaN.
template <typename Q, int D, int kRun, int kOps>
__device__ __forceinline__ void query_operands(const AttnParams &p, const Work &w, int64_t t, int gh, bool live, int g,
                                               bf16x8 (&out)[kOps]) {
  constexpr int kMul = D / 32, kParts = kOps / kMul;
  const Q *src = static_cast<const Q *>(p.q) + w.b * p.qsb + (static_cast<int64_t>(w.h) * p.G + gh) * p.qsh + t * p.qst + g * kRun;
  constexpr int kEach = kRun / 8;
#pragma unroll
  for (int y = 0; y < kMul; ++y) {
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (live) {
      struct alignas(16) Eight { Q v[8]; };
      const Eight v = *reinterpret_cast<const Eight *>(src + (y / kEach) * (4 * kRun) + (y % kEach) * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = to_f32(v.v[e]);
        if (!__builtin_isfinite(x[e])) x[e] = __builtin_nanf("");
      }
    }
#pragma unroll
    for (int piece = 0; piece < kParts; ++piece)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        out[piece * kMul + y][e] = static_cast<__bf16>(x[e]);
        if (kParts > 1) x[e] -= static_cast<float>(out[piece * kMul + y][e]);
      }
  }
}

// The running softmax of a wave's row tiles.
constexpr float kUnset = -3.0e38f;
template <int kTiles, int kDT>
struct Rows {
  floatx4 acc[kTiles][kDT];
  // ref: the exponent's reference; start: -ref / c; renew: the exponent that renews it (any, before the first key)
  float ref[kTiles], start[kTiles], renew[kTiles], l[kTiles];
  int limit[kTiles];
  int low, high;  // keys below `low` are seen by every row of the wave that counts, from `high` on by none

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      ref[i] = start[i] = l[i] = 0.f;
      renew[i] = kUnset;
#pragma unroll
      for (int d = 0; d < kDT; ++d) acc[i][d] = floatx4{0, 0, 0, 0};
    }
  }

  // After limit[]: low and high over the wave.
  __device__ __forceinline__ void bounds(int cut) {
    low = cut;
    high = 0;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      if (limit[i] > 0 && limit[i] < low) low = limit[i];
      high = max(high, limit[i]);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      low = min(low, __shfl_xor(low, off));
      high = max(high, __shfl_xor(high, off));
    }
    low = __builtin_amdgcn_readfirstlane(low);
    high = __builtin_amdgcn_readfirstlane(high);
  }

  // Exponents of a page's keys (key t * 16 + g * 4 + j in s[x][t][j]) -> weights as the second product's operands;
  // un(t): the opposite powers of the values of keys t * 16 + g * 4 ...; small (the wave's): one of the page's is small.
  template <typename Un>
  __device__ __forceinline__ void weights(floatx4 (&s)[kTiles][4], int page, int g, float inv_c, bool small, Un un,
                                          halfx8 (&w)[kTiles][2]) {
    if (page < 0 || page * kPage + kPage > low) {
#pragma unroll
      for (int x = 0; x < kTiles; ++x) {
        const int lim = (page < 0 ? 0 : limit[x] - page * kPage) - g * 4;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (t * 16 + j >= lim) s[x][t][j] = -__builtin_inff();
      }
    }
    bool renewing = false;
    float top[kTiles];
#pragma unroll
    for (int x = 0; x < kTiles; ++x) {
      float a = max3(s[x][0][0], s[x][0][1], s[x][0][2]);
#pragma unroll
      for (int j = 3; j < 15; j += 2) a = max3(a, s[x][j >> 2][j & 3], s[x][(j + 1) >> 2][(j + 1) & 3]);
      top[x] = row4_max(fmaxf(a, s[x][3][3]));
      renewing = renewing || top[x] > renew[x];
    }
    if (__ballot(renewing)) {
#pragma unroll
      for (int x = 0; x < kTiles; ++x) {
        const bool need = top[x] > renew[x];
        const float by = need ? top[x] - kHeadroom : 0.f;
        const bool scales = need && renew[x] != kUnset;
        const float a = scales ? __builtin_amdgcn_exp2f(-by) : 1.f;
        float near, far;
        two_powers(scales ? -by : 0.f, near, far);
        l[x] = l[x] * near * far;
#pragma unroll
        for (int d = 0; d < kDT; ++d) acc[x][d] *= a;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[x][t][j] -= by;
        ref[x] += by;
        start[x] = -ref[x] * inv_c;
        if (need) renew[x] = kHeadroom + kSlack;
      }
    }
    uint32_t packed[kTiles][8];
    float exact[kTiles];
    if (__builtin_expect(small, false)) {
#pragma unroll
      for (int x = 0; x < kTiles; ++x) exact[x] = l[x];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const floatx4 power = un(t) * 0x1p-60f;
#pragma unroll
        for (int x = 0; x < kTiles; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) exact[x] = fmaf(__builtin_amdgcn_exp2f(s[x][t][j] + 60.f), power[j], exact[x]);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const floatx4 power = un(t);
#pragma unroll
      for (int x = 0; x < kTiles; ++x) {
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          e[j] = __builtin_amdgcn_exp2f(s[x][t][j]);
          l[x] = fmaf(e[j], power[j], l[x]);
        }
        packed[x][t * 2] = pack_half2(e[0], e[1]);
        packed[x][t * 2 + 1] = pack_half2(e[2], e[3]);
      }
    }
    if (__builtin_expect(small, false)) {
#pragma unroll
      for (int x = 0; x < kTiles; ++x) l[x] = exact[x];
    }
#pragma unroll
    for (int x = 0; x < kTiles; ++x) {
      w[x][0] = __builtin_bit_cast(halfx8, u32x4{packed[x][0], packed[x][1], packed[x][2], packed[x][3]});
      w[x][1] = __builtin_bit_cast(halfx8, u32x4{packed[x][4], packed[x][5], packed[x][6], packed[x][7]});
    }
  }

  // The lanes' sums joined; m: the reference, -inf for a row without a key, whose sums are zeros. Sums that only NaN has
  // gone into have no reference (a maximum drops NaN), but are no empty row's: a join has to take them.
  __device__ __forceinline__ void finish(float (&m)[kTiles]) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      l[i] = row4_sum(l[i]);
      m[i] = renew[i] == kUnset && l[i] == l[i] ? -__builtin_inff() : ref[i];
      if (limit[i] == 0) {  // no key, or no row: pages that all counting rows see were not masked for it
        m[i] = -__builtin_inff();
        l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < kDT; ++d) acc[i][d] = floatx4{0, 0, 0, 0};
      }
    }
  }

  // The other waves' sums, joined by the first; `shared` holds kWaves - 1 times [kTiles * 16][D + 2].
  template <int kWaves>
  __device__ __forceinline__ void join_waves(float (&m)[kTiles], float *shared, int wave, int col, int g) {
    constexpr int D = kDT * 16;
    typedef float Sums[kTiles * 16][D + 2];
    Sums *others = reinterpret_cast<Sums *>(shared);
    __syncthreads();  // the query operands have been read
    if (wave > 0) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        float *dst = others[wave - 1][i * 16 + col];
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
    if (wave > 0) return;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      float mx = m[i];
#pragma unroll
      for (int x = 1; x < kWaves; ++x) mx = fmaxf(mx, others[x - 1][i * 16 + col][D]);
      const float a = m[i] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m[i] - mx);
      float near, far;
      two_powers(m[i] == -__builtin_inff() ? 0.f : m[i] - mx, near, far);
      l[i] = l[i] * near * far;
#pragma unroll
      for (int d = 0; d < kDT; ++d) acc[i][d] *= a;
#pragma unroll
      for (int x = 1; x < kWaves; ++x) {
        const float *src = others[x - 1][i * 16 + col];
        const float mo = src[D];
        const float c = mo == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mo - mx);
        two_powers(mo == -__builtin_inff() ? 0.f : mo - mx, near, far);
        l[i] = fmaf(src[D + 1] * far, near, l[i]);
#pragma unroll
        for (int d = 0; d < kDT; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][d][j] = fmaf(src[d * 16 + g * 4 + j], c, acc[i][d][j]);
      }
      m[i] = mx;
    }
  }

  // Results of unit rows first + 16 i + col, or this part's share of them.
  template <typename Q>
  __device__ __forceinline__ void store(const AttnParams &p, const Work &w, int first, int col, int g, const float (&m)[kTiles]) {
    constexpr int D = kDT * 16;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int r = first + i * 16 + col;
      if (r >= p.rows) continue;
      const int tl = r / p.G, gh = r - tl * p.G;
      const int64_t t = w.t0 + tl;
      if (t >= p.T) continue;
      if (p.parts == 1) {
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        Q *dst = static_cast<Q *>(p.o) + w.b * p.osb + (static_cast<int64_t>(w.h) * p.G + gh) * p.osh + t * p.ost + g * 4;
#pragma unroll
        for (int d = 0; d < kDT; ++d) {
          struct alignas(8) Four { Q v[4]; } out;
#pragma unroll
          for (int j = 0; j < 4; ++j) out.v[j] = from_f32<Q>(acc[i][d][j] * inv);
          *reinterpret_cast<Four *>(dst + d * 16) = out;
        }
      } else {
        // [unit row][part][D], behind them (m, l) alike
        const int64_t at = (w.unit_row * p.rows + r) * p.parts + w.part;
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
};

// Joins the parts of each row: D/4 lanes a row, four features each. Up to kFewParts parts one group of lanes takes them in
// turn and a workgroup has a row a group; beyond, the groups of a workgroup share one row's parts, four in flight each (one
// group took 40 us for 100 parts, each waiting for the one before).
constexpr int kFewParts = 12;

template <typename Q, int D, bool kShare>
__global__ __launch_bounds__(256) void cache_join_kernel(const AttnParams p) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ float sums[kShare ? kGroups : 1][kShare ? D + 2 : 1];
  const int grp = threadIdx.x / kLanes, d = (threadIdx.x % kLanes) * 4;
  const int64_t row = kShare ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * kGroups + grp;
  const int64_t all = p.B * p.H * p.U * static_cast<int64_t>(p.rows);
  if (row >= all) return;  // kShare: never
  const int64_t unit = row / p.rows;
  const int r = static_cast<int>(row - unit * p.rows), tl = r / p.G, gh = r - tl * p.G;
  const int u = static_cast<int>(unit % p.U);
  const int64_t bh = unit / p.U, b = bh / p.H, h = bh - b * p.H;
  const int64_t t = static_cast<int64_t>(p.u0 + u) * p.block_q + tl;
  if (t >= p.T) return;  // the same for a whole workgroup where it shares a row
  const float *o = p.ws + row * p.parts * D + d;
  const float *ml = p.ws + all * p.parts * D + row * p.parts * 2;
  constexpr int kStep = kShare ? kGroups : 1;
  floatx4 acc = {0, 0, 0, 0};
  float l = 0.f, mx = -__builtin_inff();
  for (int i0 = kShare ? grp : 0; i0 < p.parts; i0 += 4 * kStep) {
    float m[4], ls[4];
    floatx4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * kStep;
      const bool in = i < p.parts;
      m[k] = in ? ml[i * 2] : -__builtin_inff();
      ls[k] = in ? ml[i * 2 + 1] : 0.f;
      x[k] = in ? *reinterpret_cast<const floatx4 *>(o + static_cast<int64_t>(i) * D) : floatx4{0, 0, 0, 0};
    }
    const float top = fmaxf(mx, fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
    if (top == -__builtin_inff()) continue;
    float near, far;
    two_powers(mx - top, near, far);
    l = l * near * far;
    acc *= __builtin_amdgcn_exp2f(mx - top);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      two_powers(m[k] - top, near, far);
      l = fmaf(ls[k] * far, near, l);
      acc += x[k] * __builtin_amdgcn_exp2f(m[k] - top);
    }
    mx = top;
  }
  if constexpr (kShare) {
    *reinterpret_cast<float2 *>(&sums[grp][d]) = float2{acc[0], acc[1]};
    *reinterpret_cast<float2 *>(&sums[grp][d + 2]) = float2{acc[2], acc[3]};
    if (d == 0) {
      sums[grp][D] = mx;
      sums[grp][D + 1] = l;
    }
    __syncthreads();
    if (grp > 0) return;
    float top = mx;
#pragma unroll
    for (int i = 1; i < kGroups; ++i) top = fmaxf(top, sums[i][D]);
    if (top > -__builtin_inff()) {
      float near, far;
      two_powers(mx - top, near, far);
      l = l * near * far;
      acc *= __builtin_amdgcn_exp2f(mx - top);
#pragma unroll
      for (int i = 1; i < kGroups; ++i) {
        const float w = __builtin_amdgcn_exp2f(sums[i][D] - top);
        two_powers(sums[i][D] - top, near, far);
        l = fmaf(sums[i][D + 1] * far, near, l);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(sums[i][d + j], w, acc[j]);
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  struct alignas(8) Four { Q v[4]; } out;
#pragma unroll
  for (int j = 0; j < 4; ++j) out.v[j] = from_f32<Q>(acc[j] * inv);
  *reinterpret_cast<Four *>(static_cast<Q *>(p.o) + b * p.osb + (h * p.G + gh) * p.osh + t * p.ost + d) = out;
}

struct Shape {
  int kind;   // 16 rows a wave, 32, or 64 or 128 a workgroup
  int parts;
  double us;  // estimated
};

// Few rows (up to 32) or many (64, 128), and how many workgroups share a unit's pages: as many as one to four rounds of
// resident workgroups take (their registers allow 4 to 2 on a CU), or one, whichever is estimated to take least. Measured,
// in us: a wave's page where few run 0.3 (many rows, three workgroups a CU: 2.5; D = 128, two: 3), the start of a round
// 3, the join 4 and 0.25 a MB of sums. A last round that is not full takes as long as the others. With other parts than the
// rule's, in us: 144 units of a frame (the rule takes 5) 234 with 5, 279 with 4, 289 with 6, 237 with 10, 259 with 16;
// a causal chunk of 128 units (4) 208 with 4, 303 with 2, 219 with 8; 128 units of single tokens, 258 pages (4) 108 with 4,
// 138 with 1, 107 with 2, 112 with 8; of 521 pages (8) 85 with 8, 82 with 4, 83 with 16. The pages are the list's width or the
// table's, as the lengths are on the device: short sequences in a long table leave parts empty. The 0.3 holds where the loads
// of all CUs' waves overlap; a page by itself takes longer: 16 units of 18 pages, five to a wave, 10 us where the estimate says
// 4.5.
Shape attn_shape(int64_t units, int64_t rows, int64_t pages, int64_t D) {
  Shape s;
  s.kind = rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
  const int64_t resident = 256 * (D == 128 ? 2 : s.kind == 0 ? 4 : 3);
  const int64_t waves = s.kind < 2 ? 4 : 1;  // that share a workgroup's pages
  const double page_us = s.kind < 2 ? 0.3 : D == 128 ? 3.0 : 2.5, part_mb = static_cast<double>(units * rows * D) * 4e-6;
  double best = 0;
  s.parts = 0;
  for (int64_t rounds = 0; rounds <= 4; ++rounds) {
    int64_t parts = rounds == 0 ? 1 : rounds * resident / units;
    if (parts < 1) continue;
    if (parts > 256) parts = 256;
    const int64_t share = cdiv(cdiv(pages, parts), waves);  // pages of a wave
    parts = cdiv(pages, share * waves);                     // the fewest with that share
    const double us = cdiv(units * parts, resident) * (share * page_us + 3.0) + (parts > 1 ? 4.0 + 0.25 * parts * part_mb : 0.0);
    if (s.parts == 0 || us < best) {
      best = us;
      s.parts = static_cast<int>(parts);
    }
  }
  s.us = best;
  return s;
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

template <typename Q, int D>
int launch_join(const AttnParams &p, const Shape &s, hipStream_t st, const char *what) {
  if (s.parts == 1) return VASC_OK;
  const int64_t rows = p.B * p.H * p.U * static_cast<int64_t>(p.rows);
  if (s.parts > kFewParts && rows < (int64_t(1) << 16))
    hipLaunchKernelGGL((cache_join_kernel<Q, D, true>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((cache_join_kernel<Q, D, false>), dim3(static_cast<unsigned>(cdiv(rows, 256 / (D / 4)))), dim3(256), 0, st, p);
  return check_launch(what);
}

// Checks a call's arguments and fills what the kernels take (but vo, the parts and the workspace), for one launch.
int attn_params(const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st, void *o, int64_t o_sb, int64_t o_sh, int64_t o_st,
                int64_t B, int64_t Hq, int64_t H, int64_t T, int64_t D, int32_t dtype, const uint8_t *kc, const uint8_t *vc,
                const uint8_t *ks, const uint8_t *vs, int64_t pages, const int32_t *page_table, int64_t table_stride,
                int64_t max_pages, const int32_t *lengths, const int32_t *q_count, int64_t block_q, const int32_t *index,
                int64_t width, const int32_t *count, int32_t causal, float scale, AttnParams &p) {
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
  p.q = q; p.qsb = q_sb; p.qsh = q_sh; p.qst = q_st;
  p.o = o; p.osb = o_sb; p.osh = o_sh; p.ost = o_st;
  p.B = B; p.T = T;
  p.H = static_cast<int>(H);
  p.G = static_cast<int>(Hq / H);
  p.U = p.list_U = static_cast<int>(cdiv(T, block_q));
  p.kc = kc; p.vc = vc; p.ks = ks; p.vs = vs; p.pages = pages;
  p.table = page_table; p.table_stride = table_stride; p.max_pages = max_pages;
  p.lengths = lengths; p.n_q = q_count;
  p.block_q = static_cast<int>(block_q);
  p.causal = causal;
  p.index = index; p.width = width; p.count = count;
  VASC_REQUIRE(scale - scale == 0.f && (scale == 0.f || (fabsf(scale) > 1e-30f && fabsf(scale) < 1e30f)),
               "scale must be 0 or of magnitude 1e-30 to 1e30");
  // the reference is divided by c: a scale of 0 is one too small to show
  p.c = scale == 0.f ? 1e-30f : scale * 1.4426950408889634f;
  p.rows = p.block_q * p.G;
  return VASC_OK;
}

// What a launch over p.U units takes of the workspace, from `used` bytes of it on.
int take_workspace(AttnParams &p, const Shape &s, int64_t D, void *workspace, int64_t given, int64_t &used) {
  const int64_t units = p.B * p.H * p.U;
  p.parts = s.parts;
  VASC_REQUIRE(units < (int64_t(1) << 31) / s.parts, "too many units");
  VASC_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "the workspace must be 16-byte aligned");
  const int64_t need = workspace_bytes(units, p.rows, D, s.parts);
  VASC_REQUIRE(need == 0 || (workspace && given >= used + need), "workspace of %lld bytes, %lld needed", (long long)given,
               (long long)(used + need));
  p.ws = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + used);
  used += (need + 15) / 16 * 16;
  return VASC_OK;
}

}  // namespace
}  // namespace vasc
