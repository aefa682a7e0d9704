// Attention over listed pages of the 8-bit block cache.
//
// A unit's query rows (block_q tokens x G heads of one key head) are the
// columns of S^T = K Q^T, 16 to a tile. A 16-key tile is the A operand of
// 16x16x32 products, lane l holding 16 consecutive features of key l & 15: its
// codes are widened to bfloat16 in registers by a conversion that takes the
// key's power of two along (exact: e4m3 times 2^-60..60). Float16 queries are
// two bfloat16 parts (8 and 3 of their 11 bits), a product each. (The 8-bit
// matrix products would save the widening, but keep only some 14 bits of a
// sum: measured, an error of 2^-13 to 2^-16 of sum |q k|.)
// S^T leaves each lane four consecutive keys of one query row, which is what
// the second product's B operand wants of P^T; the cache holds V transposed
// with the tokens in that same order, so V too goes from memory to the matrix
// pipe without a shuffle, widened to half on the way (exact).
//
// A value row's power 2^ev enters the softmax's exponent, e = c S + ev, so the
// weights of the second product are w = 2^(e - ref) and its sum takes them
// without the power: l = sum w 2^-ev. The reference is the accumulator's start:
// S begins at -ref / c, and c S' + ev is the exponent. It is set 11 below the
// row's largest e and renewed only when that has grown by more than 4: weights
// are held in half (11 bits; bfloat16's 8 would be the largest error of a
// float16 result) up to 2^15, and those below its range are under 2^-36 of the
// row's largest.
//
// A key whose value row is small may be lost in the second product and yet be
// most of l: its w = 2^(e - ref) may lie under float32's 2^-126. With every
// exponent at -30 or more, what is lost of l is below 2^-47 of it a key (w of
// the row's largest is 2^11, its part of l 2^(11 - ev), ev at most 60). Pages
// that hold a smaller one (rows of zeros have -60) take w 2^60 and 2^(-60 - ev)
// for l instead, an exponential more a key; and l is scaled in two factors.
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
  int H, G, U;
  const uint8_t *kc, *vc, *ks, *vs;
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

// Eight e4m3 codes as halves.
__device__ __forceinline__ uint32_t two_halves(uint32_t w, bool hi) {
  return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
}
__device__ __forceinline__ halfx8 widen(uint32_t a, uint32_t b) {
  const u32x4 w = {two_halves(a, false), two_halves(a, true), two_halves(b, false), two_halves(b, true)};
  return __builtin_bit_cast(halfx8, w);
}

// Eight e4m3 codes times a power of two, as bfloat16.
__device__ __forceinline__ uint32_t two_scaled(uint32_t w, float power, bool hi) {
  return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, power, true)
                                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, power, false));
}
__device__ __forceinline__ bf16x8 widen_scaled(uint32_t a, uint32_t b, float power) {
  const u32x4 w = {two_scaled(a, power, false), two_scaled(a, power, true), two_scaled(b, power, false),
                   two_scaled(b, power, true)};
  return __builtin_bit_cast(bf16x8, w);
}

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
  int id = static_cast<int>(xcd_remap(blockIdx.x, gridDim.x));
  w.u = id % p.U;
  id /= p.U;
  w.part = id % p.parts;
  const int bh = id / p.parts;
  w.b = bh / p.H;
  w.h = bh - static_cast<int>(w.b) * p.H;
  w.L = p.lengths[w.b];
  w.nq = p.n_q ? p.n_q[w.b] : p.T;
  w.nq = w.nq < 0 ? 0 : (w.nq < p.T ? w.nq : p.T);
  w.t0 = static_cast<int64_t>(w.u) * p.block_q;
  w.t1 = w.t0 + p.block_q < w.nq ? w.t0 + p.block_q : w.nq;
  const UnitView view = unit_view(w.L, w.nq, w.t0, w.t1, p.max_pages, p.causal);
  w.cut = static_cast<int>(clamp_tokens(w.L, p.max_pages));  // below 2^30
  w.seen = static_cast<int>(view.seen);
  w.unit_row = static_cast<int64_t>(bh) * p.U + w.u;
  w.entries = w.seen;
  w.list = nullptr;
  if (p.index) {
    w.list = p.index + w.unit_row * p.width;
    const int64_t n = p.count[w.unit_row];
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

// This lane's query operands of a row: [part][product]; zeros where there is no row. An infinite query has no softmax, whatever
// the sign of its logits, which a running maximum would not see where all of them are minus infinity: it goes as NaN.
template <typename Q, int D, int kOps>
__device__ __forceinline__ void query_operands(const AttnParams &p, const Work &w, int64_t t, int gh, bool live, int g,
                                               bf16x8 (&out)[kOps]) {
  constexpr int kMul = D / 32, kParts = kOps / kMul;
  const Q *src = static_cast<const Q *>(p.q) + w.b * p.qsb + (static_cast<int64_t>(w.h) * p.G + gh) * p.qsh + t * p.qst + g * 16;
#pragma unroll
  for (int y = 0; y < kMul; ++y) {
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (live) {
      struct alignas(16) Eight { Q v[8]; };
      const Eight v = *reinterpret_cast<const Eight *>(src + (y >> 1) * 64 + (y & 1) * 8);
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

// Few rows (up to 32): the cache's bytes bound the kernel. Each of the 4 waves holds all of the unit's rows, kTiles tiles of
// 16, and takes every fourth page straight from memory to its registers; their sums are joined in LDS.
// Measured: single tokens of 16 sequences, 8 x 4 heads of 128, 258 pages each, 545 MB in 105 us (5.2 TB/s; a large copy
// reaches 4.84); more and shorter parts cost more in starts than they even out (4 pages a wave: 126 us).
template <typename Q, int D, int kTiles>
__global__ __launch_bounds__(256, 2) void cache_attn_few_kernel(const AttnParams p) {
  constexpr int kWaves = 4, kDT = D / 16, kRows = kTiles * 16;
  constexpr int kK = D / 64;   // 16-byte loads of a key per lane, two products each
  constexpr int kParts = __is_same(Q, __bf16) ? 1 : 2;
  // the query operands, 16 bytes a lane: [row tile][part][product]; after the pages, the other waves' sums
  constexpr int kOps = kParts * kK * 2;
  typedef float Sums[kRows][D + 2];
  constexpr size_t kQBytes = kTiles * kOps * 1024, kSBytes = (kWaves - 1) * sizeof(Sums);
  __shared__ __align__(16) uint8_t shared[kQBytes > kSBytes ? kQBytes : kSBytes];
  bf16x8 *query = reinterpret_cast<bf16x8 *>(shared);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const Work w = work_of(p);

  Rows<kTiles, kDT> rows;
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    int64_t t;
    int gh;
    rows.limit[i] = row_limit(p, w, i * 16 + col, t, gh);
    if (wave == 0) {
      bf16x8 ops[kOps];
      query_operands<Q, D>(p, w, t, gh, rows.limit[i] > 0, g, ops);
#pragma unroll
      for (int o = 0; o < kOps; ++o) query[(i * kOps + o) * 64 + lane] = ops[o];
    }
  }
  rows.bounds(w.cut);
  rows.init();
  __syncthreads();

  const float inv_c = 1.f / p.c;
  const uint8_t *kbase = p.kc + static_cast<int64_t>(w.h) * (kPage * D) + col * D + g * 16;
  const uint8_t *vbase = p.vc + static_cast<int64_t>(w.h) * (kPage * D) + col * kPage + g * 16;
  const uint8_t *ksbase = p.ks + static_cast<int64_t>(w.h) * kPage + col * 4;
  const uint8_t *vsbase = p.vs + static_cast<int64_t>(w.h) * kPage + g * 16;
  for (int base = w.e0; base < w.e1; base += 64) {
    int page, pid;  // lane i has those of entry base + i
    resolve(p, w, base + lane, page, pid);
    const int n = min(w.e1 - base, 64);
    u32x4 kr[4][kK];
    uint32_t kb = 0;
    auto load_keys = [&](int i) {
      const int64_t at = static_cast<int64_t>(__builtin_amdgcn_readlane(pid, i)) * p.H;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int y = 0; y < kK; ++y)
          kr[t][y] = *reinterpret_cast<const u32x4 *>(kbase + at * (kPage * D) + t * 16 * D + y * 64);
      kb = *reinterpret_cast<const uint32_t *>(ksbase + at * kPage);
    };
    if (wave < n) load_keys(wave);
    for (int i = wave; i < n; i += kWaves) {
      const int lpage = __builtin_amdgcn_readlane(page, i);
      const int64_t at = static_cast<int64_t>(__builtin_amdgcn_readlane(pid, i)) * p.H;
      // the query operands are read again for every page: held over the loop they would cost 8 to 64 registers
      asm volatile("" ::: "memory");
      u32x4 vr[kDT];
#pragma unroll
      for (int d = 0; d < kDT; ++d)
        vr[d] = *reinterpret_cast<const u32x4 *>(vbase + at * (kPage * D) + d * 16 * kPage);
      const u32x4 vb = *reinterpret_cast<const u32x4 *>(vsbase + at * kPage);

      floatx4 s[kTiles][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float power = pow2_byte((kb >> (8 * t)) & 255u);
#pragma unroll
        for (int y = 0; y < kK * 2; ++y) {
          const u32x4 k = kr[t][y >> 1];
          const bf16x8 a = y & 1 ? widen_scaled(k[2], k[3], power) : widen_scaled(k[0], k[1], power);
#pragma unroll
          for (int x = 0; x < kTiles; ++x)
#pragma unroll
            for (int piece = 0; piece < kParts; ++piece) {
              const bf16x8 q = query[(x * kOps + piece * kK * 2 + y) * 64 + lane];
              const float start = rows.start[x];
              const floatx4 c = y == 0 && piece == 0 ? floatx4{start, start, start, start} : s[x][t];
              s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q, c, 0, 0, 0);
            }
        }
      }
      // the next page's keys arrive while this one's weights are made
      if (i + kWaves < n) load_keys(i + kWaves);

      // exponents, in place: the byte's bias of 127 goes with the reference
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t vw = vb[t];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float ev = static_cast<float>((vw >> (8 * j)) & 255u);
#pragma unroll
          for (int x = 0; x < kTiles; ++x) s[x][t][j] = fmaf(s[x][t][j], p.c, ev);
        }
      }
      halfx8 wt[kTiles][2];
      // bytes up to 187: 67 and more have a top bit with 0x3d, kSmall and more with 0x1f
      static_assert(kSmall + 0x1f == 128, "the bytes' test");
      uint32_t top = 0;
#pragma unroll
      for (int t = 0; t < 4; ++t) top |= (vb[t] + 0x3d3d3d3du) & ~(vb[t] + 0x1f1f1f1fu);
      rows.weights(s, lpage, g, inv_c, __ballot(top & 0x80808080u) != 0, [&](int t) {
        const uint32_t iw = 0xfefefefeu - vb[t];  // the opposite powers
        return floatx4{pow2_byte(iw & 255u), pow2_byte((iw >> 8) & 255u), pow2_byte((iw >> 16) & 255u), pow2_byte(iw >> 24)};
      }, wt);
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
        const u32x4 v = vr[d];
        const halfx8 a0 = widen(v[0], v[1]), a1 = widen(v[2], v[3]);
#pragma unroll
        for (int x = 0; x < kTiles; ++x) {
          rows.acc[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, wt[x][0], rows.acc[x][d], 0, 0, 0);
          rows.acc[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, wt[x][1], rows.acc[x][d], 0, 0, 0);
        }
      }
    }
  }
  float m[kTiles];
  rows.finish(m);

  // the other waves' sums, joined by the first
  Sums *others = reinterpret_cast<Sums *>(shared);
  __syncthreads();  // the query operands have been read
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      float *dst = others[wave - 1][i * 16 + col];
      if (g == 0) {
        dst[D] = m[i];
        dst[D + 1] = rows.l[i];
      }
#pragma unroll
      for (int d = 0; d < kDT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[d * 16 + g * 4 + j] = rows.acc[i][d][j];
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
    rows.l[i] = rows.l[i] * near * far;
#pragma unroll
    for (int d = 0; d < kDT; ++d) rows.acc[i][d] *= a;
#pragma unroll
    for (int x = 1; x < kWaves; ++x) {
      const float *src = others[x - 1][i * 16 + col];
      const float mo = src[D];
      const float c = mo == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mo - mx);
      two_powers(mo == -__builtin_inff() ? 0.f : mo - mx, near, far);
      rows.l[i] = fmaf(src[D + 1] * far, near, rows.l[i]);
#pragma unroll
      for (int d = 0; d < kDT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) rows.acc[i][d][j] = fmaf(src[d * 16 + g * 4 + j], c, rows.acc[i][d][j]);
    }
    m[i] = mx;
  }
  rows.template store<Q>(p, w, 0, col, g, m);
}

// Many rows (up to 128): the vector and matrix pipes bound the kernel. The kWaves waves lie side by side over the rows, and
// a page is widened once for all of them: each wave turns its share of the codes into operands in LDS (keys as bfloat16 with
// their powers, values as half, and the values' exponents as floats), 16 bytes a lane in the order in which they are read.
// Two buffers and one barrier a page: the next page's codes are on their way to registers while this one is computed.
// Measured: a frame of 1041 queries over 522 of 2082 pages, 16 heads of 64, 142 GFLOP in 229 us with the join (620 TFLOP/s);
// 250 causal tokens of 32 heads of 128 over 20001, 163 GFLOP in 196 us (830). A wave's page (32 rows, D = 64) takes some
// 1800 cycles: some 220 vector instructions, 32 of them exp2, and 32 matrix ones; the same mix from registers alone takes 1110
// with three waves a SIMD, the matrix pipe by itself 516. The widening is 16 of them; the softmax's care is most: a maximum of
// 16 exponents a row (16 max3, two steps between lanes a tile, a ballot), 32 multiply-adds for the scale and the values' powers
// and 32 for the sum. The library's attention over bf16 blocks does the same tile without these in 943 cycles (no maximum a
// block, sums as matrix products, four waves a SIMD). Also built, while the kernel took 248 us, and no faster: values widened
// with their powers and weights summed by a product with ones (253 us, D = 128 slower), the next page's first product beside
// this page's exponentials (registers leave two waves a SIMD: 245 us), 64 rows a wave (265 us). All three kept the maximum.
template <typename Q, int D, int kTiles, int kWaves>
__global__ __launch_bounds__(kWaves * 64, D == 64 && kWaves == 4 ? 3 : 2) void cache_attn_many_kernel(const AttnParams p) {
  constexpr int kDT = D / 16, kK = D / 64, kMul = kK * 2;
  constexpr int kParts = __is_same(Q, __bf16) ? 1 : 2;
  constexpr int kOps = kParts * kMul;
  constexpr int kKeyTasks = 4 * kK, kTasks = (kKeyTasks + kDT) / kWaves;  // 1 KB of codes each: a key tile's half, a feature tile
  struct Page {
    bf16x8 k[4 * kMul][64];
    halfx8 v[kDT * 2][64];
    float ev[kPage], un[kPage];
    int small;
  };
  __shared__ __align__(16) Page buffer[2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const Work w = work_of(p);
  const int first = wave * kTiles * 16;

  Rows<kTiles, kDT> rows;
  bf16x8 query[kTiles][kOps];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    int64_t t;
    int gh;
    rows.limit[i] = row_limit(p, w, first + i * 16 + col, t, gh);
    query_operands<Q, D>(p, w, t, gh, rows.limit[i] > 0, g, query[i]);
  }
  rows.bounds(w.cut);
  rows.init();

  const float inv_c = 1.f / p.c;
  const int64_t head = static_cast<int64_t>(w.h) * (kPage * D);
  u32x4 raw[kTasks];
  uint32_t kb[kTasks], vb = 0;
  int turn = 0;
  for (int base = w.e0; base < w.e1; base += 64) {
    int page, pid;  // lane i has those of entry base + i
    resolve(p, w, base + lane, page, pid);
    const int n = min(w.e1 - base, 64);
    auto load = [&](int i) {
      const int64_t at = static_cast<int64_t>(__builtin_amdgcn_readlane(pid, i)) * p.H;
#pragma unroll
      for (int k = 0; k < kTasks; ++k) {
        const int task = wave + k * kWaves;
        if (task < kKeyTasks) {
          const int t = task / kK, y = task % kK;
          raw[k] = *reinterpret_cast<const u32x4 *>(p.kc + at * (kPage * D) + head + (t * 16 + col) * D + y * 64 + g * 16);
          kb[k] = p.ks[(at + w.h) * kPage + col * 4 + t];
        } else {
          const int d = task - kKeyTasks;
          raw[k] = *reinterpret_cast<const u32x4 *>(p.vc + at * (kPage * D) + head + (d * 16 + col) * kPage + g * 16);
        }
      }
      if (wave == 0) vb = p.vs[(at + w.h) * kPage + lane];
    };
    load(0);
    for (int i = 0; i < n; ++i) {
      Page &buf = buffer[turn];
      turn ^= 1;
#pragma unroll
      for (int k = 0; k < kTasks; ++k) {
        const int task = wave + k * kWaves;
        const u32x4 x = raw[k];
        if (task < kKeyTasks) {
          const float power = pow2_byte(kb[k]);
          buf.k[task * 2][lane] = widen_scaled(x[0], x[1], power);
          buf.k[task * 2 + 1][lane] = widen_scaled(x[2], x[3], power);
        } else {
          const int d = task - kKeyTasks;
          buf.v[d * 2][lane] = widen(x[0], x[1]);
          buf.v[d * 2 + 1][lane] = widen(x[2], x[3]);
        }
      }
      if (wave == 0) {
        buf.ev[lane] = static_cast<float>(vb);  // the bias of 127 goes with the reference
        buf.un[lane] = pow2_byte(254u - vb);
        const uint64_t small = __ballot(vb - 1u < kSmall - 1u);
        if (lane == 0) buf.small = small != 0;
      }
      __syncthreads();
      if (i + 1 < n) load(i + 1);
      if (rows.high == 0) continue;
      const int lpage = __builtin_amdgcn_readlane(page, i);

      floatx4 s[kTiles][4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int y = 0; y < kMul; ++y) {
          const bf16x8 a = buf.k[t * kMul + y][lane];
#pragma unroll
          for (int x = 0; x < kTiles; ++x)
#pragma unroll
            for (int piece = 0; piece < kParts; ++piece) {
              const float start = rows.start[x];
              const floatx4 c = y == 0 && piece == 0 ? floatx4{start, start, start, start} : s[x][t];
              s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, query[x][piece * kMul + y], c, 0, 0, 0);
            }
        }
      // The softmax goes before the other waves' products: the matrix pipe works on while its instructions are issued. Measured
      // in turn on one card: the frame above 241 us without, 230 with, the causal chunk 202 and 194.
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const floatx4 ev = *reinterpret_cast<const floatx4 *>(buf.ev + g * 16 + t * 4);
#pragma unroll
        for (int x = 0; x < kTiles; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[x][t][j] = fmaf(s[x][t][j], p.c, ev[j]);
      }
      halfx8 wt[kTiles][2];
      rows.weights(s, lpage, g, inv_c, __builtin_amdgcn_readfirstlane(buf.small),
                   [&](int t) { return *reinterpret_cast<const floatx4 *>(buf.un + g * 16 + t * 4); }, wt);
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
        const halfx8 a0 = buf.v[d * 2][lane], a1 = buf.v[d * 2 + 1][lane];
#pragma unroll
        for (int x = 0; x < kTiles; ++x) {
          rows.acc[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, wt[x][0], rows.acc[x][d], 0, 0, 0);
          rows.acc[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, wt[x][1], rows.acc[x][d], 0, 0, 0);
        }
      }
    }
  }
  float m[kTiles];
  rows.finish(m);
  rows.template store<Q>(p, w, first, col, g, m);
}

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
  const int64_t t = static_cast<int64_t>(u) * p.block_q + tl;
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
};

// Few rows (up to 32) or many (64, 128), and how many workgroups share a unit's pages: as many as one to four rounds of
// resident workgroups take (their registers allow 4 to 2 on a CU), or one, whichever is estimated to take least. Measured,
// in us: a wave's page where few run 0.3 (many rows, three workgroups a CU: 2.5; D = 128, two: 3), the start of a round
// 3, the join 4 and 0.25 a MB of sums. A last round that is not full takes as long as the others. With other parts than the
// rule's, in us: 144 units of a frame (the rule takes 5) 234 with 5, 279 with 4, 289 with 6, 237 with 10, 259 with 16;
// a causal chunk of 128 units (4) 208 with 4, 303 with 2, 219 with 8; 128 units of single tokens, 258 pages (4) 108 with 4,
// 138 with 1, 107 with 2, 112 with 8; of 521 pages (8) 85 with 8, 82 with 4, 83 with 16. The pages are the list's width or the
// table's, as the lengths are on the device: short sequences in a long table leave parts empty.
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
  return s;
}

template <typename Q, int D>
int launch_attn(const AttnParams &p, const Shape &s, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.B * p.H * p.U * s.parts));
  // float16 queries of 128 features are two operands: 16 rows a wave
  constexpr int kWaves = D == 128 && !__is_same(Q, __bf16) ? 8 : 4;
  switch (s.kind) {
    case 0: hipLaunchKernelGGL((cache_attn_few_kernel<Q, D, 1>), grid, dim3(256), 0, st, p); break;
    case 1: hipLaunchKernelGGL((cache_attn_few_kernel<Q, D, 2>), grid, dim3(256), 0, st, p); break;
    case 2: hipLaunchKernelGGL((cache_attn_many_kernel<Q, D, 1, 4>), grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL((cache_attn_many_kernel<Q, D, 8 / kWaves, kWaves>), grid, dim3(kWaves * 64), 0, st, p); break;
  }
  int rc = check_launch("vasc_cache_attn");
  if (rc || s.parts == 1) return rc;
  const int64_t rows = p.B * p.H * p.U * static_cast<int64_t>(p.rows);
  if (s.parts > kFewParts && rows < (int64_t(1) << 16))
    hipLaunchKernelGGL((cache_join_kernel<Q, D, true>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((cache_join_kernel<Q, D, false>), dim3(static_cast<unsigned>(cdiv(rows, 256 / (D / 4)))), dim3(256), 0, st, p);
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
  return workspace_bytes(units, rows, D, attn_shape(units, rows, width ? width : max_pages, D).parts);
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
  VASC_REQUIRE(scale - scale == 0.f && (scale == 0.f || (fabsf(scale) > 1e-30f && fabsf(scale) < 1e30f)),
               "scale must be 0 or of magnitude 1e-30 to 1e30");
  // the reference is divided by c: a scale of 0 is one too small to show
  p.c = scale == 0.f ? 1e-30f : scale * 1.4426950408889634f;
  p.rows = p.block_q * p.G;
  const int64_t units = B * H * p.U;
  const Shape s = attn_shape(units, p.rows, width ? width : max_pages, D);
  p.parts = s.parts;
  VASC_REQUIRE(units < (int64_t(1) << 31) / s.parts, "too many units");
  const int64_t need = workspace_bytes(units, p.rows, D, s.parts);
  VASC_REQUIRE(need == 0 || (workspace && workspace_bytes_given >= need), "workspace of %lld bytes, %lld needed",
               (long long)workspace_bytes_given, (long long)need);
  VASC_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "the workspace must be 16-byte aligned");
  p.ws = static_cast<float *>(workspace);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (D == 64) return dtype == 0 ? launch_attn<__bf16, 64>(p, s, st) : launch_attn<_Float16, 64>(p, s, st);
  return dtype == 0 ? launch_attn<__bf16, 128>(p, s, st) : launch_attn<_Float16, 128>(p, s, st);
}
