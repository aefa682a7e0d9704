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
#include "cache_attn.h"

namespace vasc {
namespace {

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
      query_operands<Q, D, 16>(p, w, t, gh, rows.limit[i] > 0, g, ops);
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

  rows.template join_waves<kWaves>(m, reinterpret_cast<float *>(shared), wave, col, g);
  if (wave == 0) rows.template store<Q>(p, w, 0, col, g, m);
}

// Many rows (up to 128): neither the vector nor the matrix pipe is full (63 % and 27 % of a frame's cycles); a page's chain of
// dependent steps binds, at two or three waves a SIMD. The kWaves waves lie side by side over the rows, and
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
    query_operands<Q, D, 16>(p, w, t, gh, rows.limit[i] > 0, g, query[i]);
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
  return rc ? rc : launch_join<Q, D>(p, s, st, "vasc_cache_attn");
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
  AttnParams p = {};
  int rc = attn_params(q, q_sb, q_sh, q_st, o, o_sb, o_sh, o_st, B, Hq, H, T, D, dtype, kc, vc, ks, vs, pages, page_table,
                       table_stride, max_pages, lengths, q_count, block_q, index, width, count, causal, scale, p);
  if (rc) return rc;
  const Shape s = attn_shape(B * H * p.U, p.rows, width ? width : max_pages, D);
  int64_t used = 0;
  if ((rc = take_workspace(p, s, D, workspace, workspace_bytes_given, used))) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (D == 64) return dtype == 0 ? launch_attn<__bf16, 64>(p, s, st) : launch_attn<_Float16, 64>(p, s, st);
  return dtype == 0 ? launch_attn<__bf16, 128>(p, s, st) : launch_attn<_Float16, 128>(p, s, st);
}
