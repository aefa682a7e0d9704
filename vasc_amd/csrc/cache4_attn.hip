// Attention over listed pages of the 4-bit block cache: the mathematics, the units, the softmax and the join are those of
// the 8-bit cache (cache_attn.hip, cache_attn.h); the pages' form is another.
//
// A lane's 16 bytes hold 32 e2m1 codes. Of the keys they are the features that one lane supplies to a product's A operand:
// at D = 128 32 consecutive features of one key, one group under one power; at D = 64 16 of each of two key tiles. A
// conversion widens two codes to bfloat16 and takes the group's power along (exact: two significant bits times 2^-60..60).
// Of the values, transposed, they are 16 tokens of each of two features 16 apart, which lie in one group of 32. A token's
// row has its largest group's power in the softmax's exponent, as the 8-bit cache; what a group lies below that, 0 to 14
// powers of two, goes to the widened values by packed half products, exact as well (e2m1 has two significant bits, half
// reaches down to 2^-24). The other place for it, the weights, would lose bits of those.
#include "cache_attn.h"

namespace vasc {
namespace {

// Eight e2m1 codes times a power of two, as bfloat16.
template <int kByte>
__device__ __forceinline__ uint32_t two_scaled4(uint32_t w, float power) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, kByte));
}
__device__ __forceinline__ bf16x8 widen4_scaled(uint32_t w, float power) {
  const u32x4 x = {two_scaled4<0>(w, power), two_scaled4<1>(w, power), two_scaled4<2>(w, power), two_scaled4<3>(w, power)};
  return __builtin_bit_cast(bf16x8, x);
}

// Eight powers of two as halves: 2^(n - 15) of the nibbles n of a word, those of the even places in its low half.
__device__ __forceinline__ halfx8 powers8(uint32_t w) {
  const u32x4 x = {(w << 10) & 0x3c003c00u, (w << 6) & 0x3c003c00u, (w << 2) & 0x3c003c00u, (w >> 2) & 0x3c003c00u};
  return __builtin_bit_cast(halfx8, x);
}

// Eight e2m1 codes times those, as halves.
template <int kByte>
__device__ __forceinline__ uint32_t two_halves4(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, kByte));
}
__device__ __forceinline__ halfx8 widen4(uint32_t w, const halfx8 &power) {
  const u32x4 x = {two_halves4<0>(w), two_halves4<1>(w), two_halves4<2>(w), two_halves4<3>(w)};
  return __builtin_bit_cast(halfx8, x) * power;
}

// A lane's 16 bytes of each kilobyte. kOnce: the call has one unit a head, so a sequence's pages are read once, and go past the
// caches. Measured with plain loads and so, in us: single tokens of 16 sequences up to 131072 long 285 and 253; calls again and
// again over 1 to 145 MB of codes the same to 3%, over 519 MB 102 and 92, and after the caches were emptied 5 MB 15.0 and 14.2,
// 36 MB 27 and 21.5, 145 MB 71 and 46. Units that share pages want the caches (eight of 16 tokens 32.2 and 34.1), and so do
// branches of one parent, whose tables the host does not see: eight each of four, 16384 tokens long, 80 and 82 (D = 64: 95 and
// 100), 100000 long 438 and 443 to 455, 32 of one 181 and 190.
template <bool kOnce, int n>
__device__ __forceinline__ void load_codes(u32x4 (&x)[n], const uint8_t *at) {
  if constexpr (kOnce) {
#pragma unroll
    for (int y = 0; y < n; ++y) x[y] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(at + y * 1024));
  } else {
#pragma unroll
    for (int y = 0; y < n; ++y) x[y] = *reinterpret_cast<const u32x4 *>(at + y * 1024);
  }
}

// Few rows (up to 32): the cache's bytes bound the kernel. Each of the 4 waves holds all of the unit's rows, kTiles tiles of
// 16, and takes every fourth page straight from memory to its registers; their sums are joined in LDS.
// Measured: single tokens of 16 sequences of 39000 to 131072 tokens, 8 x 4 heads of 128, 1.46 GB in 254 us (5.8 TB/s).
template <typename Q, int D, int kTiles, bool kOnce>
__global__ __launch_bounds__(256, 2) void cache4_attn_few_kernel(const AttnParams p) {
  constexpr int kWaves = 4, kDT = D / 16, kRows = kTiles * 16;
  constexpr int kG = D / 32;   // groups of a row; 16-byte loads of a page's keys, or values, per lane; products of a key tile
  constexpr int kParts = __is_same(Q, __bf16) ? 1 : 2;
  constexpr int kOps = kParts * kG;
  // Pages of a wave on their way. D = 128: single tokens of 16 sequences over up to 131072 keys (8 x 4 heads) 268 us with one,
  // 254 with two. At D = 64 two cost a wave a SIMD: eight sequences of up to 33312 tokens 45.0 us with one, 50.5 with two.
  constexpr int kAhead = D == 128 && kTiles == 1 ? 2 : 1;
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
      query_operands<Q, D, D / 4>(p, w, t, gh, rows.limit[i] > 0, g, ops);
#pragma unroll
      for (int o = 0; o < kOps; ++o) query[(i * kOps + o) * 64 + lane] = ops[o];
    }
  }
  rows.bounds(w.cut);
  rows.init();
  __syncthreads();

  const float inv_c = 1.f / p.c;
  const int64_t h = w.h;
  const int chunk = (col * 4 + g) * 16;  // this lane's 16 bytes of a kilobyte
  const uint8_t *kbase = p.kc + h * (kPage * D / 2) + chunk;
  const uint8_t *vbase = p.vc + h * (kPage * D / 2) + chunk;
  const uint8_t *ksbase = p.ks + h * (kPage * kG) + (D == 128 ? g : g >> 1) * kPage + col * 4;
  const uint8_t *vsbase = p.vs + h * kPage + g * 16;
  const uint8_t *vobase = p.vo + h * (kG * 32) + g * (kG * 8);
  for (int base = w.e0; base < w.e1; base += 64) {
    int page, pid;  // lane i has those of entry base + i
    resolve(p, w, base + lane, page, pid);
    const int n = min(w.e1 - base, 64);
    // a page is asked for as soon as the one before it in its place has been used
    struct Raw {
      u32x4 kr[kG], vr[kG], vp[kG / 2], vb;
      uint32_t kb;
    } ahead[kAhead];
    auto load_keys = [&](int i, Raw &r) {
      const int64_t at = static_cast<int64_t>(__builtin_amdgcn_readlane(pid, i)) * p.H;
      load_codes<kOnce>(r.kr, kbase + at * (kPage * D / 2));
      r.kb = *reinterpret_cast<const uint32_t *>(ksbase + at * (kPage * kG));
    };
    auto load_values = [&](int i, Raw &r) {
      const int64_t at = static_cast<int64_t>(__builtin_amdgcn_readlane(pid, i)) * p.H;
      load_codes<kOnce>(r.vr, vbase + at * (kPage * D / 2));
      r.vb = *reinterpret_cast<const u32x4 *>(vsbase + at * kPage);
#pragma unroll
      for (int y = 0; y < kG / 2; ++y) r.vp[y] = *reinterpret_cast<const u32x4 *>(vobase + at * (kG * 32) + y * 16);
    };
    auto step = [&](int i, Raw &r) {
      const int lpage = __builtin_amdgcn_readlane(page, i);
      // the query operands are read again for every page: held over the loop they would cost 8 to 64 registers
      asm volatile("" ::: "memory");
      floatx4 s[kTiles][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float power = pow2_byte((r.kb >> (8 * t)) & 255u);
#pragma unroll
        for (int y = 0; y < kG; ++y) {
          const bf16x8 a = widen4_scaled(D == 128 ? r.kr[t][y] : r.kr[t >> 1][(t & 1) * 2 + y], power);
#pragma unroll
          for (int x = 0; x < kTiles; ++x)
#pragma unroll
            for (int piece = 0; piece < kParts; ++piece) {
              const bf16x8 q = query[(x * kOps + piece * kG + y) * 64 + lane];
              const float start = rows.start[x];
              const floatx4 c = y == 0 && piece == 0 ? floatx4{start, start, start, start} : s[x][t];
              s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q, c, 0, 0, 0);
            }
        }
      }
      if (i + kAhead * kWaves < n) load_keys(i + kAhead * kWaves, r);

      // exponents, in place: the byte's bias of 127 goes with the reference
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t vw = r.vb[t];
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
      for (int t = 0; t < 4; ++t) top |= (r.vb[t] + 0x3d3d3d3du) & ~(r.vb[t] + 0x1f1f1f1fu);
      rows.weights(s, lpage, g, inv_c, __ballot(top & 0x80808080u) != 0, [&](int t) {
        const uint32_t iw = 0xfefefefeu - r.vb[t];  // the opposite powers
        return floatx4{pow2_byte(iw & 255u), pow2_byte((iw >> 8) & 255u), pow2_byte((iw >> 16) & 255u), pow2_byte(iw >> 24)};
      }, wt);
#pragma unroll
      for (int y = 0; y < kG; ++y) {
        const halfx8 p0 = powers8(r.vp[y >> 1][(y & 1) * 2]), p1 = powers8(r.vp[y >> 1][(y & 1) * 2 + 1]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int d = y * 2 + half;
          const halfx8 a0 = widen4(r.vr[y][half * 2], p0), a1 = widen4(r.vr[y][half * 2 + 1], p1);
#pragma unroll
          for (int x = 0; x < kTiles; ++x) {
            rows.acc[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, wt[x][0], rows.acc[x][d], 0, 0, 0);
            rows.acc[x][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, wt[x][1], rows.acc[x][d], 0, 0, 0);
          }
        }
      }
      if (i + kAhead * kWaves < n) load_values(i + kAhead * kWaves, r);
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (wave + k * kWaves < n) {
        load_keys(wave + k * kWaves, ahead[k]);
        load_values(wave + k * kWaves, ahead[k]);
      }
    for (int i = wave; i < n; i += kAhead * kWaves)
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (i + k * kWaves < n) step(i + k * kWaves, ahead[k]);
  }
  float m[kTiles];
  rows.finish(m);
  rows.template join_waves<kWaves>(m, reinterpret_cast<float *>(shared), wave, col, g);
  if (wave == 0) rows.template store<Q>(p, w, 0, col, g, m);
}

// Many rows (up to 128): no pipe is full (a frame: matrix 24 %, 39 % of the waves' cycles waiting, 2130 cycles a wave's page
// where the same products and exponentials from registers take 1110); what binds is a page's chain of dependent steps, from
// barrier and operands over product, maximum and exponentials to the second product, at two or three waves a SIMD. As for the
// 8-bit cache the kWaves waves lie side by side over the rows, and a page is widened once for all of them, in LDS, two buffers
// and one barrier a page.
// Measured: a frame of 1041 queries over 522 of 2082 pages, 16 heads of 64, 142 GFLOP in 238 us with the join (600 TFLOP/s);
// 250 causal tokens of 32 heads of 128 over 20001, 163 GFLOP in 193 us (840). The frame's parts, each left out of a copy for
// its time alone: the softmax 79 us, the operands' reads from LDS 27, the pages' loads 23; what stays, widening, products and
// barriers, 110, where the products by themselves need 65. Also built, and no faster: the softmax without a maximum
// beforehand (weights checked in half, sums by a product with ones, one power for the values of a page, a third fewer vector
// instructions: 283 to 330 us, as pages are done again where a row's maximum grows, and 241 had none been), loads two pages
// ahead (238), every wave widening its pages itself without LDS (306).
template <typename Q, int D, int kTiles, int kWaves>
__global__ __launch_bounds__(kWaves * 64, D == 64 && kWaves == 4 ? 3 : 2) void cache4_attn_many_kernel(const AttnParams p) {
  constexpr int kDT = D / 16, kG = D / 32;
  constexpr int kParts = __is_same(Q, __bf16) ? 1 : 2;
  constexpr int kOps = kParts * kG;
  constexpr int kTasks = 2 * kG / kWaves;  // 1 KB of codes each: a key tile (D = 64: two), a group of features
  static_assert(kTasks * kWaves == 2 * kG, "every wave has the same share");
  struct Page {
    bf16x8 k[4 * kG][64];
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
    query_operands<Q, D, D / 4>(p, w, t, gh, rows.limit[i] > 0, g, query[i]);
  }
  rows.bounds(w.cut);
  rows.init();

  const float inv_c = 1.f / p.c;
  const int chunk = (col * 4 + g) * 16;
  u32x4 raw[kTasks];
  u32x2 scale[kTasks];
  uint32_t vb = 0;
  int turn = 0;
  for (int base = w.e0; base < w.e1; base += 64) {
    int page, pid;  // lane i has those of entry base + i
    resolve(p, w, base + lane, page, pid);
    const int n = min(w.e1 - base, 64);
    auto load = [&](int i) {
      const int64_t at = static_cast<int64_t>(__builtin_amdgcn_readlane(pid, i)) * p.H + w.h;
#pragma unroll
      for (int k = 0; k < kTasks; ++k) {
        const int task = wave + k * kWaves;
        if (task < kG) {
          raw[k] = *reinterpret_cast<const u32x4 *>(p.kc + at * (kPage * D / 2) + task * 1024 + chunk);
          const uint8_t *ks = p.ks + at * (kPage * kG) + (D == 128 ? g : g >> 1) * kPage + col * 4;
          scale[k][0] = D == 128 ? ks[task] : *reinterpret_cast<const uint16_t *>(ks + task * 2);
        } else {
          raw[k] = *reinterpret_cast<const u32x4 *>(p.vc + at * (kPage * D / 2) + (task - kG) * 1024 + chunk);
          scale[k] = *reinterpret_cast<const u32x2 *>(p.vo + at * (kG * 32) + (g * kG + task - kG) * 8);
        }
      }
      if (wave == 0) vb = p.vs[at * kPage + lane];
    };
    load(0);
    for (int i = 0; i < n; ++i) {
      Page &buf = buffer[turn];
      turn ^= 1;
#pragma unroll
      for (int k = 0; k < kTasks; ++k) {
        const int task = wave + k * kWaves;
        const u32x4 x = raw[k];
        if (task < kG) {
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            // D = 128: key tile `task`, product y; D = 64: key tile 2 task + y / 2, product y % 2
            const float power = pow2_byte(D == 128 ? scale[k][0] : (scale[k][0] >> (8 * (y >> 1))) & 255u);
            buf.k[task * 4 + y][lane] = widen4_scaled(x[y], power);
          }
        } else {
          const int d = (task - kG) * 2;
          const halfx8 p0 = powers8(scale[k][0]), p1 = powers8(scale[k][1]);
          buf.v[d * 2][lane] = widen4(x[0], p0);
          buf.v[d * 2 + 1][lane] = widen4(x[1], p1);
          buf.v[d * 2 + 2][lane] = widen4(x[2], p0);
          buf.v[d * 2 + 3][lane] = widen4(x[3], p1);
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
        for (int y = 0; y < kG; ++y) {
          const bf16x8 a = buf.k[t * kG + y][lane];
#pragma unroll
          for (int x = 0; x < kTiles; ++x)
#pragma unroll
            for (int piece = 0; piece < kParts; ++piece) {
              const float start = rows.start[x];
              const floatx4 c = y == 0 && piece == 0 ? floatx4{start, start, start, start} : s[x][t];
              s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, query[x][piece * kG + y], c, 0, 0, 0);
            }
        }
      // the softmax goes before the other waves' products: the matrix pipe works on while its instructions are issued
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
int launch_attn4(const AttnParams &p, const Shape &s, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(p.B * p.H * p.U * s.parts));
  // D = 128: 16 rows a wave, which leave registers for four waves a SIMD (32 rows: two; a causal chunk 201 and 193 us, and
  // float16 queries are two operands). D = 64: 32, three waves (16 rows read the operands twice as often: a frame 311 and 238).
  constexpr int kWaves = D == 128 ? 8 : 4;
  switch (s.kind) {
    case 0:
      if (p.list_U == 1) hipLaunchKernelGGL((cache4_attn_few_kernel<Q, D, 1, true>), grid, dim3(256), 0, st, p);
      else hipLaunchKernelGGL((cache4_attn_few_kernel<Q, D, 1, false>), grid, dim3(256), 0, st, p);
      break;
    case 1:
      if (p.list_U == 1) hipLaunchKernelGGL((cache4_attn_few_kernel<Q, D, 2, true>), grid, dim3(256), 0, st, p);
      else hipLaunchKernelGGL((cache4_attn_few_kernel<Q, D, 2, false>), grid, dim3(256), 0, st, p);
      break;
    case 2: hipLaunchKernelGGL((cache4_attn_many_kernel<Q, D, 1, 4>), grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL((cache4_attn_many_kernel<Q, D, 8 / kWaves, kWaves>), grid, dim3(kWaves * 64), 0, st, p); break;
  }
  const int rc = check_launch("vasc_cache4_attn");
  return rc ? rc : launch_join<Q, D>(p, s, st, "vasc_cache4_attn");
}

// A call's units, and in a launch of its own the last one of each head where that is better.
//
// The last unit of a frame has few rows (1041 tokens: 17 of 128), but among the others it takes a workgroup's place for as long
// as they do; by itself it is one of few rows, whose four waves share its pages. Measured, in us: a frame over 522 pages, 16
// heads of 64, 246 in one launch and 235 in two (1152 tokens, nine full units, 249), two of 1036 float16 queries over 82 pages
// 112 and 102. The second launch and its join take some 8 us however small, which the estimate has to win: a frame over 130
// pages is 97 in one launch (106 in two), 270 queries over 152 pages 45 (53).
struct Plan {
  Shape body, tail;
  int64_t body_units, tail_rows;  // units of a head in the first launch; rows of the second's one (0: none)
};

Plan attn_plan(int64_t heads, int64_t G, int64_t T, int64_t D, int64_t block_q, int64_t pages) {
  Plan plan;
  plan.body_units = cdiv(T, block_q);
  plan.tail_rows = 0;
  plan.body = attn_shape(heads * plan.body_units, block_q * G, pages, D);
  const int64_t rows = (T - (plan.body_units - 1) * block_q) * G;
  if (plan.body.kind < 2 || plan.body_units < 2 || rows > 32) return plan;
  const Shape body = attn_shape(heads * (plan.body_units - 1), block_q * G, pages, D), tail = attn_shape(heads, rows, pages, D);
  if (body.us + tail.us + 8.0 >= plan.body.us) return plan;
  return {body, tail, plan.body_units - 1, rows};
}

}  // namespace
}  // namespace vasc

extern "C" int64_t vasc_cache4_attn_workspace_size(int64_t B, int64_t Hq, int64_t H, int64_t T, int64_t D,
                                                   int64_t block_q, int64_t max_pages, int64_t width) {
  using namespace vasc;
  if (!attn_sizes(B, Hq, H, T, D, block_q, max_pages, width)) return -1;
  const Plan plan = attn_plan(B * H, Hq / H, T, D, block_q, width ? width : max_pages);
  int64_t bytes = workspace_bytes(B * H * plan.body_units, block_q * (Hq / H), D, plan.body.parts);
  if (plan.tail_rows) bytes = (bytes + 15) / 16 * 16 + workspace_bytes(B * H, plan.tail_rows, D, plan.tail.parts);
  return bytes;
}

extern "C" int vasc_cache4_attn(const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st, void *o, int64_t o_sb,
                                int64_t o_sh, int64_t o_st, int64_t B, int64_t Hq, int64_t H, int64_t T, int64_t D,
                                int32_t dtype, const uint8_t *kc, const uint8_t *vc, const uint8_t *ks,
                                const uint8_t *vs, const uint8_t *vo, int64_t pages, const int32_t *page_table,
                                int64_t table_stride, int64_t max_pages, const int32_t *lengths, const int32_t *q_count,
                                int64_t block_q, const int32_t *index, int64_t width, const int32_t *count,
                                int32_t causal, float scale, void *workspace, int64_t workspace_bytes_given, void *stream) {
  using namespace vasc;
  VASC_REQUIRE(vo && (reinterpret_cast<uintptr_t>(vo) & 15) == 0, "vo must be given and 16-byte aligned");
  AttnParams p = {};
  int rc = attn_params(q, q_sb, q_sh, q_st, o, o_sb, o_sh, o_st, B, Hq, H, T, D, dtype, kc, vc, ks, vs, pages, page_table,
                       table_stride, max_pages, lengths, q_count, block_q, index, width, count, causal, scale, p);
  if (rc) return rc;
  p.vo = vo;
  const Plan plan = attn_plan(B * H, p.G, T, D, block_q, width ? width : max_pages);
  p.U = static_cast<int>(plan.body_units);
  int64_t used = 0;
  if ((rc = take_workspace(p, plan.body, D, workspace, workspace_bytes_given, used))) return rc;
  AttnParams last = p;
  if (plan.tail_rows) {
    last.u0 = p.U;
    last.U = 1;
    last.rows = static_cast<int>(plan.tail_rows);
    if ((rc = take_workspace(last, plan.tail, D, workspace, workspace_bytes_given, used))) return rc;
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const auto launch = [&](const AttnParams &a, const Shape &s) {
    if (D == 64) return dtype == 0 ? launch_attn4<__bf16, 64>(a, s, st) : launch_attn4<_Float16, 64>(a, s, st);
    return dtype == 0 ? launch_attn4<__bf16, 128>(a, s, st) : launch_attn4<_Float16, 128>(a, s, st);
  };
  if ((rc = launch(p, plan.body)) || !plan.tail_rows) return rc;
  return launch(last, plan.tail);
}
