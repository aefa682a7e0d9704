// The 8-bit block cache: writing tokens into it, reading them back, and the
// choice of the pages that a group of queries attends to.
//
// Write and read are bound by HBM (2 or 4 bytes of input and 1 + 1/D of cache
// per value). One workgroup owns one (page, head) of a call: nothing else of
// the call touches that page, so partly covered words are merged with plain
// loads and stores, and the page's key mean is recomputed from its codes, a
// function of what the page holds whatever calls brought it there.
// Measured (bf16, 16 heads of 64): 32 frames of 1041 tokens written in 47 us
// (4.4 TB/s; a large copy reaches 4.75), read back in 32 us (6.4 TB/s, partly
// from the cache behind HBM); one token of 64 sequences, 8 heads of 128, in
// 7.3 us: the latency of table, codes, barrier and merge.
#include "stream.h"

namespace vasc {
namespace {

struct CacheArgs {
  uint8_t *kc, *vc, *ks, *vs;
  uint16_t *mean;
  int64_t pages;
  const int32_t *table;
  int64_t table_stride, max_pages;
};

struct RowArgs {
  const void *k, *v;  // read: the outputs
  int64_t ksb, ksh, kst, vsb, vsh, vst;
  const int32_t *start, *count;
  int64_t B, H, T;
  int span;  // pages that T tokens can touch
};

// Eight consecutive elements as floats.
template <typename T>
__device__ __forceinline__ void load8(const T *src, float (&x)[8]) {
  struct alignas(sizeof(T) == 4 ? 16 : 8 * sizeof(T)) Eight { T v[8]; };
  const Eight e = *reinterpret_cast<const Eight *>(src);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(e.v[i]);
}

template <typename T>
__device__ __forceinline__ void store8(T *dst, const float (&x)[8]) {
  struct alignas(sizeof(T) == 4 ? 16 : 8 * sizeof(T)) Eight { T v[8]; };
  Eight e;
#pragma unroll
  for (int i = 0; i < 8; ++i) e.v[i] = from_f32<T>(x[i]);
  *reinterpret_cast<Eight *>(dst) = e;
}

// Max over the D/8 neighbouring lanes that hold a row.
template <int D>
__device__ __forceinline__ float row_max(float v) {
  v = group8_max(v);
  return D == 128 ? fmaxf(v, xor_lane(v, 8)) : v;
}

// Exponent byte of a row whose largest magnitude is `top`.
__device__ __forceinline__ int row_exponent(float top) { return power_of(top, -60, 60) + 127; }

__device__ __forceinline__ void quantise8(const float (&x)[8], int byte, uint32_t (&w)[2]) {
  const float inv = __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = fminf(fmaxf(x[i] * inv, -448.f), 448.f);
  w[0] = pack_e4m3(y[0], y[1], y[2], y[3]);
  w[1] = pack_e4m3(y[4], y[5], y[6], y[7]);
}

// Row stride of the value tile in LDS: consecutive groups of four rows start four banks apart.
template <int D>
constexpr int tile_stride() { return D + 4; }

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

template <typename T, int D>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheArgs c, const RowArgs r) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes, kS = tile_stride<D>();
  constexpr int kGroups = 256 / (D / 4);  // row groups of the mean, four columns a thread
  __shared__ __align__(16) uint8_t kt[kPage * D];
  __shared__ __align__(16) uint8_t vt[kPage * kS];
  __shared__ uint8_t ke[kPage];
  __shared__ double part[kGroups][D];
  const int tid = threadIdx.x;
  PageWork w;
  const int64_t b = blockIdx.x / (static_cast<uint32_t>(r.span) * static_cast<uint32_t>(r.H));
  if (!page_work(c, r, new_tokens(r, b), w) || w.pid < 0) return;
  const int64_t ph = w.pid * r.H + w.h;
  const int col = (tid % kLanes) * 8;
  const T *kin = static_cast<const T *>(r.k) + w.b * r.ksb + w.h * r.ksh;
  const T *vin = static_cast<const T *>(r.v) + w.b * r.vsb + w.h * r.vsh;
#pragma unroll
  for (int pass = 0; pass < kPage / kRows; ++pass) {
    const int row = pass * kRows + tid / kLanes;
    if (row < w.lo) {  // held before: its part of the mean
      *reinterpret_cast<u32x2 *>(kt + row * D + col) =
          *reinterpret_cast<const u32x2 *>(c.kc + (ph * kPage + row) * D + col);
      if (col == 0) ke[row] = c.ks[ph * kPage + key_place(row)];
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
      kmax = row_max<D>(kmax);
      vmax = row_max<D>(vmax);
      bad = row_max<D>(bad);
      int kb = row_exponent(kmax), vb = row_exponent(vmax);
      uint32_t kw[2] = {0, 0}, vw[2] = {0, 0};
      if (bad == 0.f) {
        quantise8(x, kb, kw);
        quantise8(y, vb, vw);
      } else {
        kb = 255;
        vb = 127;
      }
      const u32x2 kk = {kw[0], kw[1]};
      *reinterpret_cast<u32x2 *>(kt + row * D + col) = kk;
      *reinterpret_cast<u32x2 *>(c.kc + (ph * kPage + row) * D + col) = kk;
      *reinterpret_cast<uint32_t *>(vt + row * kS + col) = vw[0];
      *reinterpret_cast<uint32_t *>(vt + row * kS + col + 4) = vw[1];
      if (col == 0) {
        ke[row] = static_cast<uint8_t>(kb);
        c.ks[ph * kPage + key_place(row)] = static_cast<uint8_t>(kb);
        c.vs[ph * kPage + page_place(row)] = static_cast<uint8_t>(vb);
      }
    }
  }
  __syncthreads();
  // values, transposed: 16 bytes of feature d hold the tokens grp*32 + tile*16 + g*4 + i of lane group g
  for (int task = tid; task < D * 4; task += 256) {
    const int d = task >> 2, g = task & 3;
    uint8_t *dst = c.vc + (ph * D + d) * kPage + g * 16;
    uint32_t word[4];
    int full = 0, some = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int key = q * 16 + g * 4;
      word[q] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (key + i >= w.lo && key + i < w.hi) word[q] |= static_cast<uint32_t>(vt[(key + i) * kS + d]) << (8 * i);
      if (key >= w.lo && key + 4 <= w.hi) full |= 1 << q;
      if (key + 4 > w.lo && key < w.hi) some |= 1 << q;
    }
    if (full == 15) {
      *reinterpret_cast<u32x4 *>(dst) = u32x4{word[0], word[1], word[2], word[3]};
      continue;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (!(some >> q & 1)) continue;
      uint32_t *at = reinterpret_cast<uint32_t *>(dst) + q;
      if (!(full >> q & 1)) {
        const uint32_t old = *at;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = q * 16 + g * 4 + i;
          if (key < w.lo || key >= w.hi) word[q] |= old & (0xffu << (8 * i));
        }
      }
      *at = word[q];
    }
  }
  // The page's key mean, summed in float64 in an order that the slots fix (a group of threads takes every kGroups-th, the
  // groups are added in turn), whatever calls brought the rows: the same bytes in any portions. The order would not show by
  // itself only where the page's exponents lie within some 40 of one another, as then all sums are exact.
  {
    const int dcol = (tid % (D / 4)) * 4, grp = tid / (D / 4);
    double s[4] = {0, 0, 0, 0};
    for (int row = grp; row < w.hi; row += kGroups) {
      float f[4];
      unpack_e4m3(*reinterpret_cast<const uint32_t *>(kt + row * D + dcol), f);
      const float e = pow2_byte(ke[row]);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += static_cast<double>(f[i] * e);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) part[grp][dcol + i] = s[i];
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
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheArgs c, const RowArgs r) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes, kS = tile_stride<D>();
  __shared__ __align__(16) uint8_t vt[kPage * kS];
  const int tid = threadIdx.x;
  PageWork w;
  const int64_t b = blockIdx.x / (static_cast<uint32_t>(r.span) * static_cast<uint32_t>(r.H));
  const int64_t n = new_tokens(r, b);
  bool live = r.start[b] >= 0;
  if (!page_work(c, r, r.T, w)) {
    if (live) return;
    // a negative start reads nothing: its rows are zero, 64 to a workgroup
    w.s = 0;
    w.j = blockIdx.x % r.span;
    w.h = (blockIdx.x / r.span) % r.H;
    w.b = b;
    w.lo = 0;
    const int64_t hi = r.T - w.j * kPage;
    w.hi = static_cast<int>(hi < kPage ? hi : kPage);
    w.pid = -1;
    if (w.hi <= 0) return;
  }
  live = live && w.pid >= 0;
  const int64_t ph = w.pid * r.H + w.h;
  const int col = (tid % kLanes) * 8;
  if (live) {
    for (int task = tid; task < D * 4; task += 256) {
      const int d = task >> 2, g = task & 3;
      const u32x4 x = *reinterpret_cast<const u32x4 *>(c.vc + (ph * D + d) * kPage + g * 16);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t word = x[q];
#pragma unroll
        for (int i = 0; i < 4; ++i) vt[(q * 16 + g * 4 + i) * kS + d] = static_cast<uint8_t>(word >> (8 * i));
      }
    }
  }
  __syncthreads();
  T *ko = const_cast<T *>(static_cast<const T *>(r.k)) + (w.b * r.H + w.h) * r.T * D;
  T *vo = const_cast<T *>(static_cast<const T *>(r.v)) + (w.b * r.H + w.h) * r.T * D;
#pragma unroll
  for (int pass = 0; pass < kPage / kRows; ++pass) {
    const int row = pass * kRows + tid / kLanes;
    if (row < w.lo || row >= w.hi) continue;
    const int64_t t = w.j * kPage + row - w.s;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (live && t < n) {
      const u32x2 kw = *reinterpret_cast<const u32x2 *>(c.kc + (ph * kPage + row) * D + col);
      const uint32_t kb = c.ks[ph * kPage + key_place(row)];
      const float ke = pow2_byte(kb);
      const float ve = kb == 255 ? ke : pow2_byte(c.vs[ph * kPage + page_place(row)]);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float a[4], d[4];
        const uint32_t kword = kw[q];
        unpack_e4m3(kword, a);
        unpack_e4m3(*reinterpret_cast<const uint32_t *>(vt + row * kS + col + q * 4), d);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[q * 4 + i] = a[i] * ke;
          y[q * 4 + i] = d[i] * ve;
        }
      }
    }
    store8(ko + t * D + col, x);
    store8(vo + t * D + col, y);
  }
}

// ------------------------------------------------------------------ choice
struct SelectParams {
  const void *q;
  int64_t qsb, qsh, qst;
  int64_t B, T;
  int H, G, U;
  const uint16_t *mean;
  int64_t pages;
  const int32_t *table;
  int64_t table_stride, max_pages;
  const int32_t *lengths, *n_q;
  int block_q, causal, chunks, rounds;
  int64_t sink, recent, keep, width;
  float *score;
  int32_t *index, *count;
};

struct Unit {
  int64_t b, h, u;
  int64_t t0, t1;
  UnitView view;
};

__device__ __forceinline__ Unit unit_of(const SelectParams &p, int row) {
  Unit n;
  const int bh = row / p.U;
  n.u = row - bh * p.U;
  n.b = bh / p.H;
  n.h = bh - static_cast<int>(n.b) * p.H;
  int64_t nq = p.n_q ? p.n_q[n.b] : p.T;
  nq = nq < 0 ? 0 : (nq < p.T ? nq : p.T);
  n.t0 = n.u * p.block_q;
  n.t1 = n.t0 + p.block_q < nq ? n.t0 + p.block_q : nq;
  n.view = unit_view(p.lengths[n.b], nq, n.t0, n.t1, p.max_pages, p.causal);
  return n;
}

// Scores of a unit against its pages: the bf16 mean of its query rows times each page's bf16 key mean, products and sums
// in float64. Those products are exact and their sums all but always, so the order of a sum does not show in the score.
//
// Bound: the float64 pipe (a conversion, a product and a seventh of an exchange for each feature and page) and the latency
// of what depends on what (lengths, page table and queries, means). So all that can is in flight together: a workgroup
// asks for its pages' places before it has seen the lengths and for their means before it sums the queries; the sums of
// kScoreBatch pages cross the lanes together, each step leaving a lane half the pages; and a workgroup takes as many
// rounds of pages as leave the chip some four workgroups a CU.
// Measured: 16 x 131072 tokens, 8 heads of 128, in 14.0 us (3.1 TB/s); nine
// units of a frame against 2082 pages, 16 heads of 64, in 12.5 us.
constexpr int kScoreBatch = 8;

// Sums v[0..8) over the lanes that differ in the bits [lo, hi) of the lane number; a lane is left with the sum of element
// (its low three of those bits) in v[0].
__device__ __forceinline__ void scatter_sum(double (&v)[8], int lo, int hi) {
  int width = 8;
#pragma unroll
  for (int o = lo; o < hi; o <<= 1) {
    if (width > 1) {
      width >>= 1;
      const bool up = __lane_id() & o;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < width) {
          const double keep = up ? v[2 * i + 1] : v[2 * i], send = up ? v[2 * i] : v[2 * i + 1];
          v[i] = keep + xor_lane(send, o);
        }
    } else {
      v[0] += xor_lane(v[0], o);
    }
  }
}

template <typename T, int D>
__global__ __launch_bounds__(256) void cache_score_kernel(const SelectParams p) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes;  // lanes of a row or page; rows or pages of a step
  constexpr int kRound = kScoreBatch * kRows;
  const int kPages = kRound * p.rounds;
  __shared__ double part[4][D];
  __shared__ float qm[D];
  const int tid = threadIdx.x, lane = tid % kLanes, grp = tid / kLanes;
  const int64_t row = static_cast<int>(blockIdx.x) / p.chunks;
  const int first = static_cast<int>(blockIdx.x) % p.chunks * kPages;
  const int end = static_cast<int>(first + kPages < p.max_pages ? first + kPages : p.max_pages);
  const int64_t b = row / (static_cast<int64_t>(p.U) * p.H);
  int pid[kScoreBatch];
#pragma unroll
  for (int i = 0; i < kScoreBatch; ++i) {
    const int j = first + grp + i * kRows;
    pid[i] = j < end ? p.table[b * p.table_stride + j] : -1;
  }
  const Unit n = unit_of(p, static_cast<int>(row));
  const int seen = static_cast<int>(n.view.seen);
  float *out = p.score + row * p.max_pages;
  if (first >= seen) {
    for (int j = first + tid; j < end; j += 256) out[j] = -__builtin_inff();
    return;
  }
  const int rows = static_cast<int>(n.t1 - n.t0) * p.G;
  // up to 128 rows: at most kMost a lane group
  constexpr int kMost = 128 / kRows;
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  words x[kMost];
  const T *q = static_cast<const T *>(p.q) + n.b * p.qsb + n.h * p.G * p.qsh + n.t0 * p.qst + lane * 8;
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int r = grp + i * kRows, tl = r / p.G;
    x[i] = words{0, 0, 0, 0};
    if (r < rows) x[i] = *reinterpret_cast<const words *>(q + tl * p.qst + (r - tl * p.G) * p.qsh);
  }
  u32x4 m[kScoreBatch];
#pragma unroll
  for (int i = 0; i < kScoreBatch; ++i) {
    if (first + grp + i * kRows >= seen || pid[i] >= p.pages) pid[i] = -1;
    m[i] = u32x4{0, 0, 0, 0};
    if (pid[i] >= 0)
      m[i] = *reinterpret_cast<const u32x4 *>(p.mean + (static_cast<int64_t>(pid[i]) * p.H + n.h) * D + lane * 8);
  }
  {
    double s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
      if (i * kRows >= rows) break;
      struct alignas(16) Eight { T v[8]; };
      const Eight v = __builtin_bit_cast(Eight, x[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += static_cast<double>(to_f32(v.v[e]));
    }
    // lanes of different rows: D = 64 leaves a feature a lane, D = 128 two
    scatter_sum(s, kLanes, 64);
    const int at = (tid & 63) / kLanes;
    if (D == 64) {
      part[tid >> 6][lane * 8 + at] = s[0];
    } else {
      part[tid >> 6][lane * 8 + at] = s[0];
      part[tid >> 6][lane * 8 + at + 4] = s[1];
    }
  }
  __syncthreads();
  if (tid < D)
    qm[tid] = round_bf16(static_cast<float>((part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]) / rows));
  __syncthreads();
  double qd[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) qd[i] = static_cast<double>(qm[lane * 8 + i]);
  for (int j0 = first;;) {
    double sum[kScoreBatch];
#pragma unroll
    for (int i = 0; i < kScoreBatch; ++i) {
      sum[i] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t word = m[i][e >> 1];
        sum[i] = fma(qd[e], static_cast<double>(__uint_as_float(e & 1 ? word & 0xffff0000u : word << 16)), sum[i]);
      }
    }
    scatter_sum(sum, 1, kLanes);
    // lane i of the group (of its first eight) has page i of the batch
    uint32_t gone = 0;
#pragma unroll
    for (int i = 0; i < kScoreBatch; ++i) gone |= (pid[i] < 0 ? 1u : 0u) << i;
    const int i = lane & 7, j = j0 + grp + i * kRows;
    float f = static_cast<float>(sum[0]);
    if ((gone >> i & 1) || f != f) f = -__builtin_inff();
    if (lane < 8 && j < end) out[j] = f;
    j0 += kRound;
    if (j0 >= end) break;
    if (j0 >= seen) {
      for (int k = j0 + tid; k < end; k += 256) out[k] = -__builtin_inff();
      break;
    }
#pragma unroll
    for (int k = 0; k < kScoreBatch; ++k) {
      const int page = j0 + grp + k * kRows;
      pid[k] = page < seen && page < end ? p.table[b * p.table_stride + page] : -1;
    }
#pragma unroll
    for (int k = 0; k < kScoreBatch; ++k) {
      if (pid[k] >= p.pages) pid[k] = -1;
      m[k] = u32x4{0, 0, 0, 0};
      if (pid[k] >= 0)
        m[k] = *reinterpret_cast<const u32x4 *>(p.mean + (static_cast<int64_t>(pid[k]) * p.H + n.h) * D + lane * 8);
    }
  }
}

// Scores as integers in the same order (-0 as 0); anything is above 0, the mark of a page that is not free to choose.
__device__ __forceinline__ uint32_t score_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The list of one unit. Wave w holds the scores of pages [w * 64 E, (w + 1) * 64 E) in registers, page base + i * 64 + lane
// in element i, and looks for the last chosen of them: (cut, cut_page), such that a page is chosen with a higher score, or
// the same one and no higher a number.
//
// One wave finds the keep-th largest bit by bit from the top, a count of all elements a bit; a count that meets `keep`
// exactly ends it. More waves would pay a barrier a bit (9.9 us for 128 lists of 2048 pages): they sort into 2048 bins by
// the next 11 bits instead, until the bin that holds the cut has at most kRanked members (scores of one sign and size spread
// over some dozens of bins, so most lists need one turn), which are then ranked among themselves.
// Past 8192 pages a thread holds 32 elements: 8 lists (with their scores, 8 heads of 128) take 17.5 us for 8192 pages, 38
// for 8193, 51 for 32768.
// Measured: 128 lists of 2048 pages or 144 of 2082 in 8.3 us: 4.5 until the scores are there, 1.4 for the bins, 1.5 for the
// ranks, the rest for the list; latency throughout.
constexpr int kBins = 2048, kRanked = 128;

template <int kWaves, int E>
__global__ __launch_bounds__(kWaves * 64) void cache_list_kernel(const SelectParams p) {
  constexpr int kThreads = kWaves * 64;
  constexpr int kOwn = kBins / (kWaves > 1 ? kThreads : kBins);  // bins of a thread
  __shared__ uint32_t bins[kWaves > 1 ? kBins : 1];
  __shared__ __align__(16) uint64_t ranked[kWaves > 1 ? kRanked : 1];
  static_assert(kWaves == 1 || kRanked <= kThreads, "a thread a member");
  __shared__ int wave_total[kWaves], wave_equal[kWaves];
  __shared__ int found[4];  // the cut's bin, what is left to choose in it, its members; the next free place of `ranked`
  __shared__ uint64_t last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const float *score = p.score + row * p.max_pages;
  const int base = wave * 64 * E;
  float value[E];  // asked for before the lengths are known: all of max_pages are written
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int j = base + i * 64 + lane;
    value[i] = j < p.max_pages ? score[j] : 0.f;
  }
  const Unit n = unit_of(p, blockIdx.x);
  const int seen = static_cast<int>(n.view.seen), sink = static_cast<int>(p.sink);
  const int tail = static_cast<int>(n.view.own - (p.recent - 1));  // pages from here on are listed
  uint32_t key[E];  // 0: not free to choose
  uint32_t forced = 0;
  static_assert(E <= 32, "one bit an element");
  int free_pages = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int j = base + i * 64 + lane;
    key[i] = 0;
    if (j < seen) {
      if (j < sink || j >= tail)
        forced |= 1u << i;
      else
        key[i] = score_key(value[i]);
    }
  }
  {
    const int end = tail < seen ? tail : seen;  // the free pages are [sink, end)
    free_pages = end > sink ? end - sink : 0;
  }
  uint32_t cut = 1;              // chosen: above the cut, or
  int cut_page = 1 << 30;        // on it and no higher a page, or
  int ties = 0;                  // on it and (ties > 0) among the first of those
  if (p.keep < free_pages) {
    int want = static_cast<int>(p.keep);
    if (want == 0) {
      cut = 0xffffffffu;  // no score has this key (it would be a NaN)
    } else if (kWaves == 1) {
      uint32_t t = 0;
      int at = 0;
      bool exact = false;
      for (int bit = 31; bit >= 0 && !exact; --bit) {
        const uint32_t cand = t | (1u << bit);
        int c = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) c += __popcll(__ballot(key[i] >= cand));
        if (c >= want) {
          t = cand;
          at = c;
        }
        exact = c == want;
      }
      cut = t;
      if (!exact && at > want) {
        int above = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) above += __popcll(__ballot(key[i] > cut));
        ties = want - above;
      }
    } else {
      uint32_t prefix = 0, mask = 0;  // the cut's bits found so far
      for (int shift = 21; ; shift = shift == 21 ? 10 : 0) {
        const uint32_t digits = shift == 0 ? 1023u : 2047u;
        for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (key[i] != 0 && (key[i] & mask) == prefix) atomicAdd(&bins[(key[i] >> shift) & digits], 1u);
        __syncthreads();
        int mine[kOwn], own = 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          mine[i] = bins[tid * kOwn + i];
          own += mine[i];
        }
        int above = own;  // this thread's bins and those over them, in the wave and then in all
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int x = __shfl_down(above, o);
          if (lane + o < 64) above += x;
        }
        if (lane == 0) wave_total[wave] = above;
        __syncthreads();
#pragma unroll
        for (int w = 1; w < kWaves; ++w) above += w > wave ? wave_total[w] : 0;
        above -= own;
        if (above < want && above + own >= want) {  // one thread
#pragma unroll
          for (int i = kOwn - 1; i >= 0; --i) {
            const int c = mine[i];
            if (above < want && above + c >= want) {
              found[0] = tid * kOwn + i;
              found[1] = want - above;
              found[2] = c;
              found[3] = 0;
            }
            above += c;
          }
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(found[0]) << shift;
        mask |= digits << shift;
        want = found[1];
        const int members = found[2];
        if (members == want) {  // the whole bin
          cut = prefix;
          break;
        }
        if (members <= kRanked) {
#pragma unroll
          for (int i = 0; i < E; ++i)
            if (key[i] != 0 && (key[i] & mask) == prefix)
              ranked[atomicAdd(&found[3], 1)] =
                  static_cast<uint64_t>(key[i]) << 32 | static_cast<uint32_t>(~(base + i * 64 + lane));
          const int padded = (members + 7) & ~7;
          if (tid >= members && tid < padded) ranked[tid] = 0;
          __syncthreads();
          // kThreads / kRanked neighbouring threads count for a member
          constexpr int kShare = kWaves > 1 ? kThreads / kRanked : 1;
          const int member = tid / kShare;
          if (member < members) {
            const uint64_t own_key = ranked[member];
            int over = 0;
            for (int i = tid % kShare * 8; i < padded; i += 8 * kShare) {
#pragma unroll
              for (int e = 0; e < 8; ++e) over += ranked[i + e] > own_key;
            }
#pragma unroll
            for (int o = 1; o < kShare; o <<= 1) over += xor_lane(over, o);
            if (over == want - 1) last = own_key;
          }
          __syncthreads();
          cut = static_cast<uint32_t>(last >> 32);
          cut_page = static_cast<int>(~static_cast<uint32_t>(last));
          break;
        }
        if (shift == 0) {  // equal scores, more of them than are ranked
          cut = prefix;
          ties = want;
          break;
        }
        __syncthreads();  // `found` and the bins are written again
      }
    }
  }
  // places: lists ascend, so every wave needs what the waves before it chose (and how many equal the cut)
  uint64_t pick[E];
  int eq_before = 0, chosen = 0;
  if (ties > 0) {
    int eq = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) eq += __popcll(__ballot(key[i] == cut));
    if (lane == 0) wave_equal[wave] = eq;
    __syncthreads();
    for (int w = 0; w < wave; ++w) eq_before += wave_equal[w];
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    bool take = ((forced >> i) & 1) || key[i] > cut;
    if (ties > 0) {
      const uint64_t eq = __ballot(key[i] == cut);
      take = take || (key[i] == cut && eq_before + lanes_below(eq) < ties);
      eq_before += __popcll(eq);
    } else {
      // with a whole bin the cut is the least key that the bin can hold
      take = take || (key[i] == cut && base + i * 64 + lane <= cut_page);
    }
    pick[i] = __ballot(take);
    chosen += __popcll(pick[i]);
  }
  __syncthreads();  // wave_total is read above
  if (lane == 0) wave_total[wave] = chosen;
  __syncthreads();
  int at = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int c = wave_total[w];
    at += w < wave ? c : 0;
    all += c;
  }
  const int width = static_cast<int>(p.width);
  int32_t *list = p.index + row * p.width;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int place = at + lanes_below(pick[i]);
    if ((pick[i] >> lane & 1) && place < width) list[place] = base + i * 64 + lane;
    at += __popcll(pick[i]);
  }
  for (int i = all + tid; i < width; i += kThreads) list[i] = -1;
  if (tid == 0) p.count[row] = all < width ? all : width;
}

template <typename T, int D>
void launch_write(const CacheArgs &c, const RowArgs &r, hipStream_t s) {
  hipLaunchKernelGGL((cache_write_kernel<T, D>), dim3(static_cast<unsigned>(r.B * r.H * r.span)), dim3(256), 0, s, c, r);
}
template <typename T, int D>
void launch_read(const CacheArgs &c, const RowArgs &r, hipStream_t s) {
  hipLaunchKernelGGL((cache_read_kernel<T, D>), dim3(static_cast<unsigned>(r.B * r.H * r.span)), dim3(256), 0, s, c, r);
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

}  // namespace
}  // namespace vasc

extern "C" int vasc_cache_write(const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st, const void *v, int64_t v_sb,
                                int64_t v_sh, int64_t v_st, int64_t B, int64_t H, int64_t T, int64_t D, int32_t dtype,
                                const int32_t *page_table, int64_t table_stride, int64_t max_pages, const int32_t *start,
                                const int32_t *count, uint8_t *kc, uint8_t *vc, uint8_t *ks, uint8_t *vs,
                                uint16_t *mean, int64_t pages, void *stream) {
  using namespace vasc;
  int rc;
  if ((rc = check_cache(kc, vc, ks, vs, pages, page_table, table_stride, max_pages, D))) return rc;
  if ((rc = check_rows("k", k, k_sb, k_sh, k_st))) return rc;
  if ((rc = check_rows("v", v, v_sb, v_sh, v_st))) return rc;
  VASC_REQUIRE(mean && start, "mean and start are required");
  VASC_REQUIRE(B > 0 && H > 0 && T > 0, "empty tensor");
  VASC_SUPPORTED(dtype >= 0 && dtype <= 2, "dtype %d not built", dtype);
  RowArgs r = {k, v, k_sb, k_sh, k_st, v_sb, v_sh, v_st, start, count, B, H, T, 0};
  VASC_REQUIRE(T < (int64_t(1) << 30), "too many tokens");
  r.span = static_cast<int>((T + 2 * kPage - 2) / kPage);
  VASC_REQUIRE(H < (1 << 16) && B < (int64_t(1) << 24) && B * H * r.span < (int64_t(1) << 31), "too many tokens");
  const CacheArgs c = {kc, vc, ks, vs, mean, pages, page_table, table_stride, max_pages};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (D == 64)
    (dtype == 0 ? launch_write<__bf16, 64> : dtype == 1 ? launch_write<_Float16, 64> : launch_write<float, 64>)(c, r, s);
  else
    (dtype == 0 ? launch_write<__bf16, 128> : dtype == 1 ? launch_write<_Float16, 128> : launch_write<float, 128>)(c, r, s);
  return check_launch("vasc_cache_write");
}

extern "C" int vasc_cache_read(const uint8_t *kc, const uint8_t *vc, const uint8_t *ks, const uint8_t *vs,
                               int64_t pages, const int32_t *page_table, int64_t table_stride, int64_t max_pages,
                               const int32_t *start, const int32_t *count, int64_t B, int64_t H, int64_t T, int64_t D,
                               int32_t dtype, void *ko, void *vo, void *stream) {
  using namespace vasc;
  int rc;
  if ((rc = check_cache(kc, vc, ks, vs, pages, page_table, table_stride, max_pages, D))) return rc;
  if ((rc = check_rows("ko", ko, 0, 0, D))) return rc;
  if ((rc = check_rows("vo", vo, 0, 0, D))) return rc;
  VASC_REQUIRE(start, "start is required");
  VASC_REQUIRE(B > 0 && H > 0 && T > 0, "empty tensor");
  VASC_SUPPORTED(dtype >= 0 && dtype <= 2, "dtype %d not built", dtype);
  VASC_REQUIRE(T < (int64_t(1) << 30), "too many tokens");
  RowArgs r = {ko, vo, 0, 0, 0, 0, 0, 0, start, count, B, H, T, 0};
  r.span = static_cast<int>((T + 2 * kPage - 2) / kPage);
  VASC_REQUIRE(H < (1 << 16) && B < (int64_t(1) << 24) && B * H * r.span < (int64_t(1) << 31), "too many tokens");
  const CacheArgs c = {const_cast<uint8_t *>(kc), const_cast<uint8_t *>(vc), const_cast<uint8_t *>(ks),
                       const_cast<uint8_t *>(vs), nullptr, pages, page_table, table_stride, max_pages};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (D == 64)
    (dtype == 0 ? launch_read<__bf16, 64> : dtype == 1 ? launch_read<_Float16, 64> : launch_read<float, 64>)(c, r, s);
  else
    (dtype == 0 ? launch_read<__bf16, 128> : dtype == 1 ? launch_read<_Float16, 128> : launch_read<float, 128>)(c, r, s);
  return check_launch("vasc_cache_read");
}

extern "C" int vasc_cache_select(const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st, int64_t B, int64_t Hq,
                                 int64_t H, int64_t T, int64_t D, int32_t dtype, const uint16_t *mean, int64_t pages,
                                 const int32_t *page_table, int64_t table_stride, int64_t max_pages,
                                 const int32_t *lengths, const int32_t *q_count, int64_t block_q, int64_t sink,
                                 int64_t recent, int64_t keep, int32_t causal, float *score, int32_t *index,
                                 int64_t width, int32_t *count, void *stream) {
  using namespace vasc;
  int rc;
  if ((rc = check_cache(mean, mean, mean, mean, pages, page_table, table_stride, max_pages, D))) return rc;
  if ((rc = check_rows("q", q, q_sb, q_sh, q_st))) return rc;
  VASC_REQUIRE(lengths && score && index && count, "lengths, score, index and count are required");
  VASC_REQUIRE(B > 0 && H > 0 && T > 0, "empty tensor");
  VASC_REQUIRE(Hq > 0 && Hq % H == 0, "Hq %lld is no multiple of H %lld", (long long)Hq, (long long)H);
  VASC_SUPPORTED(dtype == 0 || dtype == 1, "dtype %d not built", dtype);
  SelectParams p = {};
  p.G = static_cast<int>(Hq / H);
  VASC_REQUIRE(block_q >= 1 && block_q <= 128 && Hq / H <= 128 && block_q * (Hq / H) <= 128, "block_q %lld with %lld query heads a key head: 1 to 128 rows",
               (long long)block_q, (long long)(Hq / H));
  VASC_REQUIRE(sink >= 0 && recent >= 1 && keep >= 0, "sink and keep must not be negative, recent at least 1");
  VASC_REQUIRE(sink < (1 << 24) && recent < (1 << 24) && keep < (1 << 24), "sink, recent or keep too large");
  int64_t want = sink + keep + recent + (causal ? (block_q + kPage - 2) / kPage : 0);
  if (want > max_pages) want = max_pages;
  VASC_REQUIRE(width == want, "width %lld, expected %lld", (long long)width, (long long)want);
  VASC_SUPPORTED(max_pages <= 16 * 64 * 32, "max_pages %lld not built (at most %d)", (long long)max_pages, 16 * 64 * 32);
  p.q = q; p.qsb = q_sb; p.qsh = q_sh; p.qst = q_st;
  VASC_REQUIRE(B < (1 << 24) && H < (1 << 16) && T < (int64_t(1) << 30), "too many units");
  p.B = B; p.H = static_cast<int>(H); p.T = T; p.U = static_cast<int>(cdiv(T, block_q));
  p.mean = mean; p.pages = pages;
  p.table = page_table; p.table_stride = table_stride; p.max_pages = max_pages;
  p.lengths = lengths; p.n_q = q_count;
  p.block_q = static_cast<int>(block_q);
  p.causal = causal;
  const int64_t round = kScoreBatch * (256 / (D / 8)), all = B * H * p.U * cdiv(max_pages, round);
  p.rounds = all <= 1024 ? 1 : all >= 8192 ? 8 : static_cast<int>(cdiv(all, 1024));
  p.chunks = static_cast<int>(cdiv(max_pages, round * p.rounds));
  p.sink = sink; p.recent = recent; p.keep = keep; p.width = width;
  p.score = score; p.index = index; p.count = count;
  VASC_REQUIRE(B * H < (int64_t(1) << 31) / p.U && B * H * p.U < (int64_t(1) << 31) / p.chunks, "too many units");
  const int64_t rows = B * H * p.U;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(rows * p.chunks)), list(static_cast<unsigned>(rows));
  if (D == 64) {
    if (dtype == 0) hipLaunchKernelGGL((cache_score_kernel<__bf16, 64>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((cache_score_kernel<_Float16, 64>), grid, dim3(256), 0, s, p);
  } else {
    if (dtype == 0) hipLaunchKernelGGL((cache_score_kernel<__bf16, 128>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((cache_score_kernel<_Float16, 128>), grid, dim3(256), 0, s, p);
  }
  if ((rc = check_launch("vasc_cache_select"))) return rc;
  if (max_pages <= 256) hipLaunchKernelGGL((cache_list_kernel<1, 4>), list, dim3(64), 0, s, p);
  else if (max_pages <= 2048) hipLaunchKernelGGL((cache_list_kernel<4, 8>), list, dim3(256), 0, s, p);
  else if (max_pages <= 4096) hipLaunchKernelGGL((cache_list_kernel<8, 8>), list, dim3(512), 0, s, p);
  else if (max_pages <= 8192) hipLaunchKernelGGL((cache_list_kernel<16, 8>), list, dim3(1024), 0, s, p);
  else hipLaunchKernelGGL((cache_list_kernel<16, 32>), list, dim3(1024), 0, s, p);
  return check_launch("vasc_cache_select");
}
