// The 8-bit block cache: writing tokens into it, reading them back, and the
// choice of the pages that a group of queries attends to.
//
// Write and read are bound by HBM (2 or 4 bytes of input and 1 + 1/D of cache
// per value). One workgroup owns one (page, head) of a call: nothing else of
// the call touches that page, so partly covered words are merged with plain
// loads and stores, and the page's key mean is recomputed from its codes, a
// function of what the page holds whatever calls brought it there.
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
  // the page's key mean: float64 sums of exact values, so the order of the rows does not show
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
  int block_q, causal, chunks;
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

constexpr int kScorePages = 256;  // pages of a scoring workgroup

// Scores of a unit against 256 pages: the bf16 mean of its query rows times each page's bf16 key mean, products and sums
// in float64. Those products are exact and their sums all but always, so the order of a sum does not show in the score.
template <typename T, int D>
__global__ __launch_bounds__(256) void cache_score_kernel(const SelectParams p) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes;
  __shared__ double part[kRows][D];
  __shared__ float qm[D];
  const int tid = threadIdx.x;
  const int64_t row = static_cast<int>(blockIdx.x) / p.chunks;
  const int64_t first = static_cast<int64_t>(static_cast<int>(blockIdx.x) % p.chunks) * kScorePages;
  const Unit n = unit_of(p, static_cast<int>(row));
  float *out = p.score + row * p.max_pages;
  const int64_t end = first + kScorePages < p.max_pages ? first + kScorePages : p.max_pages;
  if (first >= n.view.seen) {
    for (int64_t j = first + tid; j < end; j += 256) out[j] = -__builtin_inff();
    return;
  }
  const int lane = tid % kLanes, grp = tid / kLanes;
  const int rows = static_cast<int>((n.t1 - n.t0) * p.G);
  {
    double s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    const T *q = static_cast<const T *>(p.q) + n.b * p.qsb + n.h * p.G * p.qsh + n.t0 * p.qst + lane * 8;
    for (int r = grp; r < rows; r += kRows) {
      float x[8];
      load8(q + (r / p.G) * p.qst + (r % p.G) * p.qsh, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += static_cast<double>(x[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[grp][lane * 8 + i] = s[i];
  }
  __syncthreads();
  if (tid < D) {
    double s = 0;
    for (int i = 0; i < kRows && i < rows; ++i) s += part[i][tid];
    qm[tid] = round_bf16(static_cast<float>(s / rows));
  }
  __syncthreads();
  double qd[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) qd[i] = static_cast<double>(qm[lane * 8 + i]);
  for (int64_t j = first + grp; j < end; j += kRows) {
    int64_t pid = -1;
    if (j < n.view.seen) {
      pid = p.table[n.b * p.table_stride + j];
      if (pid >= p.pages) pid = -1;
    }
    double s = 0;
    if (pid >= 0) {
      const u32x4 m = *reinterpret_cast<const u32x4 *>(p.mean + (pid * p.H + n.h) * D + lane * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t word = m[i >> 1];
        s = fma(qd[i], static_cast<double>(__uint_as_float(i & 1 ? word & 0xffff0000u : word << 16)), s);
      }
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) s += xor_lane(s, o);
    float f = static_cast<float>(s);
    if (pid < 0 || f != f) f = -__builtin_inff();
    if (lane == 0) out[j] = f;
  }
}

// Scores as integers in the same order (-0 as 0); anything is above 0, the mark of a page that is not free to choose.
__device__ __forceinline__ uint32_t score_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The list of one unit. Wave w holds the scores of pages [w * 64 E, (w + 1) * 64 E) in registers, page base + i * 64 + lane
// in element i. The keep-th largest is found bit by bit from the top, one count of all elements a bit; a count that
// meets `keep` exactly ends it.
template <int kWaves, int E>
__global__ __launch_bounds__(kWaves * 64) void cache_list_kernel(const SelectParams p) {
  __shared__ int sums[2][kWaves], wave_total[kWaves], wave_equal[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const Unit n = unit_of(p, blockIdx.x);
  const float *score = p.score + row * p.max_pages;
  const int64_t seen = n.view.seen;
  const int64_t base = static_cast<int64_t>(wave) * 64 * E;
  const int64_t tail = n.view.own - (p.recent - 1);  // pages from here on are listed
  uint32_t key[E];
  uint32_t forced = 0;
  static_assert(E <= 32, "one bit an element");
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int64_t j = base + i * 64 + lane;
    key[i] = 0;
    if (j < seen) {
      if (j < p.sink || j >= tail)
        forced |= 1u << i;
      else
        key[i] = score_key(score[j]);
    }
  }
  int turn = 0;
  auto total = [&](uint32_t at_least) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) c += __popcll(__ballot(key[i] >= at_least));
    if (lane == 0) sums[turn][wave] = c;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += sums[turn][w];
    turn ^= 1;  // the next count writes the other half: one barrier a count
    return s;
  };
  const int free_pages = total(1);
  uint32_t cut = 1;  // chosen: key > cut, and the first `ties` of key == cut; or key >= cut
  int ties = -1;     // -1: all that equal the cut
  if (p.keep < free_pages) {
    const int keep = static_cast<int>(p.keep);
    uint32_t t = 0;
    bool exact = false;
    if (keep == 0) {
      t = 0xffffffffu;  // no score has this key (it would be a NaN)
      exact = true;
    }
    for (int bit = 31; bit >= 0 && !exact; --bit) {
      const uint32_t cand = t | (1u << bit);
      const int c = total(cand);
      if (c >= keep) t = cand;
      exact = c == keep;
    }
    cut = t;
    if (!exact) ties = keep - (t == 0xffffffffu ? 0 : total(t + 1));
  }
  // places: lists ascend, so every wave needs what the waves before it chose (and how many equal the cut)
  uint64_t pick[E];
  int eq_before = 0, chosen = 0;
  if (ties >= 0) {
    int eq = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) eq += __popcll(__ballot(key[i] == cut));
    if (lane == 0) wave_equal[wave] = eq;
    __syncthreads();
    for (int w = 0; w < wave; ++w) eq_before += wave_equal[w];
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    bool take = (forced >> i) & 1;
    if (ties < 0) {
      take = take || key[i] >= cut;
    } else {
      const uint64_t eq = __ballot(key[i] == cut);
      take = take || key[i] > cut || (key[i] == cut && eq_before + lanes_below(eq) < ties);
      eq_before += __popcll(eq);
    }
    pick[i] = __ballot(take);
    chosen += __popcll(pick[i]);
  }
  if (lane == 0) wave_total[wave] = chosen;
  __syncthreads();
  int at = 0, all = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) at += wave_total[w];
    all += wave_total[w];
  }
  int32_t *list = p.index + row * p.width;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int place = at + lanes_below(pick[i]);
    if ((pick[i] >> lane & 1) && place < p.width) list[place] = static_cast<int32_t>(base + i * 64 + lane);
    at += __popcll(pick[i]);
  }
  for (int64_t i = all + tid; i < p.width; i += kWaves * 64) list[i] = -1;
  if (tid == 0) p.count[row] = all < p.width ? all : static_cast<int32_t>(p.width);
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
  p.chunks = static_cast<int>(cdiv(max_pages, kScorePages));
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
  else if (max_pages <= 8192) hipLaunchKernelGGL((cache_list_kernel<16, 8>), list, dim3(1024), 0, s, p);
  else hipLaunchKernelGGL((cache_list_kernel<16, 32>), list, dim3(1024), 0, s, p);
  return check_launch("vasc_cache_select");
}
