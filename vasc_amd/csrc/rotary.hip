// Rotary positions with several axes (time, height, width, ...): every pair
// (j, j + d/2) of an axis' section turns by position * frequency.
//
// Bound: HBM, each element read and written once. A workgroup takes a tile of
// tokens and computes its cos / sin once, into LDS, for all heads: the angle
// is a float64 product (a float32 one is off by whole radians at positions of
// some millions), reduced mod 2 pi in float64 and handed to sincosf as a
// float32 with its rounding error, which a first-order term puts back. The
// rows then stream through registers, V elements of each half per thread and
// load: V is the widest vector (at most 16 bytes) that the sections' halves,
// the strides and the pointers allow.
// Measured (bf16, 16 + 16 heads of 64, sections 16 + 24 + 24, so V = 4): 24
// frames of 1041 tokens in 46 us, 4.45 TB/s where a large copy reaches 4.75;
// one frame in 6.0 us, the latency of positions, sines, barrier and rows.
// A section whose half is odd leaves V = 1: the clip again and again, partly
// from the cache behind HBM, 34 us with V = 4, 58 with sections 6 + 28 + 30,
// 75 with 6 + 28 + 28, whose 33 pieces a row leave 25 of 256 threads idle.
#include "common.h"
#include "stream.h"

namespace vasc {
namespace {

constexpr int kMaxAxes = 4;

struct RotaryTensor {
  const void *in;
  int64_t sb, sh, st;
  void *out;
  int64_t ob, oh, ot;
  int heads;
};

struct RotaryParams {
  RotaryTensor t[2];  // q, k (heads 0: absent)
  int64_t B, T;
  int D, R, tile;  // R: pairs of all sections
  int half[kMaxAxes];
  const int32_t *pos;
  int64_t psb, pst;
  int axes;
  const double *freq;
  int inverse;
  int head_inner[2];  // rows walk heads inside tokens (the memory order of [B,T,H,D])
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

template <typename T, int V>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
  extern __shared__ float lds[];
  const int tid = threadIdx.x;
  const int64_t tiles = cdiv(p.T, p.tile);
  const int64_t b = blockIdx.x / tiles;
  const int64_t t0 = (blockIdx.x % tiles) * p.tile;
  const int nt = static_cast<int>(min(static_cast<int64_t>(p.tile), p.T - t0));
  float *lcos = lds, *lsin = lds + p.tile * p.R;
  for (int i = tid; i < nt * p.R; i += 256) {
    const int t = i / p.R, f = i % p.R;
    int a = 0, first = 0;
    while (f >= first + p.half[a]) first += p.half[a++];
    const double ang = static_cast<double>(p.pos[b * p.psb + (t0 + t) * p.pst + a]) * p.freq[f];
    const double n = rint(ang * 0.15915494309189535);  // 1 / (2 pi)
    double r = fma(-n, 6.283185307179586, ang);
    r = fma(-n, 2.4492935982947064e-16, r);
    const float rh = static_cast<float>(r), rl = static_cast<float>(r - static_cast<double>(rh));
    float s, c;
    sincosf(rh, &s, &c);
    const float s2 = fmaf(c, rl, s), c2 = fmaf(-s, rl, c);
    lcos[i] = c2;
    lsin[i] = p.inverse ? -s2 : s2;
  }
  __syncthreads();
  // V-wide pieces of a row: first the pairs, then the features that are copied
  const int pairs = p.R / V, tail = (p.D - 2 * p.R) / V;
  const int pieces = pairs + tail;
  const int c = tid % pieces, lanes = 256 / pieces;
  const int r0 = tid / pieces;
  if (r0 >= lanes) return;
  int lo = 2 * p.R + (c - pairs) * V, hi = -1, f = 0;
  if (c < pairs) {
    int a = 0, first = 0;
    f = c * V;
    while (f >= first + p.half[a]) first += p.half[a++];
    lo = 2 * first + (f - first);
    hi = lo + p.half[a];
  }
  for (int w = 0; w < 2; ++w) {
    const RotaryTensor &x = p.t[w];
    const int rows = nt * x.heads;
    const T *in = static_cast<const T *>(x.in) + b * x.sb + t0 * x.st;
    T *out = static_cast<T *>(x.out) + b * x.ob + t0 * x.ot;
#pragma unroll 4
    for (int r = r0; r < rows; r += lanes) {
      int t, h;
      if (p.head_inner[w]) {
        t = r / x.heads;
        h = r - t * x.heads;
      } else {
        h = r / nt;
        t = r - h * nt;
      }
      const T *src = in + t * x.st + h * x.sh;
      T *dst = out + t * x.ot + h * x.oh;
      if (hi < 0) {
        *reinterpret_cast<Pack<T, V> *>(dst + lo) = *reinterpret_cast<const Pack<T, V> *>(src + lo);
        continue;
      }
      const Pack<T, V> l = *reinterpret_cast<const Pack<T, V> *>(src + lo);
      const Pack<T, V> g = *reinterpret_cast<const Pack<T, V> *>(src + hi);
      Pack<T, V> lo_out, hi_out;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float cs = lcos[t * p.R + f + e], sn = lsin[t * p.R + f + e];
        const float xl = to_f32(l.v[e]), xh = to_f32(g.v[e]);
        lo_out.v[e] = from_f32<T>(xl * cs - xh * sn);
        hi_out.v[e] = from_f32<T>(xh * cs + xl * sn);
      }
      *reinterpret_cast<Pack<T, V> *>(dst + lo) = lo_out;
      *reinterpret_cast<Pack<T, V> *>(dst + hi) = hi_out;
    }
  }
}

template <typename T, int V>
int launch(const RotaryParams &p, hipStream_t s) {
  const int64_t grid = p.B * cdiv(p.T, p.tile);
  hipLaunchKernelGGL((rotary_kernel<T, V>), dim3(static_cast<unsigned>(grid)), dim3(256),
                     static_cast<unsigned>(2 * p.tile * p.R * sizeof(float)), s, p);
  return check_launch("vasc_rotary_axes");
}

template <typename T>
int launch_width(const RotaryParams &p, int width, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (width >= 8) return launch<T, 8>(p, s);
  }
  if (width >= 4) return launch<T, 4>(p, s);
  if (width >= 2) return launch<T, 2>(p, s);
  return launch<T, 1>(p, s);
}

}  // namespace
}  // namespace vasc

extern "C" int vasc_rotary_axes(const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st, void *qo, int64_t qo_sb,
                                int64_t qo_sh, int64_t qo_st, int64_t Hq, const void *k, int64_t k_sb, int64_t k_sh,
                                int64_t k_st, void *ko, int64_t ko_sb, int64_t ko_sh, int64_t ko_st, int64_t Hk,
                                int64_t B, int64_t T, int64_t D, const int32_t *pos, int64_t pos_sb, int64_t pos_st,
                                int32_t axes, const int64_t *sections, const double *inv_freq, int32_t dtype,
                                int32_t inverse, void *stream) {
  using namespace vasc;
  VASC_REQUIRE(q && qo && pos && inv_freq && sections, "q, qo, pos, inv_freq and sections are required");
  VASC_REQUIRE((k == nullptr) == (ko == nullptr), "k and ko go together");
  VASC_REQUIRE(B > 0 && T > 0 && Hq > 0 && (!k || Hk > 0), "empty tensor");
  VASC_REQUIRE(D > 0 && D <= 256, "D %lld outside [1, 256]", (long long)D);
  VASC_REQUIRE(Hq < (1 << 16) && Hk < (1 << 16), "too many heads");
  VASC_REQUIRE(axes >= 1 && axes <= kMaxAxes, "axes %d outside [1, %d]", axes, kMaxAxes);
  VASC_SUPPORTED(dtype >= 0 && dtype <= 2, "dtype %d not built", dtype);
  RotaryParams p = {};
  int64_t width = dtype == 2 ? 4 : 8, at = 0;
  auto fit = [&](int64_t x) {
    while (x % width) width >>= 1;
  };
  for (int a = 0; a < axes; ++a) {
    VASC_REQUIRE(sections[a] > 0 && sections[a] % 2 == 0 && sections[a] <= D, "section %lld must be even and positive",
                 (long long)sections[a]);
    p.half[a] = static_cast<int>(sections[a] / 2);
    fit(p.half[a]);
    at += sections[a];
  }
  VASC_REQUIRE(at <= D, "the sections hold %lld features, the head %lld", (long long)at, (long long)D);
  p.R = static_cast<int>(at / 2);
  fit(D);
  const int64_t size = dtype == 2 ? 4 : 2;
  auto fit_tensor = [&](const void *ptr, int64_t sb, int64_t sh, int64_t st) {
    fit(static_cast<int64_t>(reinterpret_cast<uintptr_t>(ptr) / size));
    fit(sb);
    fit(sh);
    fit(st);
  };
  fit_tensor(q, q_sb, q_sh, q_st);
  fit_tensor(qo, qo_sb, qo_sh, qo_st);
  if (k) {
    fit_tensor(k, k_sb, k_sh, k_st);
    fit_tensor(ko, ko_sb, ko_sh, ko_st);
  }
  p.t[0] = {q, q_sb, q_sh, q_st, qo, qo_sb, qo_sh, qo_st, static_cast<int>(Hq)};
  p.t[1] = {k, k_sb, k_sh, k_st, ko, ko_sb, ko_sh, ko_st, k ? static_cast<int>(Hk) : 0};
  p.head_inner[0] = qo_sh <= qo_st;
  p.head_inner[1] = ko_sh <= ko_st;
  p.B = B;
  p.T = T;
  p.D = static_cast<int>(D);
  p.pos = pos;
  p.psb = pos_sb;
  p.pst = pos_st;
  p.axes = axes;
  p.freq = inv_freq;
  p.inverse = inverse;
  p.tile = 8;
  while (p.tile > 1 && B * cdiv(T, p.tile) < 512) p.tile >>= 1;
  VASC_REQUIRE(B * cdiv(T, p.tile) < (int64_t(1) << 31), "too many tokens");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int w = static_cast<int>(width);
  if (dtype == 0) return launch_width<__bf16>(p, w, s);
  if (dtype == 1) return launch_width<_Float16>(p, w, s);
  return launch_width<float>(p, w, s);
}
