// Pages of a block cache (8 or 4 bits): copies of whole pages, tokens moved to the front of other pages, and the page
// tables of sequences that share pages (fork, reserve, free), whose holders are counted in refs[pages].
//
// The counts are all that is kept: a page is free where its count is not positive, and the lowest free pages are given out
// first. So what a call gives does not depend on the order of earlier calls, of its own atomics, or of its workgroups.
//
// Measured, in us: eight branches of four sequences of up to 64 pages: fork 2.6, reserve 6.6, copy 4.5, free 2.5, the latency
// of a few loads that depend on one another; 256 branches of 64 sequences of up to 1024 pages, in a pool of 45000: 9.2,
// 7.2 and 5.8, 5.8, 9.3. A host that calls them one by one takes longer for each (5 to 12): the four calls 32 and 37, in a
// graph 14.5 and 35.
#include "cache_page.h"

namespace vasc {
namespace {

// ------------------------------------------------------------------ copies
// The arrays of a cache as pieces of 16 bytes: a page is contiguous in each.
struct PageArrays {
  u32x4 *at[6];
  int32_t size[6];  // 16-byte pieces of a page
  int32_t all;
};

constexpr int kCopyPieces = 1024;  // of a workgroup: 16 KB, four loads a thread in flight

// Bound by HBM (or, few pages, by the latency of list, load and store).
__global__ __launch_bounds__(256) void page_copy_kernel(const PageArrays a, const int32_t *src, const int32_t *dst,
                                                        int64_t pages, int chunks) {
  const int64_t i = static_cast<uint32_t>(blockIdx.x) / static_cast<uint32_t>(chunks);
  const int64_t s = src[i], d = dst[i];
  if (s < 0 || s >= pages || d < 0 || d >= pages || s == d) return;
  const int first = (static_cast<int>(blockIdx.x) - static_cast<int>(i) * chunks) * kCopyPieces + threadIdx.x;
  u32x4 x[4];
  u32x4 *to[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    int at = first + k * 256;
    to[k] = nullptr;
    if (at >= a.all) continue;
#pragma unroll
    for (int n = 0; n < 6; ++n) {
      if (at >= 0 && at < a.size[n]) {
        x[k] = a.at[n][s * a.size[n] + at];
        to[k] = a.at[n] + d * a.size[n] + at;
      }
      at -= a.size[n];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (to[k]) *to[k] = x[k];
}

// ------------------------------------------------------------------ compaction
struct CompactArgs {
  CacheArgs c;  // table: of the sequences that are read
  const int32_t *index;
  int64_t isb, ish;
  const int32_t *count;  // tokens of a sequence, or NULL: n
  int64_t n;
  const int32_t *out_table;
  int64_t out_stride, out_pages;
  int32_t H, span;
};

// The 4x4 bytes that a quad of lanes holds, transposed: lane q gets byte q of lanes 0..3.
__device__ __forceinline__ uint32_t quad_transpose(uint32_t v) {
  const int q = __lane_id() & 3;
  const uint32_t a = __builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x00, 0xf, 0xf, false);
  const uint32_t b = __builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x55, 0xf, 0xf, false);
  const uint32_t c = __builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xaa, 0xf, 0xf, false);
  const uint32_t d = __builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xff, 0xf, 0xf, false);
  const int sh = 8 * q;
  return (a >> sh & 255u) | (b >> sh & 255u) << 8 | (c >> sh & 255u) << 16 | (d >> sh & 255u) << 24;
}

// One workgroup writes one (page, head), 64 chosen tokens from wherever they lie. Keys are rows. Values lie transposed, a
// byte (or half of one) of a feature a token: a wave reads a feature of its 64 tokens at a time, which is one 64-byte line
// where they are neighbours and never more than a line a token, and turns 4 x 4 bytes between lanes for the store.
// Bound by the accesses to the first cache where single tokens are kept, and by HBM where runs are: a quarter of the tokens of
// 16 sequences, others for each of 8 heads of 128 (4 bits), in 51 us, 24.1e6 accesses (94000 in a CU's 141000 cycles, some 30 a
// load of a feature) and 126 MB of traffic (2.5 TB/s); 32 of 128 frames, 16 heads of 64 (8 bits), in 31 us (4.4 TB/s).
template <int D, int kBits>
__global__ __launch_bounds__(256) void compact_kernel(const CompactArgs p) {
  constexpr int kG = D / 32, kRowBytes = D * kBits / 8;
  constexpr int kPiece = kBits == 4 && D == 64 ? 8 : 16;  // contiguous bytes of a key row
  constexpr int kLanes = kRowBytes / kPiece, kRows = 256 / kLanes;
  constexpr int kS = kRowBytes + 4;
  constexpr int kKeyScales = kBits == 8 ? 1 : kG;
  constexpr int kCodes = kBits == 8 ? 4 : 8;                      // of a word
  constexpr int kWords = D / kCodes, kGroups = 256 / kWords;      // the mean: a word of columns a thread
  __shared__ int64_t from[kPage];                                 // (page, head) of the source, or -1
  __shared__ uint8_t slot[kPage];
  __shared__ __align__(16) uint8_t kt[kPage * kS];
  __shared__ uint8_t ke[kPage][kKeyScales], vn[kPage][kG];
  __shared__ double part[kGroups][D];
  const CacheArgs &c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t ph0 = blockIdx.x / static_cast<uint32_t>(p.span);
  const int64_t j = blockIdx.x - ph0 * static_cast<uint32_t>(p.span);
  const int64_t b = ph0 / static_cast<uint32_t>(p.H), h = ph0 - static_cast<uint32_t>(b) * static_cast<uint32_t>(p.H);
  int64_t n = p.count ? p.count[b] : p.n;
  n = n < 0 ? 0 : (n < p.n ? n : p.n);
  const int hi = static_cast<int>(n - j * kPage < kPage ? n - j * kPage : kPage);
  if (hi <= 0 || j >= p.out_pages) return;
  const int64_t pid = p.out_table[b * p.out_stride + j];
  if (pid < 0 || pid >= c.pages) return;
  const int64_t ph = pid * p.H + h;
  if (tid < kPage) {
    int64_t f = -1;
    int64_t t = -1;
    if (tid < hi) t = p.index[b * p.isb + h * p.ish + j * kPage + tid];
    if (t >= 0 && t < c.max_pages * kPage) {
      f = c.table[b * c.table_stride + t / kPage];
      f = f < 0 || f >= c.pages ? -1 : f * p.H + h;
    }
    from[tid] = f;
    slot[tid] = static_cast<uint8_t>(t & (kPage - 1));
  }
  __syncthreads();
  // values: lane = token. All of a wave's loads are on their way at once (in two batches, after the keys: 66 us for 8 heads'
  // quarter of the tokens of 16 sequences up to 16384 long, single tokens by chance; so 51).
  constexpr int kFeatures = D / 4;  // of a wave
  const int64_t f_lane = lane < hi ? from[lane] : -1;
  const int at = page_place(slot[lane]);
  uint32_t x[kFeatures];
  {
    const uint8_t *src = c.vc + f_lane * (kPage * kRowBytes);
#pragma unroll
    for (int i = 0; i < kFeatures; ++i) {
      const int d = wave * kFeatures + i;
      x[i] = 0;
      if (f_lane >= 0) x[i] = kBits == 8 ? src[d * kPage + at] : src[value4_at(d, at >> 4) + (at & 15) / 2];
    }
  }
  // keys; a token that does not exist is zeros under the smallest power
#pragma unroll
  for (int pass = 0; pass < kPage / kRows; ++pass) {
    const int row = pass * kRows + tid / kLanes, piece = tid % kLanes;
    if (row >= hi) continue;
    const int64_t f = from[row];
    const int s = slot[row];
    typedef uint32_t piece_t __attribute__((ext_vector_type(kPiece / 4)));
    piece_t x = {};
    auto place = [&](int t) { return kBits == 8 ? t * D + piece * 16 : key4_at<D>(t, piece * 16 * (kPiece / 8)); };
    if (f >= 0) x = *reinterpret_cast<const piece_t *>(c.kc + f * (kPage * kRowBytes) + place(s));
    *reinterpret_cast<piece_t *>(c.kc + ph * (kPage * kRowBytes) + place(row)) = x;
#pragma unroll
    for (int i = 0; i < kPiece / 4; ++i) *reinterpret_cast<uint32_t *>(kt + row * kS + piece * kPiece + i * 4) = x[i];
  }
  if (tid < kPage * kKeyScales) {
    const int row = tid & 63, gr = tid >> 6;
    if (row < hi) {
      const int64_t f = from[row];
      const uint8_t e = f >= 0 ? c.ks[(f * kKeyScales + gr) * kPage + key_place(slot[row])] : 67;
      ke[row][gr] = e;
      c.ks[(ph * kKeyScales + gr) * kPage + key_place(row)] = e;
    }
  }
  if (kBits == 4 && tid < kPage * kG) {
    const int row = tid & 63, gr = tid >> 6;
    if (row < hi) {
      const int64_t f = from[row];
      const int at = page_place(slot[row]), i = at & 15;
      uint32_t off = 15;
      if (f >= 0)
        off = *reinterpret_cast<const uint32_t *>(c.vo + f * (kG * 32) + ((at >> 4) * kG + gr) * 8 + (i >> 3) * 4) >> offset4_bit(i & 7) & 15u;
      vn[row][gr] = static_cast<uint8_t>(off);
    }
  }
  {
    const int to = page_place(lane & ~3);
    const bool whole = (lane | 3) < hi;
    if (wave == 0 && lane < hi) c.vs[ph * kPage + page_place(lane)] = f_lane >= 0 ? c.vs[f_lane * kPage + at] : 67;
    uint8_t *dst = c.vc + ph * (kPage * kRowBytes);
#pragma unroll
    for (int i = 0; i < kFeatures; i += 4) {
      if (kBits == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[i + k] = x[i + k] >> (4 * (at & 1)) & 15u;
      }
      // this lane's feature of the quad's four tokens
      uint32_t v = quad_transpose(x[i] | x[i + 1] << 8 | x[i + 2] << 16 | x[i + 3] << 24);
      const int d = wave * kFeatures + i + (lane & 3);
      if (kBits == 8) {
        uint8_t *o = dst + d * kPage + to;
        if (whole) {
          *reinterpret_cast<uint32_t *>(o) = v;
        } else {
#pragma unroll
          for (int k = 0; k < 3; ++k)
            if ((lane & ~3) + k < hi) o[k] = static_cast<uint8_t>(v >> (8 * k));
        }
      } else {
        v = (v | v >> 4) & 0x00ff00ffu;
        v = (v | v >> 8) & 0xffffu;
        uint16_t *o = reinterpret_cast<uint16_t *>(dst + value4_at(d, to >> 4) + (to & 15) / 2);
        const int have = hi - (lane & ~3);
        if (have < 4 && have > 0) {
          const uint32_t cover = (1u << (4 * have)) - 1u;
          v = (v & cover) | (*o & ~cover);
        }
        if (have > 0) *o = static_cast<uint16_t>(v);
      }
    }
  }
  __syncthreads();
  if (kBits == 4 && tid < 8 * kG) {  // the offsets: a word holds eight tokens of a group
    const int half = tid & 1, grp = (tid >> 1) % kG, g = tid / (2 * kG);
    uint32_t cover = 0, out = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int t = token4_of(g, half * 8 + k);
      if (t >= hi) continue;
      cover |= 15u << offset4_bit(k);
      out |= static_cast<uint32_t>(vn[t][grp]) << offset4_bit(k);
    }
    if (cover) {
      uint32_t *o = reinterpret_cast<uint32_t *>(c.vo + ph * (kG * 32) + (g * kG + grp) * 8 + half * 4);
      if (cover != 0xffffffffu) out |= *o & ~cover;
      *o = out;
    }
  }
  // the page's key mean, as a write sums it
  {
    const int grp = tid / kWords, word = tid % kWords;
    double s[kCodes];
#pragma unroll
    for (int i = 0; i < kCodes; ++i) s[i] = 0;
    for (int row = grp; row < hi; row += kGroups) {
      float f[kCodes];
      const uint32_t w = *reinterpret_cast<const uint32_t *>(kt + row * kS + word * 4);
      const float e = pow2_byte(ke[row][kBits == 8 ? 0 : word / 4]);
      if constexpr (kBits == 8) {
        unpack_e4m3(w, f);
#pragma unroll
        for (int i = 0; i < kCodes; ++i) f[i] *= e;
      } else {
        unpack_e2m1(w, f, e);
      }
#pragma unroll
      for (int i = 0; i < kCodes; ++i) s[i] += static_cast<double>(f[i]);
    }
#pragma unroll
    for (int i = 0; i < kCodes; ++i) part[grp][word * kCodes + i] = s[i];
  }
  __syncthreads();
  if (tid < D) {
    double s = 0;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) s += part[i][tid];
    c.mean[ph * D + tid] = f32_to_bf16(static_cast<float>(s / hi));
  }
}

// ------------------------------------------------------------------ page tables
// Pages of so many tokens.
__device__ __forceinline__ int64_t pages_of(int64_t tokens) { return (tokens + kPage - 1) / kPage; }

// Rows of a table that share their pages with the rows they come from: an entry a thread.
__global__ __launch_bounds__(256) void fork_kernel(int32_t *refs, int64_t pages, const int32_t *table, int64_t stride,
                                                   int64_t max_pages, const int32_t *lengths, int64_t B,
                                                   const int32_t *source, int32_t *out, int32_t *out_lengths, int chunks) {
  const int64_t row = blockIdx.x / static_cast<uint32_t>(chunks);
  const int64_t j = static_cast<int64_t>(blockIdx.x - static_cast<uint32_t>(row) * static_cast<uint32_t>(chunks)) * 256 + threadIdx.x;
  const int64_t s = source[row];
  const int64_t L = s >= 0 && s < B ? clamp_tokens(lengths[s], max_pages) : 0;
  if (j == 0) out_lengths[row] = static_cast<int32_t>(L);
  if (j >= max_pages) return;
  int32_t e = -1;
  if (j < pages_of(L)) {
    e = table[s * stride + j];
    if (e >= 0 && e < pages) atomicAdd(refs + e, 1);
    else e = -1;
  }
  out[row * max_pages + j] = e;
}

// Gives back what lies behind the first `keep` tokens. The length's new value gives the same pages as the old.
__global__ __launch_bounds__(256) void free_kernel(int32_t *refs, int64_t pages, int32_t *table, int64_t stride,
                                                   int64_t max_pages, int32_t *lengths, const int32_t *keep, int chunks) {
  const int64_t row = blockIdx.x / static_cast<uint32_t>(chunks);
  const int64_t j = static_cast<int64_t>(blockIdx.x - static_cast<uint32_t>(row) * static_cast<uint32_t>(chunks)) * 256 + threadIdx.x;
  int64_t L = clamp_tokens(lengths[row], max_pages);
  if (keep) {
    const int64_t k = keep[row];
    L = k < L ? (k > 0 ? k : 0) : L;
  } else {
    L = 0;
  }
  if (j == 0) lengths[row] = static_cast<int32_t>(L);
  if (j >= max_pages || j < pages_of(L)) return;
  const int32_t e = table[row * stride + j];
  if (e >= 0 && e < pages) atomicSub(refs + e, 1);
  table[row * stride + j] = -1;
}

constexpr int32_t kMissing = -1, kKept = -2;
constexpr int32_t kRefused = -1;

struct ReserveArgs {
  int32_t *refs;
  int64_t pages;
  int32_t *table;
  int64_t stride, max_pages;
  const int32_t *lengths, *count;
  int64_t tokens;
  int32_t B, span, chunks;
  int32_t *granted, *src, *dst;
  uint64_t *free;          // a bit a page
  int32_t *chunk, *need;   // free pages of each chunk, pages that each sequence needs
  int32_t *list;           // [B][span]: a sequence's new pages
  int32_t *mark;           // [B][span]: of the pages that it touches, the one to be replaced, kMissing or kKept
};

constexpr int kChunk = 4096;  // pages of a chunk: a word of free bits a lane

struct Growth {
  int64_t L, fit;  // tokens held, and to come
  int64_t first;   // the first page that these touch
  int n;           // how many they touch
};
__device__ __forceinline__ Growth growth(const ReserveArgs &p, int64_t b) {
  Growth w;
  w.L = clamp_tokens(p.lengths[b], p.max_pages);
  w.fit = p.count ? p.count[b] : p.tokens;
  w.fit = w.fit < p.tokens ? w.fit : p.tokens;
  w.fit = w.fit < p.max_pages * kPage - w.L ? w.fit : p.max_pages * kPage - w.L;
  if (w.fit < 0) w.fit = 0;
  w.first = w.L / kPage;
  w.n = w.fit > 0 ? static_cast<int>(pages_of(w.L + w.fit) - w.first) : 0;
  return w;
}

// A wave's 1024 pages: the words of their free bits; returns how many are free.
__device__ __forceinline__ int count_free(const ReserveArgs &p, int64_t base, uint64_t *free) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  int32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t at = base + i * 64 + lane;
    r[i] = at < p.pages ? p.refs[at] : 1;
  }
  uint64_t mine = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t bits = __ballot(r[i] <= 0);
    n += __popcll(bits);
    if (lane == i) mine = bits;
  }
  if (lane < 16) free[base / 64 + lane] = mine;
  return n;
}

// The pages that sequence b needs, or kRefused. All of it is decided here, on the holders before the call: a page that nobody
// counts is free, so it may be given to any sequence of the call, and its count says nothing from then on. Such a page is
// missing; where it is the one with the sequence's last tokens, they may be gone, and the sequence gets nothing.
// The table keeps its entries until the sequence is served.
__device__ __forceinline__ int count_needs(const ReserveArgs &p, int64_t b) {
  const int lane = threadIdx.x & 63;
  const Growth w = growth(p, b);
  int n = 0;
  for (int i0 = 0; i0 < w.n; i0 += 64) {
    const int i = i0 + lane;
    int32_t mark = kKept;
    bool lost = false;
    if (i < w.n) {
      const int32_t e = p.table[b * p.stride + w.first + i];
      const bool page = e >= 0 && e < p.pages;
      const int32_t holders = page ? p.refs[e] : 0;
      if (holders != 1) mark = holders > 0 ? e : kMissing;
      p.mark[b * p.span + i] = mark;
      lost = page && holders <= 0 && i == 0 && w.L % kPage;
    }
    if (__ballot(lost)) return kRefused;
    n += __popcll(__ballot(mark != kKept));
  }
  return n;
}

__device__ __forceinline__ int wave_scan(int v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o);
    if (__lane_id() >= static_cast<unsigned>(o)) v += u;
  }
  return v;
}

// Serves sequence b: it has the free pages of ranks [before, before + need), if there are so many.
__device__ __forceinline__ void take_pages(const ReserveArgs &p, int64_t b, const uint64_t *free, const int32_t *chunk,
                                           const int32_t *needs) {
  const int lane = threadIdx.x & 63;
  const Growth w = growth(p, b);
  const int need = needs[b];
  int32_t src = -1, dst = -1;
  int64_t granted = need == kRefused ? 0 : w.fit;
  if (need > 0) {
    int64_t before = 0;
    {
      int v = 0;
      for (int i = lane; i < b; i += 64) v += max(needs[i], 0);
      before = wave_sum_int(v);
    }
    const int64_t end = before + need;
    // a lane's word of each chunk that holds some of the ranks
    int64_t seen = 0;
    int32_t *list = p.list + b * p.span;
    for (int c0 = 0; c0 < p.chunks && seen < end; c0 += 64) {
      const int mine = c0 + lane < p.chunks ? chunk[c0 + lane] : 0;
      const int upto = wave_scan(mine);
      const int all = __shfl(upto, 63);
      uint64_t hit = __ballot(mine > 0 && seen + upto > before && seen + upto - mine < end);
      while (hit) {
        const int i = __ffsll(static_cast<unsigned long long>(hit)) - 1;
        hit &= hit - 1;
        const int64_t base = static_cast<int64_t>(c0 + i) * kChunk + lane * 64;
        uint64_t bits = free[base / 64];
        const int n = __popcll(bits);
        int64_t rank = seen + __shfl(upto - mine, i) + wave_scan(n) - n;  // of this word's first
        if (rank + n <= before || rank >= end) continue;
        for (; bits && rank < end; ++rank, bits &= bits - 1)
          if (rank >= before) list[rank - before] = static_cast<int32_t>(base + __ffsll(static_cast<unsigned long long>(bits)) - 1);
      }
      seen += all;
    }
    __threadfence_block();  // the list's lanes are others than those that wrote it
    __builtin_amdgcn_wave_barrier();
    const bool ok = seen >= end;
    if (!ok) granted = 0;
    int done = 0;
    for (int i0 = 0; ok && i0 < w.n; i0 += 64) {
      const int i = i0 + lane;
      const int32_t old = i < w.n ? p.mark[b * p.span + i] : kKept;
      const uint64_t flags = __ballot(old != kKept);
      if (old != kKept) {
        const int32_t page = list[done + lanes_below(flags)];
        p.table[b * p.stride + w.first + i] = page;
        p.refs[page] = 1;  // it was free, and `old` was not: no other store of the call meets this one
        if (old >= 0) atomicSub(p.refs + old, 1);
        if (i == 0 && w.L % kPage && old >= 0) {
          src = old;
          dst = page;
        }
      }
      done += __popcll(flags);
    }
  }
  if (lane == 0) {
    p.granted[b] = static_cast<int32_t>(granted);
    p.src[b] = src;
    p.dst[b] = dst;
  }
}

// First: what is free (a wave 1024 pages), and what each sequence needs (a wave a sequence).
__global__ __launch_bounds__(256) void reserve_count_kernel(const ReserveArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (static_cast<int>(blockIdx.x) < p.chunks) {
    __shared__ int sum[4];
    const int n = count_free(p, static_cast<int64_t>(blockIdx.x) * kChunk + wave * (kChunk / 4), p.free);
    if (lane == 0) sum[wave] = n;
    __syncthreads();
    if (threadIdx.x == 0) p.chunk[blockIdx.x] = sum[0] + sum[1] + sum[2] + sum[3];
    return;
  }
  const int64_t b = (static_cast<int64_t>(blockIdx.x) - p.chunks) * 4 + wave;
  if (b >= p.B) return;
  const int n = count_needs(p, b);
  if (lane == 0) p.need[b] = n;
}

// Second: a wave a sequence.
__global__ __launch_bounds__(256) void reserve_take_kernel(const ReserveArgs p) {
  const int64_t b = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (b < p.B) take_pages(p, b, p.free, p.chunk, p.need);
}

// Both in one workgroup, for small pools and batches, a wave a sequence. Measured, with a free of the same table, in us among
// others and alone: 16 sequences, 4000 pages 15.0 and 26.3, in two launches 17.8 and 27.8; one sequence of 30000 tokens, 16000
// pages 18.9 and 35.4, 19.5 and 36.2; 32 sequences of 100 tokens, two to a wave, 20.0 and 36.2, 17.8 and 31.9.
constexpr int kFewPages = 4 * kChunk, kFewSequences = 16;

__global__ __launch_bounds__(1024) void reserve_few_kernel(const ReserveArgs p) {
  __shared__ uint64_t free[kFewPages / 64];
  __shared__ int32_t sum[16], chunk[4], need[kFewSequences];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = count_free(p, wave * 1024, free);
  if (lane == 0) sum[wave] = n;
  if (wave < p.B) {
    const int k = count_needs(p, wave);
    if (lane == 0) need[wave] = k;
  }
  __syncthreads();
  if (threadIdx.x < 4) chunk[threadIdx.x] = sum[threadIdx.x * 4] + sum[threadIdx.x * 4 + 1] + sum[threadIdx.x * 4 + 2] + sum[threadIdx.x * 4 + 3];
  __syncthreads();
  if (wave < p.B) take_pages(p, wave, free, chunk, need);
}

int check_pool(const void *refs, int64_t pages, const void *table, int64_t stride, int64_t max_pages, const void *lengths, int64_t B) {
  VASC_REQUIRE(refs && table && lengths, "refs, the page table and lengths are required");
  VASC_REQUIRE(pages > 0 && pages < (int64_t(1) << 26), "pages outside [1, 2^26)");
  VASC_REQUIRE(max_pages > 0 && max_pages < (int64_t(1) << 24) && stride >= max_pages, "max_pages %lld with a row stride of %lld",
               (long long)max_pages, (long long)stride);
  VASC_REQUIRE(B > 0 && B <= 65536, "B %lld outside [1, 65536]", (long long)B);
  return VASC_OK;
}

int check_bits(int32_t bits, const void *vo) {
  VASC_SUPPORTED(bits == 8 || bits == 4, "bits %d not built (4, 8)", bits);
  VASC_REQUIRE((bits == 4) == (vo != nullptr), "vo belongs to the 4-bit cache");
  VASC_REQUIRE((reinterpret_cast<uintptr_t>(vo) & 15) == 0, "the cache must be 16-byte aligned");
  return VASC_OK;
}

}  // namespace
}  // namespace vasc

extern "C" int vasc_cache_copy(int32_t bits, uint8_t *kc, uint8_t *vc, uint8_t *ks, uint8_t *vs, uint8_t *vo, uint16_t *mean,
                               int64_t pages, int64_t H, int64_t D, const int32_t *src, const int32_t *dst, int64_t n,
                               void *stream) {
  using namespace vasc;
  int rc;
  if ((rc = check_bits(bits, vo))) return rc;
  if ((rc = check_cache(kc, vc, ks, vs, pages, src, 0, 1, D))) return rc;
  VASC_REQUIRE(mean && (reinterpret_cast<uintptr_t>(mean) & 15) == 0, "mean must be given and 16-byte aligned");
  VASC_REQUIRE(src && dst, "src and dst are required");
  VASC_REQUIRE(H > 0 && H < (1 << 16) && n > 0, "no heads or no pages");
  const int64_t code = H * kPage * D * bits / 8 / 16, power = H * kPage / 16;
  const int64_t size[6] = {code, code, bits == 8 ? power : power * (D / 32), power, bits == 8 ? 0 : H * D / 16, H * D / 8};
  void *at[6] = {kc, vc, ks, vs, vo, mean};
  PageArrays a;
  a.all = 0;
  for (int i = 0; i < 6; ++i) {
    a.at[i] = static_cast<u32x4 *>(at[i]);
    a.size[i] = static_cast<int32_t>(size[i]);
    a.all += a.size[i];
  }
  const int64_t chunks = cdiv(a.all, kCopyPieces);
  VASC_REQUIRE(n < (int64_t(1) << 31) / chunks, "too many pages");
  hipLaunchKernelGGL(page_copy_kernel, dim3(static_cast<unsigned>(n * chunks)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                     a, src, dst, pages, static_cast<int>(chunks));
  return check_launch("vasc_cache_copy");
}

extern "C" int vasc_cache_compact(int32_t bits, uint8_t *kc, uint8_t *vc, uint8_t *ks, uint8_t *vs, uint8_t *vo,
                                  uint16_t *mean, int64_t pages, int64_t H, int64_t D, const int32_t *page_table,
                                  int64_t table_stride, int64_t max_pages, const int32_t *index, int64_t index_sb,
                                  int64_t index_sh, const int32_t *count, int64_t B, int64_t n, const int32_t *out_table,
                                  int64_t out_stride, int64_t out_pages, void *stream) {
  using namespace vasc;
  int rc;
  if ((rc = check_bits(bits, vo))) return rc;
  if ((rc = check_cache(kc, vc, ks, vs, pages, page_table, table_stride, max_pages, D))) return rc;
  VASC_REQUIRE(mean && index && out_table, "mean, index and out_table are required");
  VASC_REQUIRE(out_pages > 0 && (out_stride >= out_pages || out_stride == 0), "out_stride %lld below out_pages", (long long)out_stride);
  VASC_REQUIRE(index_sb >= 0 && index_sh >= 0, "negative strides");
  VASC_REQUIRE(B > 0 && H > 0 && n > 0 && n < (int64_t(1) << 30), "empty tensor, or too many tokens");
  CompactArgs p = {};
  p.c = {kc, vc, ks, vs, mean, pages, page_table, table_stride, max_pages, vo};
  p.index = index; p.isb = index_sb; p.ish = index_sh;
  p.count = count; p.n = n;
  p.out_table = out_table; p.out_stride = out_stride; p.out_pages = out_pages;
  p.H = static_cast<int32_t>(H);
  p.span = static_cast<int32_t>(cdiv(n, kPage));
  VASC_REQUIRE(H < (1 << 16) && B < (int64_t(1) << 24) && B * H * p.span < (int64_t(1) << 31), "too many tokens");
  const dim3 grid(static_cast<unsigned>(B * H * p.span));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (bits == 8) {
    if (D == 64) hipLaunchKernelGGL((compact_kernel<64, 8>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((compact_kernel<128, 8>), grid, dim3(256), 0, s, p);
  } else {
    if (D == 64) hipLaunchKernelGGL((compact_kernel<64, 4>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((compact_kernel<128, 4>), grid, dim3(256), 0, s, p);
  }
  return check_launch("vasc_cache_compact");
}

extern "C" int vasc_pages_fork(int32_t *refs, int64_t pages, const int32_t *page_table, int64_t table_stride,
                               int64_t max_pages, const int32_t *lengths, int64_t B, const int32_t *source, int64_t rows,
                               int32_t *out_table, int32_t *out_lengths, void *stream) {
  using namespace vasc;
  int rc;
  if ((rc = check_pool(refs, pages, page_table, table_stride, max_pages, lengths, B))) return rc;
  VASC_REQUIRE(source && out_table && out_lengths, "source, out_table and out_lengths are required");
  const int64_t chunks = cdiv(max_pages, 256);
  VASC_REQUIRE(rows > 0 && rows < (int64_t(1) << 31) / chunks, "rows %lld", (long long)rows);
  hipLaunchKernelGGL(fork_kernel, dim3(static_cast<unsigned>(rows * chunks)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                     refs, pages, page_table, table_stride, max_pages, lengths, B, source, out_table, out_lengths,
                     static_cast<int>(chunks));
  return check_launch("vasc_pages_fork");
}

extern "C" int vasc_pages_free(int32_t *refs, int64_t pages, int32_t *page_table, int64_t table_stride, int64_t max_pages,
                               int32_t *lengths, int64_t B, const int32_t *keep, void *stream) {
  using namespace vasc;
  int rc;
  if ((rc = check_pool(refs, pages, page_table, table_stride, max_pages, lengths, B))) return rc;
  const int64_t chunks = cdiv(max_pages, 256);
  VASC_REQUIRE(B < (int64_t(1) << 31) / chunks, "too many pages");
  hipLaunchKernelGGL(free_kernel, dim3(static_cast<unsigned>(B * chunks)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                     refs, pages, page_table, table_stride, max_pages, lengths, keep, static_cast<int>(chunks));
  return check_launch("vasc_pages_free");
}

namespace vasc {
namespace {
// Workspace: free bits, free pages of the chunks, needs, lists, marks.
int64_t reserve_bytes(int64_t pages, int64_t B, int64_t span, int64_t (&at)[5]) {
  const int64_t chunks = cdiv(pages, kChunk);
  const int64_t size[5] = {chunks * (kChunk / 8), chunks * 4, B * 4, B * span * 4, B * span * 4};
  int64_t sum = 0;
  for (int i = 0; i < 5; ++i) {
    at[i] = sum;
    sum += static_cast<int64_t>(align256(size[i]));
  }
  return sum;
}
int64_t reserve_span(int64_t tokens, int64_t max_pages) {
  const int64_t span = (tokens + 2 * kPage - 2) / kPage;
  return span < max_pages ? span : max_pages;
}
}  // namespace
}  // namespace vasc

extern "C" int64_t vasc_pages_reserve_workspace_size(int64_t pages, int64_t max_pages, int64_t B, int64_t tokens) {
  using namespace vasc;
  if (!(pages > 0 && pages < (int64_t(1) << 26) && max_pages > 0 && max_pages < (int64_t(1) << 24) && B > 0 && B <= 65536 &&
        tokens > 0 && tokens < (int64_t(1) << 30)))
    return -1;
  const int64_t span = reserve_span(tokens, max_pages);
  if (B * span >= (int64_t(1) << 31)) return -1;
  int64_t at[5];
  return reserve_bytes(pages, B, span, at);
}

extern "C" int vasc_pages_reserve(int32_t *refs, int64_t pages, int32_t *page_table, int64_t table_stride, int64_t max_pages,
                                  const int32_t *lengths, int64_t B, int64_t tokens, const int32_t *count, int32_t *granted,
                                  int32_t *src, int32_t *dst, void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace vasc;
  int rc;
  if ((rc = check_pool(refs, pages, page_table, table_stride, max_pages, lengths, B))) return rc;
  VASC_REQUIRE(granted && src && dst, "granted, src and dst are required");
  VASC_REQUIRE(tokens > 0 && tokens < (int64_t(1) << 30), "tokens %lld outside [1, 2^30)", (long long)tokens);
  ReserveArgs p = {};
  p.refs = refs; p.pages = pages;
  p.table = page_table; p.stride = table_stride; p.max_pages = max_pages;
  p.lengths = lengths; p.count = count; p.tokens = tokens;
  p.B = static_cast<int32_t>(B);
  p.span = static_cast<int32_t>(reserve_span(tokens, max_pages));
  VASC_REQUIRE(B * p.span < (int64_t(1) << 31), "too many pages for one call");  // ranks are 32 bits
  p.chunks = static_cast<int32_t>(cdiv(pages, kChunk));
  p.granted = granted; p.src = src; p.dst = dst;
  int64_t at[5];
  const int64_t need = reserve_bytes(pages, B, p.span, at);
  VASC_REQUIRE(workspace && workspace_bytes >= need, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  VASC_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "the workspace must be 16-byte aligned");
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  p.free = reinterpret_cast<uint64_t *>(ws + at[0]);
  p.chunk = reinterpret_cast<int32_t *>(ws + at[1]);
  p.need = reinterpret_cast<int32_t *>(ws + at[2]);
  p.list = reinterpret_cast<int32_t *>(ws + at[3]);
  p.mark = reinterpret_cast<int32_t *>(ws + at[4]);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (pages <= kFewPages && B <= kFewSequences) {
    hipLaunchKernelGGL(reserve_few_kernel, dim3(1), dim3(1024), 0, s, p);
    return check_launch("vasc_pages_reserve");
  }
  const unsigned rows = static_cast<unsigned>(cdiv(B, 4));
  hipLaunchKernelGGL(reserve_count_kernel, dim3(static_cast<unsigned>(p.chunks) + rows), dim3(256), 0, s, p);
  if ((rc = check_launch("vasc_pages_reserve"))) return rc;
  hipLaunchKernelGGL(reserve_take_kernel, dim3(rows), dim3(256), 0, s, p);
  return check_launch("vasc_pages_reserve");
}
