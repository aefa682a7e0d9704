/*
 * Streaming ops of libvasc_hip.so: the operators of a global layer whose
 * frames (or single query tokens) arrive one after another. Keys and values
 * stay in an 8-bit block cache; queries attend to cache blocks that a cheap
 * score chooses. They have no counterpart in the reference, which sees a
 * whole clip at once; vasc_amd/streaming.py calls them.
 *
 * Conventions as in vasc_hip.h: raw device pointers, int64 sizes and element
 * strides, the HIP stream as void*, an int status (0 ok) with the message in
 * vasc_last_error(), no allocation. dtype: 0 bfloat16, 1 float16, 2 float32.
 *
 * The block cache. Pages of 64 tokens; with pages P, key heads H, head
 * dimension D (64 or 128), all contiguous:
 *   kc   uint8    [P, H, 64, D]  e4m3 codes of the keys
 *   vc   uint8    [P, H, D, 64]  e4m3 codes of the values, transposed
 *   ks   uint8    [P, H, 64]     exponents of the key rows, 2^(byte - 127)
 *   vs   uint8    [P, H, 64]     exponents of the value rows
 *   mean bfloat16 [P, H, D]      mean of the page's keys
 * vc's last dimension and vs hold token t of the page at
 *   ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3),
 * ks at (t & 15) * 4 + (t >> 4): the orders in which the lanes of a matrix
 * product consume them. A row's exponent is the smallest e in [-60, 60] with
 * max|x| <= 448 * 2^e: every value is exact in bfloat16, values past 448 * 2^60
 * saturate and those under 2^-70 are zero. A token whose key or value row of a
 * head holds a value that is not finite has key exponent byte 255 there and
 * zero codes: both rows read back as NaN. A cache starts as zeros.
 *
 * Sequence b's page j is page_table[b * table_stride + j], j < max_pages
 * (int32). Entries outside [0, P) are no page: nothing is written there, and
 * their tokens are never seen. Lengths past max_pages * 64 are cut to it (the
 * positions of causal rows are not).
 */
#ifndef VASC_STREAM_H
#define VASC_STREAM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rotary positions with several axes over q and (or NULL) k in one launch.
 * q [B,Hq,T,D], k [B,Hk,T,D] strided (unit stride over D), qo and ko alike,
 * of one dtype. Axis a (of `axes`, 1..4) owns the next sections[a] features
 * (a host array of even numbers whose sum is at most D); its pair
 * (j, j + sections[a]/2) turns by pos[b,t,a] * inv_freq[j of the axis]:
 *   lo' = lo cos - hi sin,  hi' = hi cos + lo sin  (inverse != 0: -angle).
 * Features past the sections are copied. pos: int32, element (b,t,a) at
 * pos[b*pos_sb + t*pos_st + a]; inv_freq: float64 on the device, the axes'
 * sections[a]/2 values one after another. Angles are float64.
 */
int vasc_rotary_axes(const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st, void *qo, int64_t qo_sb, int64_t qo_sh,
                     int64_t qo_st, int64_t Hq, const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st, void *ko,
                     int64_t ko_sb, int64_t ko_sh, int64_t ko_st, int64_t Hk, int64_t B, int64_t T, int64_t D,
                     const int32_t *pos, int64_t pos_sb, int64_t pos_st, int32_t axes, const int64_t *sections,
                     const double *inv_freq, int32_t dtype, int32_t inverse, void *stream);

/*
 * Writes count[b] (NULL: T) tokens of k, v [B,H,T,D] (strided) at positions
 * start[b].. of sequence b, and renews the key mean of every page touched:
 * the mean of the page's tokens up to the last one written, from the 8-bit
 * values, as bf16(f32(float64 sum / tokens)). Tokens before them in the page
 * must have been written. A negative start writes nothing. No page may be
 * written twice in one call.
 */
int vasc_cache_write(const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st, const void *v, int64_t v_sb, int64_t v_sh,
                     int64_t v_st, int64_t B, int64_t H, int64_t T, int64_t D, int32_t dtype,
                     const int32_t *page_table, int64_t table_stride, int64_t max_pages, const int32_t *start,
                     const int32_t *count, uint8_t *kc, uint8_t *vc, uint8_t *ks, uint8_t *vs, uint16_t *mean,
                     int64_t pages, void *stream);

/*
 * Reads tokens start[b].. of sequence b back: ko, vo [B,H,T,D] contiguous of
 * `dtype`; rows past count[b] (NULL: T) and rows without a page are zero.
 */
int vasc_cache_read(const uint8_t *kc, const uint8_t *vc, const uint8_t *ks, const uint8_t *vs, int64_t pages,
                    const int32_t *page_table, int64_t table_stride, int64_t max_pages, const int32_t *start,
                    const int32_t *count, int64_t B, int64_t H, int64_t T, int64_t D, int32_t dtype, void *ko, void *vo,
                    void *stream);

/*
 * Block choice. A unit is block_q consecutive query tokens (block_q * G at
 * most 128) of the G = Hq / H query heads of one key head; U = ceil(T /
 * block_q). q [B,Hq,T,D] (strided, bfloat16 or float16); q_count[b] (NULL: T)
 * queries of sequence b count, the last ones of its `lengths[b]` tokens where
 * causal. score [B,H,U,max_pages] float32 (workspace or output): of each page
 * j that the unit sees (causal: up to its last row's own position)
 *   f32(sum over d, float64, of bf16(f32(mean of the unit's q rows)) * mean[j]),
 * NaN as -inf; -inf elsewhere. Listed, ascending, are the first `sink` pages,
 * the last `recent` (>= 1; causal: counted back from the first row's own page,
 * with every page after it), and the `keep` highest scores of the others,
 * equal scores in page order. index [B,H,U,width] int32, -1 behind the list;
 * count [B,H,U]; width = min(max_pages, sink + keep + recent + (causal ?
 * (block_q + 62) / 64 : 0)).
 */
int vasc_cache_select(const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st, int64_t B, int64_t Hq, int64_t H,
                      int64_t T, int64_t D, int32_t dtype, const uint16_t *mean, int64_t pages,
                      const int32_t *page_table, int64_t table_stride, int64_t max_pages, const int32_t *lengths,
                      const int32_t *q_count, int64_t block_q, int64_t sink, int64_t recent, int64_t keep,
                      int32_t causal, float *score, int32_t *index, int64_t width, int32_t *count, void *stream);

/* Bytes of workspace that vasc_cache_attn needs for these sizes (0: none); -1 for sizes that it refuses. */
int64_t vasc_cache_attn_workspace_size(int64_t B, int64_t Hq, int64_t H, int64_t T, int64_t D, int64_t block_q,
                                       int64_t max_pages, int64_t width);

/*
 * Attention of q over the cache: o = softmax(scale * q k^T) v over the keys
 * of the listed pages (index NULL: of all pages) below lengths[b] (causal: at
 * or before the row's own position lengths[b] - q_count[b] + t). Rows that
 * see no key and rows past q_count[b] are zero; a row that sees a NaN token,
 * or whose query is not finite, is NaN. index [B,H,U,width], count
 * [B,H,U] as vasc_cache_select writes them: ascending logical pages; entries
 * that are not above the one before them in the list (skipped or not),
 * negative or not below max_pages are skipped. block_q as there (index NULL: any block_q with block_q * G <= 128).
 * q, o [B,Hq,T,D] strided, bfloat16 or float16. scale: 0, or of magnitude
 * 1e-30 to 1e30. Logits of finite values that pass float32 are not held.
 */
int vasc_cache_attn(const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st, void *o, int64_t o_sb, int64_t o_sh,
                    int64_t o_st, int64_t B, int64_t Hq, int64_t H, int64_t T, int64_t D, int32_t dtype,
                    const uint8_t *kc, const uint8_t *vc, const uint8_t *ks, const uint8_t *vs, int64_t pages,
                    const int32_t *page_table, int64_t table_stride, int64_t max_pages, const int32_t *lengths,
                    const int32_t *q_count, int64_t block_q, const int32_t *index, int64_t width, const int32_t *count,
                    int32_t causal, float scale, void *workspace, int64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* VASC_STREAM_H */
