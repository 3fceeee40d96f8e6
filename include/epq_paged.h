/* epq_paged.h -- several sequences decoding together (libepq.so): rotary positions,
 * a paged key-value cache that may hold 8-bit values, and the attention of one new
 * token a sequence over it.
 *
 * Not part of the reference's op interface (include/epq.h): the reference leaves
 * attention and its cache to the Hugging Face model around its PackedLinear modules
 * (epure/runtime.py:214-305 swaps only the linears).  Conventions are those of
 * epq.h: plain pointers, epq_dtype codes, a cudaStream_t passed as void*, EPQ_OK or
 * a negative status with epq_last_error().  Positions, lengths and page tables are
 * read on the device, so a captured step replays at any position.  What is wrong in
 * them is reported by epq_device_error: bit 4 for a position, length or sequence
 * outside the cache or the rotary table, bit 5 for a page outside the pool.
 */
#ifndef EPQ_PAGED_H
#define EPQ_PAGED_H

#include <stdint.h>

#include "epq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A strided view [rows, heads, head_dim] (element strides; the values of a head are
 * contiguous), e.g. the q part of a fused projection's output. */
typedef struct epq_heads {
    void* data;
    int64_t stride_row;
    int64_t stride_head;
    int32_t heads;
    int32_t reserved0;
} epq_heads;

/* Rotary positions.  For count (1 or 2) tensors x[i], y[i] [m, heads_i, head_dim] and
 * every row r at p = pos[r], the pairs (a, b) = (j, j + rotary_dim / 2), or
 * (2j, 2j + 1) where interleaved != 0, with c = cos_tab[p, j], s = sin_tab[p, j]
 * (float32 [max_len, rotary_dim / 2]):
 *     y_a = x_a c - x_b s,   y_b = x_b c + x_a s,
 * computed in float32 and rounded once; values past rotary_dim are copied.
 * inverse != 0 turns by -s: the gradient of the call with respect to x.  y[i] may be
 * x[i] (in place, with its strides), and may not overlap it otherwise; no two heads of
 * y[i] may overlap (EPQ_ESHAPE).  A position outside
 * [0, max_len) writes zeros.  rotary_dim even, 2..head_dim; head_dim <= 1024. */
int epq_rope(const epq_heads* x, const epq_heads* y, int32_t count, const int64_t* pos, int64_t m,
             int32_t head_dim, int32_t rotary_dim, const float* cos_tab, const float* sin_tab, int64_t max_len,
             int32_t interleaved, int32_t inverse, int32_t dtype, void* stream);

/* How a cache holds its values: in the activations' type, or as one 8-bit code a
 * value with one float32 scale a token and head (value = code * scale):
 *   INT8  scale = max|x| * (1 / 127), code = x * (127 / max|x|) rounded to even
 *   FP8   scale = max|x| * (1 / 448), code = x * (448 / max|x|) rounded to e4m3
 * (every operation in float32, rounded by itself).
 * A row of zeros has scale 0; a row that holds an infinity or NaN reads back as NaN. */
enum epq_cache_format { EPQ_CACHE_SAME = 0, EPQ_CACHE_INT8 = 1, EPQ_CACHE_FP8 = 2 };

/* The paged cache of one layer.  Token t of sequence s lives in slot t % page_size of
 * page table[s * table_stride + t / page_size]; k and v hold
 * [pages][kv_heads][page_size][head_dim] values with page_stride elements between
 * pages (the rest contiguous), k_scale and v_scale [pages][kv_heads][page_size] with
 * scale_stride between pages.  head_dim is a multiple of 16 up to 256; k, v and the
 * page stride are 16-byte aligned. */
typedef struct epq_pages {
    void* k;
    void* v;
    float* k_scale;            /* NULL for EPQ_CACHE_SAME */
    float* v_scale;
    const int32_t* table;
    int64_t page_stride;
    int64_t scale_stride;
    int64_t table_stride;
    int64_t pages;
    int32_t seqs;              /* rows of the table */
    int32_t max_pages;         /* its columns */
    int32_t page_size;
    int32_t kv_heads;
    int32_t head_dim;
    int32_t format;            /* enum epq_cache_format */
} epq_pages;

/* Writes m rows of k and v [m, kv_heads, head_dim], row r as token pos[r] of sequence
 * seq[r].  qk_norm != 0 first normalises every head of q and k (RMSNorm, weight 1);
 * with cos_tab / sin_tab (NULL: none) q and k are then rotated as by epq_rope.  Both
 * results are rounded to dtype, as the tensors of a model are, before k is quantised.
 * q [m, heads, head_dim] may be NULL; q_out receives it (q_out may be q, as in epq_rope).  A row with
 * a negative position is padding: nothing is written to the cache, zeros to q_out.  No
 * two rows may name the same token. */
int epq_paged_write(const epq_pages* pages, const epq_heads* q, const epq_heads* q_out, const epq_heads* k,
                    const epq_heads* v, const int32_t* seq, const int64_t* pos, int64_t m, const float* cos_tab,
                    const float* sin_tab, int64_t max_len, int32_t rotary_dim, int32_t interleaved,
                    int32_t qk_norm, float eps, int32_t dtype, void* stream);

/* Reads m cached rows back: k_out, v_out [m, kv_heads, head_dim] (contiguous, 16-byte
 * aligned) = code * scale, rounded once to dtype (an EPQ_CACHE_SAME cache holds dtype).
 * Rows with a negative position are zero. */
int epq_paged_read(const epq_pages* pages, const int32_t* seq, const int64_t* pos, int64_t m, void* k_out,
                   void* v_out, int32_t dtype, void* stream);

/* One new token a sequence: for row b, sequence s = seq ? seq[b] : b, length
 * n = lengths[b] and every head h,
 *     out[b, h] = sum_t softmax_t(scale * q[b, h] . K[s, t, g]) V[s, t, g],
 * g = h / (heads / kv_heads), over the tokens t < n (the last `window` of them where
 * window > 0); lse[b, h] (may be NULL) = log sum_t exp(scale * q . K).  A length of 0
 * gives zeros and -inf, and so does a row whose every score is -inf.  q
 * [batch, heads, head_dim] is f16 or bf16 (4-byte aligned, even strides), and so is an
 * EPQ_CACHE_SAME cache; out [batch, heads, head_dim] is contiguous and
 * 16-byte aligned.  lengths and seq must not change while the call runs: its CTAs
 * read them one by one, and share the work by them.  The workspace
 * (256-byte aligned) has to be zeroed once before its first use and is left ready for
 * the next call; calls that share one must not overlap.
 * units = kv_heads * ceil(heads / kv_heads / 16): batch * units <= 65536, and with
 * blocks = batch * (max_pages * page_size / 16 + 13), blocks < 2^31 and blocks * units < 2^37. */
int64_t epq_paged_attend_workspace_bytes(const epq_pages* pages, int64_t batch, int32_t heads);
int epq_paged_attend(const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                     int64_t batch, float scale, int64_t window, void* out, float* lse, int32_t dtype,
                     void* workspace, int64_t workspace_bytes, void* stream);

/* epq_paged_attend where rows share their first tokens, which are read once for all of them:
 * rows starts[g] .. starts[g + 1) - 1 (int32, groups + 1 of them, ascending) have the same
 * prefix[g] first tokens: their sequences' tables name pages that hold the same values there,
 * and those of one of the rows are read for all.  A row whose length is below prefix[g] attends over its own length.  The rows may be sequences
 * behind a common prompt or several new tokens of one sequence (rows of one seq with growing
 * lengths).  Rows of no group share nothing; where starts are not ascending or outside the batch,
 * or a prefix is not in 0..max_pages * page_size, that is reported (bit 4) and none does.  Which
 * rows are taken together, and whether any are, follows from sizes and lengths alone: groups for which reading row
 * by row is reckoned to be faster are read that way, unless `always` is not 0.  With `always` too nothing is shared
 * in pages whose size is no multiple of 8, by 8-bit heads above 128, with more than 128 query heads a key head, and where q
 * is not 16-byte aligned with positive strides of a multiple of 8 values.  Rows are taken together in tiles of a group's
 * consecutive rows, up to 256 query rows each (128 for heads above 128), as far as the shortest of a tile's lengths
 * (empty rows aside): one row of 5 tokens among 64 that share 8192 leaves all of them row by row (67 us, with it 211).
 * batch <= 65536; a workspace of its own bytes, with epq_paged_attend's rules.
 * epq_device_error bit 1: a wait of the kernel's own gave up. */
int64_t epq_paged_attend_shared_workspace_bytes(const epq_pages* pages, int64_t batch, int32_t heads, int64_t groups,
                                                int32_t always);
int epq_paged_attend_shared(const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                            int64_t batch, const int32_t* starts, const int64_t* prefix, int64_t groups, int32_t always,
                            float scale, void* out, float* lse, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream);

/* The bounds of a page's keys: bounds [pages][kv_heads][2][head_dim] hold, of every value of a
 * head, the least and the largest over the page's tokens, in the cache's own 16-bit type or,
 * for 8-bit caches (code * scale in float32), rounded to bf16; infinities are held as the
 * largest finite value and NaN stays.  bounds_stride values lie between pages (a multiple of 8,
 * 16-byte aligned).  For row b, tokens first[b] (NULL: 0) to lengths[b] - 1 of sequence
 * s = seq ? seq[b] : b are new: every page that holds one of them gets the bounds of all its
 * tokens below lengths[b].  Nothing is done where lengths[b] <= first[b].  Two rows with a page
 * in common must agree about its tokens. */
int epq_paged_bounds(const epq_pages* pages, void* bounds, int64_t bounds_stride, int32_t dtype, const int32_t* seq,
                     const int64_t* first, const int64_t* lengths, int64_t batch, void* stream);

/* The blocks (pages) to attend over, by a score that bounds q . K[t] for a block's tokens:
 *     score(j) = max over the query heads h of key head g of
 *                sum_d max(q[b, h, d] lo_j[d], q[b, h, d] hi_j[d])
 * in float32, products first, then neighbouring dims' sums, then neighbours of those (head_dim
 * padded with zeros to a power of two; lo <= hi, as epq_paged_bounds leaves them).  No q . K[t] passes it, up to float32's
 * rounding of the sums, over a 16-bit cache with finite keys; the bounds of an 8-bit one are rounded to the nearest bf16, by up
 * to 2^-8 of their value, and infinite keys are held as finite ones, so there a product can.  Of the n = ceil(lengths[b] / page_size) blocks of a row
 * chosen[b, g, 0..count) receives, in ascending order, the first `sinks`, the last `recent` and
 * those of the others with the largest scores (NaN first), the lowest of equal ones; all of them
 * where n <= count, and -1 behind the last.  A block whose page is outside the pool comes last.
 * The workspace is epq_paged_attend's in its rules, and the two may share one on a stream.
 * batch * kv_heads <= 65536, max_pages < 2^21. */
int64_t epq_paged_select_workspace_bytes(const epq_pages* pages, int64_t batch);
int epq_paged_select(const epq_pages* pages, const void* bounds, int64_t bounds_stride, int32_t bounds_dtype,
                     const epq_heads* q, int32_t dtype, const int32_t* seq, const int64_t* lengths, int64_t batch,
                     int32_t count, int32_t sinks, int32_t recent, int32_t* chosen, void* workspace, int64_t workspace_bytes,
                     void* stream);

/* epq_paged_attend over the tokens of listed blocks: blocks [batch, kv_heads, count] names pages
 * of the row's sequence for each key head (token t is in block t / page_size), each at most
 * once, -1 for none; of a list the first min(count, ceil(lengths[b] / page_size)) entries are
 * looked at.  Tokens at lengths[b] and behind are not attended over.  A block at or past
 * max_pages is skipped and reported (bit 4).  No window. */
int epq_paged_attend_blocks(const epq_pages* pages, const epq_heads* q, const int32_t* seq, const int64_t* lengths,
                            int64_t batch, const int32_t* blocks, int32_t count, float scale, void* out, float* lse,
                            int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* EPQ_PAGED_H */
