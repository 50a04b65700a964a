/*
 * axkv.h — C ABI of the paged KV cache and its decode attention on B200.
 *
 * The cache lives in caller-owned device memory.  Per layer, K and V are
 * arrays of pages [n_pages][n_kv_heads][page_tokens][head_dim] (fp16, or fp32
 * with kv_fp32 = 1); token p of sequence s lives in page
 * block_table[s * max_blocks + p / page_tokens], slot p % page_tokens (the
 * block table is a caller-owned device array of int32).  A page id outside the
 * pool (-1: no page) is left out by an append, which reports it in the device
 * status word; decode and prefill attention read the pool's last page in its
 * place, so that row's result is undefined and nothing is read beyond.  Same
 * conventions as axq8.h: plain C, status codes, axq8_last_error().
 *
 * Reference interfaces replaced (paths inside the reference project):
 *   PagedKVCache::initialize / append   inference/cpp/runtime/paged_kv.hpp:18-41,
 *                                       paged_kv.cpp:44-120 (fp32 rows of
 *                                       page_size x hidden; here fp16 pages of
 *                                       16 tokens per KV head)
 *   append_row (KV append per token)    inference/cpp/runtime/streaming_executor.cpp:255-266
 *   mha_attention_incremental           inference/cpp/runtime/mha.cpp:227-285
 *   mha_attention (causal, prefill)     inference/cpp/runtime/mha.cpp:126-198
 */
#ifndef AXION_B200_AXKV_H
#define AXION_B200_AXKV_H

#include <stdint.h>

#include "axq8_status.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct axkv_cache {
    void* k_pages;               /* device, n_pages * n_kv_heads * page_tokens * head_dim elements */
    void* v_pages;               /* device, same shape */
    const int32_t* block_table;  /* device [sequences][max_blocks] page ids */
    int32_t n_pages;
    int32_t max_blocks;          /* pages per sequence (block table row length) */
    int32_t n_kv_heads;
    int32_t head_dim;            /* 32, 64 or 128 */
    int32_t page_tokens;         /* 16 */
    int32_t kv_fp32;             /* 0: fp16 pages, 1: fp32 pages */
} axkv_cache_t;

/* Bytes of one layer's K (or V) pages. */
int64_t axkv_pages_bytes(const axkv_cache_t* c);

/* Append n_rows token rows: row r of k_rows / v_rows (device fp32
 * [n_rows][n_kv_heads * head_dim], K after RoPE) is written, rounded to the
 * page type, at position row_pos[r] of sequence row_seq[r] (device int32
 * arrays).  PagedKVCache::append for one layer. */
int axkv_paged_append(const axkv_cache_t* c, const float* k_rows, const float* v_rows,
                      int32_t n_rows, const int32_t* row_seq, const int32_t* row_pos,
                      void* stream);

/* Workspace bytes axkv_paged_decode_attn needs for n_seq sequences of
 * n_heads query heads (split partials and per-(sequence, kv head) counters). */
int64_t axkv_decode_attn_workspace(const axkv_cache_t* c, int32_t n_seq, int32_t n_heads);

/* One query row per sequence against its cached tokens:
 * mha_attention_incremental (mha.cpp:227-285) — GQA kv head h / (n_heads /
 * n_kv_heads), scores scaled by 1/sqrt(head_dim) after the dot, max-subtracted
 * softmax.  q [n_seq][n_heads * head_dim] (device fp32, after RoPE); query s
 * sits at position q_pos[s] (device int32) and attends to tokens 0 ..
 * q_pos[s] of sequence s (append its own K/V first); out [n_seq][n_heads *
 * head_dim] device fp32.  The workspace (axkv_decode_attn_workspace bytes,
 * 16-byte aligned) must be zero before its first use; every call leaves it
 * zero again.  Calls sharing a workspace must not overlap on the GPU. */
int axkv_paged_decode_attn(const axkv_cache_t* c, const float* q, int32_t n_seq, int32_t n_heads,
                           const int32_t* q_pos, float* out, void* workspace,
                           int64_t workspace_bytes, void* stream);

/* Causal attention of a prompt chunk over the cache: mha_attention /
 * sdpa_causal (mha.cpp:126-198) for positions p0 .. p0 + T - 1 of n_seq
 * sequences whose K/V (those positions included) are already in the pages.
 * q rows [n_seq * T][n_heads * head_dim] (device fp32, after RoPE; row
 * s * T + t is sequence s at position p0 + t) with row pitch ldq floats;
 * out rows [n_seq * T][n_heads * head_dim] device fp32.  When xq is not null
 * the rows are instead quantized for the next Q8_0 product (the O
 * projection): xq [n_seq * T][n_heads * head_dim] int8 and transposed block
 * scales dxT [n_heads * head_dim / 32][Mp], Mp = n_seq * T rounded up to 4
 * (the layout of axq8_quantize_act_t); out is then unused.  fp16 pages, head
 * dim 64 or 128, n_heads / n_kv_heads <= 8 or a multiple of 8.  No workspace. */
int axkv_paged_prefill_attn(const axkv_cache_t* c, const float* q, int64_t ldq, int32_t n_seq,
                            int32_t T, int32_t p0, int32_t n_heads, float* out, int8_t* xq,
                            float* dxT, void* stream);

/* ---- the cache in 4 bits ---------------------------------------------------
 * The same paged cache with K and V held as 4-bit codes and 16-bit scales:
 * 0.5625 byte per value.  A block is 32 dims of one token of one KV head:
 *   lo = min(0, min x), hi = max(0, max x), R = hi - lo (fp32),
 *   d  = the smallest fp16 number of at most 7 significant bits (low 4
 *        mantissa bits clear) with 15 d >= R,
 *   n(x) = floor(x / d + 1/2), z = -n(lo), q = min(n(x) + z, 15),
 * and the block holds d * (q - z), which is always an fp16 number.  Values
 * beyond +-32768 are clamped and NaN is stored as 0; the device status word
 * then reads AXQ8_ERR_INVALID.
 *
 * A page holds, per KV head, 18 * head_dim bytes for 16 tokens: K codes
 * (8 head_dim), V codes (8 head_dim), K scales, V scales (head_dim each).
 * Scales: [token][block] 16 bits, bits 0x7ff0 the fp16 d, bits 0x000f z.
 * K codes: [token][t 4][block] 32-bit words, nibble e = dim 32 block + 8 t + e.
 * V codes: [group][g 8][t 4][tile] 32-bit words (tile = 16 dims, up to four to
 * a group); byte 2u + w is token 2t + u + 8w, low nibble dim 16 tile + g, high
 * nibble dim 16 tile + g + 8: the words are the operand registers of the
 * attention's matrix instructions. */
typedef struct axkv4_cache {
    void* pages;                 /* device, n_pages * n_kv_heads * 18 * head_dim bytes, 16-byte aligned */
    const int32_t* block_table;  /* device [n_seqs][max_blocks] page ids */
    int32_t n_seqs;
    int32_t max_blocks;          /* pages per sequence (block table row length) */
    int32_t n_pages;
    int32_t n_kv_heads;
    int32_t head_dim;            /* 32, 64 or 128 */
    int32_t page_tokens;         /* 16 */
} axkv4_cache_t;

/* Bytes of one layer's pages (K and V). */
int64_t axkv4_pages_bytes(const axkv4_cache_t* c);

/* Append rows as axkv_paged_append does, quantized to 4 bits.  Row r of k_rows /
 * v_rows (device fp32 [n_rows][n_kv_heads * head_dim], K after RoPE, row pitch
 * ld floats, 16-byte aligned, ld a multiple of 4) goes to position row_pos[r]
 * of sequence row_seq[r].  Rows outside the table, or whose page id is, are
 * left out and reported in the status word; a position named twice in one call
 * holds parts of either row. */
int axkv4_append(const axkv4_cache_t* c, const float* k_rows, const float* v_rows, int64_t ld,
                 int32_t n_rows, const int32_t* row_seq, const int32_t* row_pos, void* stream);

/* The values held at those positions, as fp32 rows (zeros, and the status
 * word, for positions outside the table). */
int axkv4_read(const axkv4_cache_t* c, float* k_rows, float* v_rows, int64_t ld, int32_t n_rows,
               const int32_t* row_seq, const int32_t* row_pos, void* stream);

/* Workspace bytes of axkv4_decode_attn for n_rows rows of n_heads query heads
 * (-1: unsupported). */
int64_t axkv4_decode_attn_workspace(const axkv4_cache_t* c, int32_t n_rows, int32_t n_heads);

/* Attention of one query row per sequence over the 4-bit cache, as
 * axkv_paged_decode_attn: row r of q (device fp32, row pitch ldq floats) sits
 * at position q_pos[r] of sequence q_seq[r] (q_seq null: sequence r) and
 * attends to tokens 0 .. q_pos[r]; out [n_rows][n_heads * head_dim] fp32.  A
 * row with q_pos < 0 attends to nothing and gives zeros (padding of a batch).
 * Pages whose id is outside the pool count as masked and are reported in the
 * status word, as are sequences and positions outside the table.  n_heads a
 * multiple of n_kv_heads, at most 16 times as many; at most 2^20 rows.  q and out
 * may be the same memory.  The workspace's contents need not be set; calls sharing
 * it must not overlap on the GPU, and come from one host thread at a time (a call
 * is two kernels).
 *
 * Accuracy: sums, weights and scores are held in fp32, q and the weights enter
 * the products as two fp16 parts (22 bits).  Relative to its norm a row is off by
 * 3e-7 to 8e-7 in this call and in short chunks, and by 1e-6 to 2e-6 in long ones
 * (8e-6 over long contexts of values of one sign, 2.1e-5 where all tokens are
 * alike), as measured.  A NaN or an infinity in q makes its heads' rows NaN; finite q should
 * stay below 2^100. */
int axkv4_decode_attn(const axkv4_cache_t* c, const float* q, int64_t ldq, int32_t n_rows,
                      int32_t n_heads, const int32_t* q_seq, const int32_t* q_pos, float* out,
                      void* workspace, int64_t workspace_bytes, void* stream);

/* Workspace bytes of axkv4_chunk_attn (same rules; -1: unsupported). */
int64_t axkv4_chunk_attn_workspace(const axkv4_cache_t* c, int32_t n_chunks, int32_t max_rows,
                                   int32_t n_heads);

/* Causal attention of n_chunks ragged chunks of rows over the 4-bit cache
 * (prompts, chunks after a past, draft tokens to check): rows q_start[i] ..
 * q_start[i + 1] - 1 of q are sequence q_seq[i] (q_seq null: sequence i) at
 * positions q_pos[i], q_pos[i] + 1, ...; each attends to tokens 0 .. its
 * position, their K and V already appended.  q_start (n_chunks + 1 device
 * int32) does not decrease; a chunk has at most max_rows rows (one that has
 * more, or rows outside q, is left out and reported; with max_rows 0 the call
 * does nothing).  At most 65535 chunks of 2^24 rows.  q and out have n_rows rows
 * and may be the same memory; rows of no chunk are left as they are in out.
 * Rows at negative positions give zeros; reports as in axkv4_decode_attn.
 *
 * One kernel takes the whole call, by n_chunks and max_rows: the one for long
 * chunks does not share a chunk's context among SMs.  Single rows over long
 * contexts belong in an axkv4_decode_attn call of their own rather than beside a
 * long prompt (15 of them over 16,384 tokens with 2048 prompt rows: 816 us in one
 * call, 142 + 100 us in two), and max_rows should be near the longest chunk. */
int axkv4_chunk_attn(const axkv4_cache_t* c, const float* q, int64_t ldq, int32_t n_rows,
                     int32_t n_chunks, int32_t max_rows, int32_t n_heads, const int32_t* q_seq,
                     const int32_t* q_start, const int32_t* q_pos, float* out, void* workspace,
                     int64_t workspace_bytes, void* stream);

/* ---- pages of a cache -------------------------------------------------------
 * Sequences that share pages.  The state is device memory of the caller: the
 * block table, -1 where a row holds no page (a row's pages come first), and
 * for every page the number of table entries that name it; a page of count 0
 * is free.  A page is moved in every pool (the K and V pages of each layer of
 * an axkv_cache, the pages of each layer of an axkv4_cache).  New pages are the
 * lowest-numbered free ones, in the order of the request, so results do not
 * depend on timing.  A reserve or fork with an invalid entry, or with more
 * pages to allocate than are free, changes nothing and is reported in the
 * status word (AXQ8_ERR_INVALID, AXQ8_ERR_ALLOC); a free or copy leaves
 * invalid entries out and reports them.  Calls on one state must not overlap
 * on the GPU, and come from one host thread at a time: a reserve, fork or compact
 * is two kernels, between which no other call on the state may be launched. */
typedef struct axkv_pages {
    int32_t* block_table;        /* device [n_seqs][max_blocks] */
    int32_t* ref_count;          /* device [n_pages] */
    void* const* pools;          /* device array of n_pools base addresses, 16-byte aligned */
    int64_t page_bytes;          /* bytes of a page in one pool, a multiple of 16 */
    int32_t n_pools;             /* may be 0: bookkeeping only */
    int32_t n_seqs;
    int32_t max_blocks;
    int32_t n_pages;             /* at most 2,000,000 */
} axkv_pages_t;

/* Workspace bytes of a reserve, fork or compact call of up to n entries; its
 * contents need not be set.  Calls sharing a workspace must not overlap. */
int64_t axkv_pages_workspace(const axkv_pages_t* p, int32_t n);

/* Sequence seqs[i] gets pages for tokens[i] tokens (device int32 arrays; pages
 * that it holds are kept).  A sequence is named at most once in a call. */
int axkv_pages_reserve(const axkv_pages_t* p, const int32_t* seqs, const int32_t* tokens, int32_t n,
                       void* workspace, int64_t workspace_bytes, void* stream);

/* Sequence children[i], which holds no page, becomes a copy of the first
 * tokens[i] tokens of parents[i]: full pages are shared, a page that tokens[i]
 * fills in part is copied to a new one.  Shared pages are full, so appending
 * behind those tokens to either sequence leaves the other as it is.  It does not
 * where a sequence is taken back (rejected draft tokens) to before the last full
 * page that it shares and written again from there: the pages are not copied on
 * a write.  Fork it at the shorter length instead, and free the old one.  A child
 * is named once in a call and is no parent in it. */
int axkv_pages_fork(const axkv_pages_t* p, const int32_t* parents, const int32_t* children,
                    const int32_t* tokens, int32_t n, void* workspace, int64_t workspace_bytes,
                    void* stream);

/* Sequence seqs[i] gives its pages up (naming it twice is naming it once). */
int axkv_pages_free(const axkv_pages_t* p, const int32_t* seqs, int32_t n, void* stream);

/* Live pages to the front: with n_live pages in use, the k-th used page of
 * those from n_live on moves to the k-th free page below n_live, in every pool
 * and in the table.  *n_live (device int32) receives the number; pages from it
 * on are free. */
int axkv_pages_compact(const axkv_pages_t* p, int32_t* n_live, void* workspace,
                       int64_t workspace_bytes, void* stream);

/* Page src[i] copied to page dst[i] in every pool (device int32 arrays).  No
 * destination is named twice or is a source; pages outside the pool are left
 * out and reported. */
int axkv_pages_copy(const axkv_pages_t* p, const int32_t* src, const int32_t* dst, int32_t n,
                    void* stream);

#ifdef __cplusplus
}
#endif
#endif /* AXION_B200_AXKV_H */
