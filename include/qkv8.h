/*
 * qkv8.h — C ABI of the 8-bit paged KV cache and its decode attention on B200
 * (sm_100a).  Part of libqcache.so; includes qcache.h for the status codes,
 * qc_stream and QC_PAGE.
 *
 * The bf16 cache of qcache.h costs 4096 bytes per position and layer, which is
 * most of what a decode step reads.  This cache holds the same rows in 8 bits,
 * half the bytes, for any number of KV heads of 64, 128 or 256 dims.  Like
 * qc_attn_decode_noalloc the calls work on buffers of the caller: they allocate
 * nothing, keep nothing between calls and can be captured into CUDA graphs.
 *
 * Format.  A page holds QC_PAGE tokens of every KV head of one layer, in blocks
 * of QC_KV8_BLOCK = 16 tokens of one head.  A block has one scale for its K and
 * one for its V values, a power of two (the shared exponent of the BFP8_B
 * weights, qbfp8.h, over 16 tokens x head_dim): value = code * scale, code a
 * whole number in [-127, 127].  A page is qc_kv8_page_bytes bytes, page p of a
 * pool starts at p times that; inside a page the bytes stand in the order in
 * which the attention kernel's lanes read them, so a pool is written and read
 * through the calls below.  Page ids are the caller's, for instance those that
 * qc_seq_pages gives for a sequence of a context; the context knows nothing of the
 * pool, so where it gives tokens another page (a shared page's private copy, a
 * restored tail) the pool's bytes are the caller's to copy or to write again.
 *
 * Quantisation (qc_kv8_write).  A block's scale is the smallest power of two
 * 2^e, -126 <= e <= 120, for which every value fits (|x| <= 127 * 2^e), and
 * code = round-to-nearest-even(x / 2^e).  Infinities and values beyond
 * 127 * 2^120 count as that value, NaN as 0.  When tokens are appended to a
 * block that holds older ones and need a larger scale, the older codes become
 * round-to-nearest-even(code * old scale / new scale); a block's scale never
 * shrinks while it keeps a token.  The result depends only on which rows each
 * call wrote.
 *
 * All positions are int32 (arrays 4-byte aligned), all offsets 64-bit.  A page id
 * outside the pool, a position outside the page table's row or a row index outside
 * the input is skipped and recorded as QC_ERR_BOUNDS, which qc_kv8_check reports.
 * Calls that touch the same pages, and calls that share a workspace, must not
 * overlap on the GPU: enqueue them on one stream or order the streams (two
 * graphs that may run at once need a workspace each).
 */
#ifndef QKV8_H
#define QKV8_H

#include "qcache.h"

#ifdef __cplusplus
extern "C" {
#endif

#define QC_KV8_BLOCK     16      /* tokens that share a scale */
#define QC_KV8_MAX_SEQS  1024    /* sequences per call */
#define QC_KV8_MAX_HEADS 256     /* KV heads */
#define QC_KV8_MAX_GROUP 8       /* query heads per KV head */

/* Describes a pool; host memory, read before a call returns. */
typedef struct qc_kv8_cache {
  uint8_t* pool;        /* device, n_pages * qc_kv8_page_bytes, 16-byte aligned */
  int32_t n_pages;
  int32_t n_kv_heads;   /* 1 .. QC_KV8_MAX_HEADS */
  int32_t head_dim;     /* 64, 128 or 256 */
  int32_t reserved;     /* 0 */
} qc_kv8_cache;

/* Bytes of one page; 0 for a shape that is not supported. */
int64_t qc_kv8_page_bytes(int32_t n_kv_heads, int32_t head_dim);

/* Appends rows to n sequences (n <= QC_KV8_MAX_SEQS).  Sequence i gets the rows
 * row_start[i] .. row_start[i+1]-1 (may be none) of k and v at positions
 * pos[i], pos[i]+1, ...; afterwards its tokens from there on are undefined, as
 * nothing is kept behind the last row.  row_start_dev NULL: row i goes to
 * sequence i (n_rows == n), a decode step.
 *   page_table_dev  [n][pt_stride] int32: page of positions 64j .. 64j+63
 *   pos_dev         [n] int32; row_start_dev [n+1] int32, ascending
 *   k_dev, v_dev    bf16; row r's heads [n_kv_heads][head_dim] at r * k_ld
 *                   (v_ld) elements, so both may point into projection rows;
 *                   16-byte aligned, k_ld and v_ld multiples of 8, at least
 *                   n_kv_heads * head_dim
 * A sequence may appear once per call, and no page in two of its rows. */
int qc_kv8_write(const qc_kv8_cache* cache, const int32_t* page_table_dev, int32_t pt_stride,
                 const int32_t* pos_dev, const int32_t* row_start_dev, int32_t n, int32_t n_rows,
                 const uint16_t* k_dev, int64_t k_ld, const uint16_t* v_dev, int64_t v_ld,
                 qc_stream stream);

/* The reverse: the cached values (code * scale, exact in bf16) of the same
 * positions into the rows of k_dev and v_dev.  Arguments as qc_kv8_write. */
int qc_kv8_read(const qc_kv8_cache* cache, const int32_t* page_table_dev, int32_t pt_stride,
                const int32_t* pos_dev, const int32_t* row_start_dev, int32_t n, int32_t n_rows,
                uint16_t* k_dev, int64_t k_ld, uint16_t* v_dev, int64_t v_ld, qc_stream stream);

/* Decode attention: one query token per sequence over its cached tokens,
 *   out[i][h] = sum_j softmax_j(scale * q[i][h] . K[j]) V[j]  [* sigmoid(gate)]
 * over positions j < len[i] of KV head h / (n_head / n_kv_heads).
 *   len_dev    [n] int32, at most 64 * pt_stride; 0 gives a row of zeros
 *   q_dev      bf16, head h of sequence i at i * q_ld + h * q_head elements
 *              (already normalised and rotated, qrope.h); 16-byte aligned,
 *              strides multiples of 8
 *   gate_dev   NULL, or the gate's logits with q's strides (the layer's output
 *              gate, src/engine.cpp:3557-3561: [16][q | gate] rows pass q_dev
 *              and q_dev + head_dim when q was rotated in place)
 *   out_dev    bf16 [n_head][head_dim] per sequence at i * out_ld; 16-byte
 *              aligned, out_ld a multiple of 8
 * n_head is a multiple of n_kv_heads, at most QC_KV8_MAX_GROUP times it.
 * out must not overlap q, the gate or the pool.
 * workspace: at least qc_kv8_attn_workspace_bytes bytes of device memory, 16-
 * byte aligned, for this call alone while it runs; its contents do not matter.
 * Products of queries and codes are exact (of a query value below 2^-30 of its head's
 * largest, what is below 2^-38 of that is rounded) and sums are kept in f32; the softmax
 * weights, with V's scales, enter the second product with 22 bits (one below 2^-10 of
 * the largest with an error of 2^-32 of that).  The result rounds to bf16 once.  It
 * depends on the shapes and values alone: the same bits on every call.  A NaN or
 * infinity in q makes its head's row NaN, and scores beyond f32 may.  Scores up to
 * 2^100 are formed without leaving f32 however far apart q, K and the scale are. */
int64_t qc_kv8_attn_workspace_bytes(const qc_kv8_cache* cache, int32_t n, int32_t n_head);
int qc_kv8_attn_decode(const qc_kv8_cache* cache, const int32_t* page_table_dev,
                       int32_t pt_stride, const int32_t* len_dev, int32_t n, int32_t n_head,
                       const uint16_t* q_dev, int64_t q_ld, int64_t q_head,
                       const uint16_t* gate_dev, float scale, uint16_t* out_dev, int64_t out_ld,
                       void* workspace, int64_t workspace_bytes, qc_stream stream);

/* Synchronises `stream`, no other one, and returns the first error that the
 * kernels of this header have recorded on the current device since the last call
 * (QC_ERR_BOUNDS, QC_ERR_TIMEOUT), clearing it.  The device has one such word:
 * whoever checks gets what any caller's kernels recorded, each error once.  May be
 * called from several threads; not while `stream` is being captured.  The first
 * call loads a kernel, for which the driver may wait for other streams. */
int qc_kv8_check(qc_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* QKV8_H */
