/*
 * qrope.h — C ABI of the rotary position embedding on B200 (sm_100a), with the
 * optional per-head RMSNorm in front of it.  Part of libqcache.so; includes
 * qcache.h for the status codes and qc_stream.
 *
 * qc_attn_decode and qc_attn_prefill rotate inside their kernels, for the one
 * shape of their model (64 of 256 dims, half layout, base 1e7, the reference's
 * f32 angles).  This is the same step (src/engine.cpp:3497-3519, 2422-2432) as
 * a call of its own, for callers that keep their own cache (qkv8.h) or need
 * another layout, head size or context scaling.
 *
 * For every row r, head h and pair i < rot_dim / 2, with y the row's head
 * (normalised first, y * rsqrt(mean(y^2) + eps) * norm_w, when norm_w is given)
 * and a = pos[r] * inv_freq[i]:
 *   out[p] = mscale * (y[p] cos a - y[q] sin a)
 *   out[q] = mscale * (y[q] cos a + y[p] sin a)
 * (p, q) = (i, i + rot_dim/2) in the half layout, (2i, 2i + 1) in the
 * interleaved one.  Dims from rot_dim on are copied (normalised if asked).
 * Angles are formed and reduced in 64 bits for any int32 position, also a
 * negative one; the arithmetic is f32 and rounds to bf16 once, to nearest even.
 * NaN and infinity stay within their own head.  Without the norm they reach the
 * pair they stand in.  Through the norm a NaN reaches the whole head; an infinity
 * makes the mean infinite, so that it and its pair become NaN and all other dims 0
 * (of either sign), as the formula has it.  Finite values are normalised right
 * however large or small they are.
 */
#ifndef QROPE_H
#define QROPE_H

#include "qcache.h"

#ifdef __cplusplus
extern "C" {
#endif

#define QC_ROPE_MAX_DIM   256     /* largest head_dim and rot_dim */
#define QC_ROPE_MAX_PARTS 4
#define QC_ROPE_MAX_HEADS 16384 /* heads of a part */

/* pair layouts */
#define QC_ROPE_HALF        0
#define QC_ROPE_INTERLEAVED 1

/* frequency scaling for contexts longer than the trained one; f is the factor
 * (> 0) and w_i = base^(-2i / rot_dim):
 *   PLAIN   w_i
 *   LINEAR  w_i / f                         (position interpolation)
 *   NTK     w_i with base * f^(rot_dim / (rot_dim - 2)); rot_dim > 2
 *   YARN    w_i / f * g + w_i * (1 - g), g = clamp((i - low) / max(high - low,
 *           0.001), 0, 1), low = floor(c(beta_fast)) >= 0, high =
 *           ceil(c(beta_slow)) <= rot_dim - 1, c(b) = rot_dim * ln(orig_ctx /
 *           (2 pi b)) / (2 ln base); mscale = 0.1 ln f + 1 (1 for f <= 1).
 *           The method is Peng et al., "YaRN: Efficient Context Window
 *           Extension of Large Language Models" (2023). */
#define QC_ROPE_PLAIN  0
#define QC_ROPE_LINEAR 1
#define QC_ROPE_NTK    2
#define QC_ROPE_YARN   3

typedef struct qc_rope_config {
  int32_t rot_dim;    /* rotated dims of a head: even, 2 .. QC_ROPE_MAX_DIM */
  int32_t layout;     /* QC_ROPE_HALF or QC_ROPE_INTERLEAVED */
  int32_t scaling;    /* QC_ROPE_PLAIN .. QC_ROPE_YARN */
  int32_t orig_ctx;   /* trained context length (YARN; ignored otherwise) */
  double base;        /* > 1 */
  double factor;      /* > 0 (ignored by PLAIN) */
  double beta_fast;   /* YARN; 0 for the method's 32 */
  double beta_slow;   /* YARN; 0 for the method's 1 */
  double mscale;      /* factor on the rotated dims; 0 for the scaling's own */
} qc_rope_config;

/* Frequencies worked out by qc_rope_init.  Plain data: copy it, keep it on the
 * stack; no call keeps a pointer to it. */
typedef struct qc_rope {
  int32_t rot_dim;
  int32_t layout;
  double mscale;
  double inv_freq[QC_ROPE_MAX_DIM / 2];
} qc_rope;

/* Host function: fills *rope from *cfg. */
int qc_rope_init(const qc_rope_config* cfg, qc_rope* rope);

/* One group of heads of every row, such as a projection row's queries or keys:
 * head h of row r is the head_dim values at x + r * x_ld + h * x_head
 * (elements), its result goes to out + r * out_ld + h * out_head.  out == x
 * with equal strides rotates in place; any other overlap is undefined. */
typedef struct qc_rope_part {
  const uint16_t* x;     /* bf16, device */
  uint16_t* out;         /* bf16, device */
  int64_t n_heads;       /* 1 .. QC_ROPE_MAX_HEADS */
  int64_t x_ld, x_head, out_ld, out_head;
  const float* norm_w;   /* [head_dim] f32, device; NULL: no norm */
} qc_rope_part;

/* Applies the rotation to n_parts groups of n_rows rows in one launch.
 * head_dim: a multiple of 8, rot_dim <= head_dim <= QC_ROPE_MAX_DIM; x, out
 * 16-byte aligned with strides multiples of 8 elements; norm_w 16-byte
 * aligned; pos_dev [n_rows] int32, 4-byte aligned; n_rows 0 is a no-op.  eps >= 0 is the
 * norm's.  rope and parts are host pointers, read before the call returns.
 * The part's memory has to be on the current device.  No allocation; CUDA-
 * graph capturable.  QC_OK, QC_ERR_ARG or QC_ERR_CUDA (qc_last_error(NULL)). */
int qc_rope_apply(const qc_rope* rope, int32_t head_dim, float eps, const int32_t* pos_dev,
                  int32_t n_rows, const qc_rope_part* parts, int32_t n_parts, qc_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* QROPE_H */
