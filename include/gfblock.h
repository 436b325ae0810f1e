/*
 * gfblock.h -- C ABI of the transformer-block operators in libgfield.so
 * (B200, sm_100a): the gated feed-forward block, counter-based dropout and
 * the product in 8-bit integers that serves a merged weight.
 *
 * The conventions are those of gfield.h: DEVICE pointers unless stated
 * otherwise, caller-owned memory (workspace sizes come from the *_bytes
 * functions and workspaces are 256-byte aligned; none needs zeroing), every
 * launch on `stream` of the current device, no synchronisation except in
 * gf_block_status(), a gf_status from every call, its message from the
 * library's last-error function.  Calls that overlap use different workspaces.
 *
 * Matrices are row-major; a leading dimension counts elements.  They may have
 * any size and leading dimension and start at any element (a pointer that is
 * no multiple of its element's size is refused): operands whose rows do not
 * start on 16-byte boundaries, and a w_in whose hidden size is no multiple of
 * 64, are first copied into the workspace, which costs one pass over them.
 */
#ifndef GFBLOCK_H
#define GFBLOCK_H

#include "gfield.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types, beside gf_dtype's GF_F32 and GF_BF16. */
#define GF_F16 2

typedef enum gf_activation {
  GF_ACT_GELU = 0, /* g * Phi(g), the exact (error-function) form */
  GF_ACT_SILU = 1  /* g / (1 + exp(-g)) */
} gf_activation;

/* Condition bits of gf_block_status(). */
#define GF_FLAG_TIMEOUT 0x10u /* a kernel gave up waiting for its own copies or products; its output is not valid */

/* Dropout: element (row, col) is kept when word col % 4 of Philox-4x32-10
 * (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011)
 * with key (seed low, seed high) and counter (col / 4, row low, site, row
 * high) is at least round(p * 2^32), and is then multiplied by 1 / (1 - p);
 * a dropped element is 0 whatever it held.  The mask is a function of these
 * numbers alone, so the backward makes it again and nothing is stored. */
typedef struct gf_dropout_rule {
  double p;                   /* 0 <= p < 1; 0 = no dropout */
  uint64_t seed;              /* used when seed_ptr is NULL */
  const uint64_t* seed_ptr;   /* device: the seed is read when the kernel runs, so a captured graph sees new values */
  uint32_t site;              /* tells apart the dropouts that share a seed */
  uint32_t reserved;          /* 0 */
} gf_dropout_rule;

/* The gated feed-forward block:
 *   u = x w_in^T + b_in          [tokens, 2 * hidden]: value half, gate half
 *   h = dropout(u_value * act(u_gate))
 *   y = h w_out^T + b_out        [tokens, out_features]
 * Products accumulate in fp32; h and the gradient of u are rounded to `dtype`
 * where they are stored (tensor-core operands), y and the gradients once at
 * the end.
 *
 * The forward writes h, with leading dimension Hp = hidden rounded up to a
 * multiple of 64.  The backward takes the forward's inputs, computes u and the
 * dropout again from them, and needs the saved h when dw_out is wanted only. */
typedef struct gf_gated_ff {
  int64_t tokens, in_features, hidden, out_features; /* tokens >= 0, the others > 0, each < 2^31 - 512 */
  int32_t dtype;      /* GF_BF16 or GF_F16, of every matrix and vector */
  int32_t activation; /* gf_activation */
  gf_dropout_rule dropout;
  const void* x;     int64_t ld_x;     /* [tokens, in_features] */
  const void* w_in;  int64_t ld_w_in;  /* [2 * hidden, in_features] */
  const void* b_in;                    /* [2 * hidden] or NULL */
  const void* w_out; int64_t ld_w_out; /* [out_features, hidden] */
  const void* b_out;                   /* [out_features] or NULL */
  void* h;                             /* [tokens, Hp]; 16-byte aligned */
  void* y;           int64_t ld_y;     /* [tokens, out_features] (forward) */
  /* backward: the gradient of y, and the wanted gradients (NULL = not wanted; contiguous) */
  const void* dy;    int64_t ld_dy;    /* [tokens, out_features] */
  void* dx;                            /* [tokens, in_features] */
  void* dw_in;                         /* [2 * hidden, in_features] */
  void* db_in;                         /* [2 * hidden] */
  void* dw_out;                        /* [out_features, hidden] */
  void* db_out;                        /* [out_features] */
} gf_gated_ff;

/* Workspace bytes of a pass (from the sizes, leading dimensions, pointers'
 * alignment and the wanted gradients).  0 with an error when the description
 * is not valid; a valid description needs at least 256. */
size_t gf_gated_ff_workspace_bytes(const gf_gated_ff* ff, gf_pass pass);
gf_status gf_gated_ff_forward(const gf_gated_ff* ff, void* workspace, size_t workspace_bytes, gf_stream stream);
gf_status gf_gated_ff_backward(const gf_gated_ff* ff, void* workspace, size_t workspace_bytes, gf_stream stream);

/* y = dropout(x) (+ residual).  x and residual are [rows, cols] with any
 * strides (in elements); y is contiguous.  Its gradient with respect to x is
 * the same call on dy without the residual.  dtype: GF_F32, GF_BF16, GF_F16. */
gf_status gf_dropout(int64_t rows, int64_t cols, int32_t dtype, const gf_dropout_rule* rule, const void* x,
                     int64_t x_row_stride, int64_t x_col_stride, const void* residual, int64_t r_row_stride,
                     int64_t r_col_stride, void* y, gf_stream stream);

/* Symmetric quantisation of each row to 8 bits: scale = max|x| / 127,
 * q = round-to-even(x * (127 / max|x|)), both in fp32; a row of zeros gives
 * zeros with scale 0, and so does one whose maximum is below 2^-100; a row
 * that holds an infinity or a NaN gives zeros with scale NaN.  q has leading
 * dimension ld_q >= cols; columns cols .. ld_q - 1 are set to zero. */
gf_status gf_quantize_rows(int64_t rows, int64_t cols, int32_t dtype, const void* x, int64_t ld_x, int8_t* q,
                           int64_t ld_q, float* scale, gf_stream stream);

/* out[m, n] = (sum_k a[m, k] * b[n, k]) * a_scale[m] * b_scale[n] + bias[n].
 * The sum is exact (32-bit integers, k <= 131071); the scales are applied in
 * fp32 and the result is rounded once to `dtype`, which is also the bias's. */
typedef struct gf_int8_product {
  int64_t m, n, k;                    /* m >= 0, n > 0, 0 < k <= 131071 */
  int32_t dtype;                      /* GF_F32, GF_BF16 or GF_F16 */
  int32_t reserved;                   /* 0 */
  const int8_t* a;  int64_t ld_a;     /* [m, k] */
  const int8_t* b;  int64_t ld_b;     /* [n, k] */
  const float* a_scale;               /* [m] */
  const float* b_scale;               /* [n] */
  const void* bias;                   /* [n] or NULL */
  void* out;        int64_t ld_out;   /* [m, n] */
} gf_int8_product;

size_t gf_int8_product_workspace_bytes(const gf_int8_product* p);
gf_status gf_int8_matmul(const gf_int8_product* p, void* workspace, size_t workspace_bytes, gf_stream stream);

/* out = quantise(x) b^T with x [m, k] of x_dtype, quantised row by row as
 * gf_quantize_rows does; a, ld_a and a_scale of the product are not used. */
size_t gf_int8_linear_workspace_bytes(const gf_int8_product* p);
gf_status gf_int8_linear(const gf_int8_product* p, const void* x, int64_t ld_x, int32_t x_dtype, void* workspace,
                         size_t workspace_bytes, gf_stream stream);

/* Synchronises `stream` and returns the condition bits that these operators
 * set on the current device since the last reset. */
gf_status gf_block_status(gf_stream stream, int reset, uint32_t* flags_out);

/* Enqueues a copy of those bits, as they are once the work before it on
 * `stream` is done, into device memory; does not synchronise. */
gf_status gf_block_status_async(uint32_t* flags_out, gf_stream stream);

#ifdef __cplusplus
}
#endif
#endif
