/*
 * newt_ops.h - C ABI of libnewt_ops.so: the hand-written gfx950 operators of a
 * decoder's serving step. They stand beside the kernels that newt compiles at
 * run time (include/newt_hip.h) and follow the same conventions: plain pointers
 * and sizes, streams as void* (a hipStream_t, NULL = default stream), 0 on
 * success, a hipError_t below 10000 or NEWT_ERR_INVALID otherwise, and the
 * detailed message of the calling thread's last failure in
 * newt_ops_last_error(). Each call only launches on the stream it is given: it
 * allocates nothing, keeps nothing and does not wait. All device pointers must
 * be of the stream's device, which must be the current one. Strides count
 * elements; where none is given for a dimension it is contiguous.
 * newt_amd/serving.py fills these structs; the field order is its pack format.
 */
#ifndef NEWT_OPS_H
#define NEWT_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "newt_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NEWT_OPS_ABI_VERSION 1

/* element types */
#define NEWT_F32 0
#define NEWT_F16 1
#define NEWT_BF16 2
#define NEWT_E4M3 3 /* OCP float8_e4m3fn: 4 exponent, 3 mantissa bits, largest 448 */

int newt_ops_abi_version(void);
const char* newt_ops_last_error(void);

/* hidden = x + residual (rounded to x's type; without a residual x itself),
 * out = hidden * rsqrt(mean(hidden^2) + eps) * w over each row; an E4M3 `out`
 * holds out / scale, with scale = max(amax |out| / 448, 2^-126) of each `group`
 * columns (0: of the row). */
typedef struct {
  const void* x;        /* [rows, cols] of dtype */
  const void* residual; /* as x, or NULL */
  const void* w;        /* [cols] of w_dtype */
  void* out;            /* [rows, cols] of dtype, or E4M3 */
  void* hidden;         /* as x (may be x or residual itself); NULL without a residual */
  float* scale;         /* [rows, cols / group] fp32, NULL unless out is E4M3 */
  int64_t rows, cols;
  int64_t x_stride, residual_stride, out_stride, hidden_stride;
  float eps;
  int32_t dtype, w_dtype, out_dtype;
  int32_t group; /* 0, 32, 64, 128 or 256; divides cols */
  int32_t reserved;
} newt_rmsnorm_params;
int newt_rmsnorm(const newt_rmsnorm_params* p, void* stream);

/* Per row of logits, with x = logits / temperature: logp[t] = x[token] -
 * logsumexp(x), the entropy of softmax(x), and the `top` largest log
 * probabilities with their ids, the lowest id first among equal ones. */
typedef struct {
  const void* logits;   /* [rows, vocab] of dtype */
  const void* tokens;   /* [rows] int64; -1: no token, logp 0; else outside [0, vocab): NaN */
  float* logp;          /* [rows] */
  float* entropy;       /* [rows] */
  float* top_logp;      /* [rows, top] */
  int64_t* top_ids;     /* [rows, top] */
  void* workspace;      /* newt_token_logprobs_workspace() bytes, or NULL if that is 0 */
  int64_t rows, vocab, stride;
  float inv_temperature;
  int32_t dtype;
  int32_t top;          /* 0..64 */
  int32_t reserved;
} newt_logprobs_params;
int newt_token_logprobs(const newt_logprobs_params* p, void* stream);
size_t newt_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t top, int32_t dtype);

/* The 8-bit cache: `blocks` blocks of `block_size` tokens of kv_heads heads.
 *   k [blocks, kv_heads, block_size, head_dim], v [blocks, kv_heads, head_dim,
 *   block_size] E4M3, k_scale and v_scale [blocks, kv_heads] fp32, all
 *   contiguous; a value is its byte's times its block's and head's scale, which
 *   is not negative. */
typedef struct {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t blocks;
  int32_t kv_heads, block_size, head_dim, reserved;
} newt_kv_cache;

/* Writes count[b] new tokens of each sequence to positions start[b] on. No block
 * may be written at two places by one call. */
typedef struct {
  newt_kv_cache cache;
  const void* k;            /* [batch, kv_heads, tokens, head_dim] of dtype */
  const void* v;
  const int32_t* table;     /* [batch, table_width] block ids */
  const int32_t* start;     /* [batch] */
  const int32_t* count;     /* [batch], or NULL: all `tokens` */
  int64_t batch, tokens, table_width, table_stride;
  int64_t k_stride_b, k_stride_h, k_stride_t;
  int64_t v_stride_b, v_stride_h, v_stride_t;
  int32_t dtype, reserved;
} newt_kv_append_params;
int newt_kv_append(const newt_kv_append_params* p, void* stream);

/* Attention of q's tokens, the last `q_len` of each sequence, over the cache. */
typedef struct {
  newt_kv_cache cache;
  const void* q;            /* [batch, heads, q_len, head_dim] of dtype */
  void* out;                /* as q; rows that overlap, in part too, are refused */
  const int32_t* table;     /* [batch, table_width] block ids */
  const int32_t* lens;      /* [batch] tokens of each sequence, q's among them */
  void* workspace;          /* newt_cached_attention_workspace() bytes, or NULL if that is 0 */
  int64_t batch, q_len, table_width, table_stride;
  int64_t q_stride_b, q_stride_h, q_stride_t;
  int64_t o_stride_b, o_stride_h, o_stride_t;
  int64_t window;           /* tokens that a query sees, itself among them; 0: all before it */
  int64_t sinks;            /* first tokens that stay visible behind the window */
  float scale;
  int32_t heads, dtype, reserved;
} newt_cached_attention_params;
int newt_cached_attention(const newt_cached_attention_params* p, void* stream);
size_t newt_cached_attention_workspace(const newt_cached_attention_params* p);

/* Causal attention in a window, with sinks. Query i of sequence b is at
 * position q_start[b] + i (q_start NULL: kv_len - q_len + i) and sees key j if
 * j <= position and (position - j < window or j < sinks). */
typedef struct {
  const void* q;            /* [batch, heads, q_len, head_dim] of dtype */
  const void* k;            /* [batch, kv_heads, kv_len, head_dim] */
  const void* v;
  void* out;                /* as q */
  const int32_t* q_start;   /* [batch] or NULL */
  void* workspace;          /* newt_window_attention_workspace() bytes, or NULL if that is 0 */
  int64_t batch, q_len, kv_len;
  int64_t q_stride_b, q_stride_h, q_stride_t;
  int64_t k_stride_b, k_stride_h, k_stride_t;
  int64_t v_stride_b, v_stride_h, v_stride_t;
  int64_t o_stride_b, o_stride_h, o_stride_t;
  int64_t window, sinks;
  float scale;
  int32_t heads, kv_heads, head_dim, dtype, reserved;
} newt_window_attention_params;
int newt_window_attention(const newt_window_attention_params* p, void* stream);
size_t newt_window_attention_workspace(const newt_window_attention_params* p);

#ifdef __cplusplus
}
#endif

#endif /* NEWT_OPS_H */
