/*
 * nb_block.h -- C ABI of the operators around attention in a transformer block: norms and position rotation of
 * queries and keys (in front of the SDPA call, src/nanobrain/modules.py:59-62), and a gated feed-forward block (in
 * the place of the reference's Mlp, src/nanobrain/modules.py:68-85).
 *
 * Conventions as in nb_attn.h: device pointers, asynchronous on `stream`, nothing is allocated and nothing kept;
 * return values are enum nb_attn_error codes; `status` is the word that kernels write a code of enum nb_attn_status
 * to (optional). bf16 tensors, 16-byte aligned; strides in elements.
 */
#ifndef NB_BLOCK_H_
#define NB_BLOCK_H_

#include <stddef.h>
#include <stdint.h>

#include "nb_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- queries and keys: RMS norm over each head's 64 values, then rotation by the token's position ----------
 * n = x / sqrt(mean(x^2) + eps) * weight; pair i of a head (values i and i + 32, or 2 i and 2 i + 1 where
 * `interleaved`) is turned by angle sum_a position[a] * freqs[a][i], computed in 64 bits. The sum of squares is in
 * fp32 (values beyond 1e18 overflow it); results are rounded once. */
#define NB_ROPE_MAX_AXES 4

enum nb_position_type { NB_POSITION_I32 = 0, NB_POSITION_I64 = 1, NB_POSITION_F32 = 2 };

typedef struct nb_qk_side {
  nb_attn_tensor x;        /* input */
  nb_attn_tensor y;        /* forward: output; backward: the gradient of x */
  nb_attn_tensor dy;       /* backward: the output's gradient */
  const float* weight;     /* [64], or NULL: ones */
  float* d_weight;         /* backward: [64] (required) */
  const void* positions;   /* [axes] contiguous per token */
  int64_t position_stride_batch, position_stride_token;
  int32_t heads;
  int32_t tokens;          /* per sequence of the batch */
} nb_qk_side;

typedef struct nb_qk_norm_rope_args {
  nb_qk_side q, k;
  int32_t batch;           /* packed tokens are one sequence; 0: there is nothing to do but zeros in d_weight */
  int32_t axes;            /* position coordinates per token; 0: no rotation */
  int32_t position_type;   /* enum nb_position_type */
  int32_t interleaved;
  const float* freqs;      /* [axes][32] */
  float eps;
  void* workspace;         /* backward: nb_qk_norm_rope_bwd_workspace_bytes() bytes */
  size_t workspace_bytes;
} nb_qk_norm_rope_args;

int nb_qk_norm_rope_fwd(const nb_qk_norm_rope_args* args, void* stream);
int nb_qk_norm_rope_bwd(const nb_qk_norm_rope_args* args, void* stream);
size_t nb_qk_norm_rope_bwd_workspace_bytes(void);

/* ---- gated feed-forward block: y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd ------------------------------
 * x [tokens][dim], Wg, Wu [hidden][dim], Wd [dim][hidden], y [tokens][dim]; dim and hidden multiples of 8, rows at
 * strides that are multiples of 8. Biases are bf16 and optional (each on its own). */
enum nb_activation { NB_ACT_SILU = 0, NB_ACT_GELU = 1 /* with erf */ };

/* What the forward keeps of a = x Wg^T + bg and b = x Wu^T + bu for the backward: in 16 bits fp16 values with a power of
 * two per 32 features of a token (2^-12 of the value or of 2^-29 of the group's largest; a group with a value that is not
 * finite is kept as plain fp16); in 8 bits whole multiples of max |.| / 127 rounded up to bf16, per 32 features of a token
 * (zeros where that is below 2^-100; a group with a value that is not finite is NaN as a whole).
 *
 * Products are summed in fp32. What a product takes from another is rounded to bf16 first, as the tensor cores want it:
 * act(a) b in front of Wd, and in the backward the gradients of a and b (those of the biases are summed before that). */
enum nb_checkpoint { NB_CHECKPOINT_NONE = 0, NB_CHECKPOINT_16BIT = 1, NB_CHECKPOINT_8BIT = 2 };

typedef struct nb_matrix {
  void* ptr;
  int64_t stride; /* between rows */
} nb_matrix;

typedef struct nb_gated_mlp_shape {
  int64_t tokens;
  int32_t dim, hidden;
  int32_t activation, checkpoint;
} nb_gated_mlp_shape;

size_t nb_gated_mlp_checkpoint_bytes(const nb_gated_mlp_shape* shape);

typedef struct nb_gated_mlp_fwd_args {
  nb_gated_mlp_shape shape;
  nb_matrix x, w_gate, w_up, w_down, y;
  const void *b_gate, *b_up, *b_down;
  nb_matrix h;      /* [tokens][hidden]: the product in front of Wd; the backward wants it unless the checkpoint has 8 bits.
                     * A stride that is a multiple of 64 is faster */
  void* checkpoint; /* nb_gated_mlp_checkpoint_bytes(&shape) bytes, 256-byte aligned */
  int32_t* status;
} nb_gated_mlp_fwd_args;

int nb_gated_mlp_fwd(const nb_gated_mlp_fwd_args* args, void* stream);

typedef struct nb_gated_mlp_bwd_args {
  nb_gated_mlp_shape shape;
  nb_matrix x, w_gate, w_up, w_down, dy;
  nb_matrix h;            /* ptr NULL with an 8-bit checkpoint */
  const void* checkpoint;
  nb_matrix dx, d_w_gate, d_w_up, d_w_down; /* ptr NULL: not wanted */
  void *d_b_gate, *d_b_up, *d_b_down;       /* bf16, NULL: not wanted */
  void* workspace;        /* nb_gated_mlp_bwd_workspace_bytes(args) bytes, 256-byte aligned */
  size_t workspace_bytes;
  int32_t* status;
} nb_gated_mlp_bwd_args;

int nb_gated_mlp_bwd(const nb_gated_mlp_bwd_args* args, void* stream);
/* Goes by the shape and by which gradients are wanted; on the current device. */
size_t nb_gated_mlp_bwd_workspace_bytes(const nb_gated_mlp_bwd_args* args);

#ifdef __cplusplus
}
#endif
#endif /* NB_BLOCK_H_ */
