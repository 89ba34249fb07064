/*
 * minigrid_ops.h — C ABI of the learning operators of libminigrid_hip.so: what turns the batched environments' observations into actions and their
 * trajectories into a gradient.  minigrid_amd/csrc/ops/mg_torch.cpp and minigrid_amd/ops.py are
 * the binding (torch tensors, autograd).
 *
 * Conventions
 *   - plain C types only; every function returns MG_OK (0) or a negative mg_status (minigrid_hip.h); mg_ops_last_error() has the text of the calling
 *     thread's last failure.
 *   - stateless: no handle, no allocation, no synchronisation.  All pointers are device memory of `device`; work is enqueued on `stream` (a
 *     hipStream_t; NULL = the null stream).  A call may be captured into a graph.  Two calls that may run at once need two workspaces.
 *   - `ld*` are row strides in ELEMENTS; the columns of a row are contiguous.  Types are mg_dtype values.
 *   - results overlap neither operands nor each other.
 *   - a workspace is scratch: its content before a call does not matter and after it means nothing; it has to be 256-byte aligned.
 */
#ifndef MINIGRID_OPS_H
#define MINIGRID_OPS_H

#include "minigrid_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum mg_dtype { MG_DT_F32 = 0, MG_DT_BF16 = 1, MG_DT_F16 = 2, MG_DT_U8 = 3, MG_DT_F64 = 4, MG_DT_I32 = 5, MG_DT_I64 = 6 } mg_dtype;
typedef enum mg_activation { MG_ACTIVATION_NONE = 0, MG_ACTIVATION_RELU = 1, MG_ACTIVATION_TANH = 2, MG_ACTIVATION_GELU = 3, MG_ACTIVATION_SILU = 4,
  MG_ACTIVATION_TANH_Z32 = 18 /* tanh whose z is f32 whatever the dtype: from a z rounded to 16 bits its slope loses the most */ } mg_activation;

MG_API const char* mg_ops_last_error(void);

/* ---- a layer of a policy network: y = act(x wT + b) + r ----
 * x (rows, k) of `dtype` or bytes (x_dtype = MG_DT_U8: an observation as the environments write it), w (n, k), b (n) or NULL, r (rows, n) or NULL,
 * y (rows, n), all of `dtype` (f32, bf16, f16).  z (rows, n, contiguous; `dtype`, f32 for MG_ACTIVATION_TANH_Z32) or NULL: the values in front of the
 * activation, for the backward pass.  Sums are held in 32 bits.  act = gelu is x Phi(x) with the normal distribution function itself. */
MG_API int mg_op_linear_workspace(int64_t rows, int64_t k, int64_t n, int dtype, int64_t* forward, int64_t* backward_input, int64_t* backward_weight);
MG_API int mg_op_linear(int device, void* stream, int dtype, int x_dtype, int act, int64_t rows, int64_t k, int64_t n, const void* x, int64_t ldx,
                        const void* w, int64_t ldw, const void* b, const void* r, int64_t ldr, void* y, int64_t ldy, void* z, void* ws, int64_t ws_bytes);
/* dz = dy * act'(z), z as a forward pass with the same act has left it (dz: rows, n, contiguous; NULL allowed for act = none) and db = the column sums of dz (n, `dtype`; NULL = not wanted).
 * ws: mg_op_linear_dz_workspace bytes (needed for db only). */
MG_API int mg_op_linear_dz_workspace(int64_t rows, int64_t n, int64_t* bytes);
MG_API int mg_op_linear_dz(int device, void* stream, int dtype, int act, int64_t rows, int64_t n, const void* dy, int64_t lddy, const void* z, void* dz,
                           void* db, void* ws, int64_t ws_bytes);
/* dx (rows, k, contiguous) = dz w */
MG_API int mg_op_linear_dx(int device, void* stream, int dtype, int64_t rows, int64_t k, int64_t n, const void* dz, int64_t lddz, const void* w, int64_t ldw,
                           void* dx, void* ws, int64_t ws_bytes);
/* dw (n, k, contiguous) = dzT x */
MG_API int mg_op_linear_dw(int device, void* stream, int dtype, int x_dtype, int64_t rows, int64_t k, int64_t n, const void* dz, int64_t lddz, const void* x,
                           int64_t ldx, void* dw, void* ws, int64_t ws_bytes);

/* ---- the clipped policy loss with KL and entropy terms ----
 * logits (rows, vocab), action (rows; u8, i32 or i64), old_lp / adv / ref_lp (rows, f32; ref_lp may be NULL), mask (rows, u8; NULL = all rows count).
 * With lp = log softmax(logits)[action], q = exp(lp - old_lp), H = the entropy of softmax(logits), the loss is the mean over the counted rows of
 *     -min(q adv, clamp(q, 1 - clip_lo, 1 + clip_hi) adv) + kl_coef (exp(ref_lp - lp) - (ref_lp - lp) - 1) - ent_coef H.
 * out (6 f32): loss, mean policy term, mean KL term, mean entropy, share of clipped rows, number of counted rows.  No counted row: all 0.
 * save ((rows + 1) x 16 bytes) is what the backward call needs; NULL = no backward pass will follow.  Rows that do not count are not read.
 * A counted row's action outside 0..vocab-1 makes the loss and the row's gradient NaN. */
MG_API int mg_op_policy_loss_workspace(int64_t rows, int64_t vocab, int64_t* bytes);
MG_API int mg_op_policy_loss(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const void* action, int action_dtype,
                             const float* old_lp, const float* adv, const float* ref_lp, const uint8_t* mask, double clip_lo, double clip_hi, double kl_coef,
                             double ent_coef, float* out, void* save, void* ws, int64_t ws_bytes);
/* The same, and dlogits (rows, vocab, contiguous; NULL = not wanted) = d loss / d logits along with it.  For rows of more than 64
 * columns and at most 160 KB: mg_op_policy_loss_makes_gradient says whether (1 or 0). */
MG_API int mg_op_policy_loss_makes_gradient(int dtype, int64_t vocab);
MG_API int mg_op_policy_loss_with_gradient(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const void* action, int action_dtype,
                                           const float* old_lp, const float* adv, const float* ref_lp, const uint8_t* mask, double clip_lo, double clip_hi, double kl_coef,
                                           double ent_coef, float* out, void* save, void* ws, int64_t ws_bytes, void* dlogits);
/* dlogits (rows, vocab, contiguous) = grad[0] * d loss / d logits; rows that do not count get 0 */
MG_API int mg_op_policy_loss_backward(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const void* action, int action_dtype,
                                      const uint8_t* mask, double ent_coef, const void* save, const float* grad, void* dlogits);

/* the same for a dlogits that already holds the gradient for the factor 1: left as it is where grad[0] is 1, else computed anew */
MG_API int mg_op_policy_loss_rescale(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const void* action, int action_dtype,
                                     const uint8_t* mask, double ent_coef, const void* save, const float* grad, void* dlogits);

/* ---- one draw per row: action = the lowest k with sum_{j<=k} e^{l_j} > u sum_j e^{l_j}, sums in 64 bits; u NULL: the lowest index of the largest logit ----
 * u (rows, f32 in [0, 1)); action: u8 where vocab <= 256, else i32; lp (rows, f32) = log softmax(logits)[action].  A row without a finite largest logit
 * gives action 0 and lp NaN. */
MG_API int mg_op_sample_workspace(int64_t rows, int64_t vocab, int64_t* bytes);
MG_API int mg_op_sample(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const float* u, void* action, float* lp,
                        void* ws, int64_t ws_bytes);

/* ---- generalised advantages of a rollout of `steps` x `envs` ----
 * reward (f64 or f32), value, terminated, truncated: element (t, e) at t * s?[0] + e * s?[1] elements; last_value (envs); done0 (envs, u8) or NULL: whether
 * an episode ended in the step before the first; final_value or NULL (same_step only): the value of the observation a truncated step ended on.
 * next_step != 0 is the environments' default autoreset: the step behind an end only resets, counts for nothing (valid = 0, advantage 0), and its
 * observation is the one the episode ended on.  next_step = 0: the step behind an end is the first of the next episode.
 * Where reward (f64), terminated and truncated are the first fields of 16-byte records at 16-byte addresses, as the environments write them, records are read whole.
 * advantage, ret (f32) and valid (u8): (steps, envs), contiguous. */
typedef struct mg_advantages_args {
  int64_t steps, envs;
  const void* reward; int64_t s_reward[2];
  const void* value; int64_t s_value[2];
  const void* final_value; int64_t s_final[2];
  const uint8_t* terminated; int64_t s_term[2];
  const uint8_t* truncated; int64_t s_trunc[2];
  const void* last_value;
  const uint8_t* done0;
  float* advantage; float* ret; uint8_t* valid;
  double gamma, lam;
  int32_t reward_dtype, value_dtype, next_step, reserved;
} mg_advantages_args;
MG_API int mg_op_advantages(int device, void* stream, const mg_advantages_args* args);

#ifdef __cplusplus
}
#endif
#endif
