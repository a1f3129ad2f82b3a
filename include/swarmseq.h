/*
 * swarmseq.h — C ABI of the sequence-policy operators in libswarmstep.so.
 *
 * The trainers' own memory is an LSTM of at most 64 units (swarmtrain.h) and their categorical losses
 * take at most 64 choices in float32. These operators serve policies over long sequences, wide
 * memories and large action spaces, in float32, bfloat16 and float16:
 *
 *   swarm_gated_scan_*     a gated linear recurrence over whole sequences, its gradients and one step of it
 *   swarm_residual_norm_*  root-mean-square norm of a residual sum, and its gradients
 *   swarm_policy_loss_*    the clipped policy loss with a KL term and an entropy bonus, from logits
 *   swarm_log_probs        log-probability of the taken action and entropy of every row of logits
 *
 * Conventions as swarmstep.h: caller-owned device pointers, async on `stream`, 0 = ok, negative =
 * swarm_status_t. `dtype` is a swarm_dtype_t and names the element type behind `void` pointers; they
 * need the alignment of that type only. Sums, norms, softmax statistics and states are float32.
 * Workspaces are the caller's: two calls that may overlap need their own. Sizes of zero are legal
 * wherever a bound below says >= 0; such a call launches nothing that it does not need.
 */
#ifndef SWARMSEQ_H
#define SWARMSEQ_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    SWARM_F32 = 0,
    SWARM_BF16 = 1,
    SWARM_F16 = 2
} swarm_dtype_t;

/* Gated linear recurrence over n >= 0 sequences of T >= 1 steps and U >= 1 channels. With the gate
 * pre-activations of step t in three blocks, gates[i][t] = forget xf[U] | candidate xz[U] | output xo[U]:
 *     p_t = keep[t-1] c_{t-1} (p_0 = c0)     f = sigmoid(xf), o = sigmoid(xo)
 *     c_t = f p_t + (1 - f) xz               h_t = o c_t
 * Steps t >= lengths[i] (clamped to [0, T]) are padding: the state stands still, h is 0, and what gates,
 * keep and d_h hold there is not used (NaN included).
 *   gates: element (i, t, c) at gates[i * gates_n + t * gates_t + c]; c0: [n][U] f32 or NULL (zeros);
 *   keep: [n][T] f32 within [-1, 1] or NULL (ones; steps are joined by products of f and keep, which larger values
 *   would carry out of range); lengths: [n] int64 or NULL (T).
 *   h: [n][T][U]; c_last: [n][U] f32, the state behind the last step;
 *   tile_states: [n][SWARM_GATED_TILES(T)][U] f32, the state before every SWARM_GATED_TILE-th step, for the
 *   backward pass (NULL: not kept); work: swarm_gated_scan_workspace(n, T, U) floats (NULL where that is 0). */
#define SWARM_GATED_TILE 32
#define SWARM_GATED_TILES(T) (((int64_t)(T) + SWARM_GATED_TILE - 1) / SWARM_GATED_TILE)
int64_t swarm_gated_scan_workspace(int64_t n, int64_t T, int64_t U);
int32_t swarm_gated_scan_forward(int32_t dtype, int64_t n, int64_t T, int64_t U, const void* gates, int64_t gates_n,
                                 int64_t gates_t, const float* c0, const float* keep, const int64_t* lengths, void* h,
                                 float* c_last, float* tile_states, float* work, void* stream);

/* Gradients of swarm_gated_scan_forward from its inputs and tile_states: d_h with strides as gates
 * (d_h_n, d_h_t), d_last: [n][U] f32; either may be NULL (zeros). d_gates: [n][T][3U] (every element,
 * zeros in the padding); d_c0: [n][U] f32 or NULL. */
int32_t swarm_gated_scan_backward(int32_t dtype, int64_t n, int64_t T, int64_t U, const void* gates, int64_t gates_n,
                                  int64_t gates_t, const float* keep, const int64_t* lengths,
                                  const float* tile_states, const void* d_h, int64_t d_h_n, int64_t d_h_t,
                                  const float* d_last, void* d_gates, float* d_c0, float* work, void* stream);

/* One step: c_out = f (keep c) + (1 - f) xz, h = o c_out for rows >= 0 rows of gates (row stride
 * gates_row); keep: [rows] f32 or NULL; c, c_out: [rows][U] f32, c_out may be c. */
int32_t swarm_gated_step(int32_t dtype, int64_t rows, int64_t U, const void* gates, int64_t gates_row, const float* c,
                         const float* keep, void* h, float* c_out, void* stream);

/* stream_out = x + residual (rounded to dtype; residual NULL: x, and stream_out is not written), and of
 * that sum before its rounding y = sum * rstd * weight, rstd = 1 / sqrt(mean(sum^2) + eps), per row of D >= 1
 * elements. x and residual rows are x_row / res_row elements apart; y, stream_out: [rows][D]; weight: [D] of
 * dtype or NULL (ones); rstd: [rows] f32 or NULL. */
int32_t swarm_residual_norm_forward(int32_t dtype, int64_t rows, int64_t D, const void* x, int64_t x_row,
                                    const void* residual, int64_t res_row, const void* weight, float eps, void* y,
                                    void* stream_out, float* rstd, void* stream);

/* d_x = rstd (w d_y - n mean(w d_y n)) + d_stream with n = sum * rstd (the gradient of x and of residual
 * alike), sum = x + residual before any rounding, d_weight = column sums of d_y n in a fixed order. x,
 * residual, weight: as in the forward pass, which wrote rstd; d_y, d_stream: rows dy_row / ds_row apart,
 * d_stream may be NULL; d_x: [rows][D]; d_weight: [D <= 2^27 - 32] of dtype or NULL; work:
 * swarm_residual_norm_workspace(rows, D) floats, needed with d_weight. */
int64_t swarm_residual_norm_workspace(int64_t rows, int64_t D);
int32_t swarm_residual_norm_backward(int32_t dtype, int64_t rows, int64_t D, const void* x, int64_t x_row,
                                     const void* residual, int64_t res_row, const void* weight, const float* rstd,
                                     const void* d_y, int64_t dy_row, const void* d_stream, int64_t ds_row, void* d_x,
                                     void* d_weight, float* work, void* stream);

int64_t swarm_log_probs_workspace(int64_t M, int64_t K);
/* log_probs[m] = z[m][a_m] - logsumexp(z[m]) and entropy[m] = -sum_k p_k log p_k over M >= 0 rows of K >= 1
 * logits (rows row_stride apart). A logit of -inf is a choice that cannot be taken. An action outside [0, K)
 * gives NaN and sets *bad_actions (device int32, or NULL) to 1. work: swarm_log_probs_workspace(M, K) floats (NULL
 * where that is 0). */
int32_t swarm_log_probs(int32_t dtype, int64_t M, int64_t K, const void* logits, int64_t row_stride,
                        const int64_t* actions, float* log_probs, float* entropy, float* work, int32_t* bad_actions,
                        void* stream);

/* The clipped policy loss over the active rows (mask_u8, NULL: all) of M >= 0 rows of K logits:
 *     l = log p(a),  r = exp(l - old),  pg = -min(r A, clamp(r, clip_lo, clip_hi) A)
 *     d = ref - l,   kl = exp(d) - d - 1 (0 without ref),   H = entropy
 *     *loss = sum(pg + kl_coef kl - entropy_coef H) / denom
 *     terms[4] = the means of pg, kl, H and of the share of rows with r outside [clip_lo, clip_hi]
 * l - old and d are bounded to [-20, 20] (no gradient outside). denom: *denom if given, else
 * max(active rows, 1); the one used goes to *used_denom. Inactive rows are not looked at.
 *   old, ref, adv: [M] f32; row_stats: [M][4] f32 for the backward pass; d_logits: [M][K], the gradient for an
 *   incoming gradient of 1, formed from the logits while they are at hand (NULL: not formed); partials:
 *   SWARM_POLICY_LOSS_PARTIALS floats of workspace. An active row's action outside [0, K) makes the loss NaN
 *   and sets *bad_actions to 1. */
#define SWARM_POLICY_LOSS_PARTIALS (2048 * 6)
int32_t swarm_policy_loss_forward(int32_t dtype, int64_t M, int64_t K, const void* logits, int64_t row_stride,
                                  const int64_t* actions, const float* old_log_probs, const float* ref_log_probs,
                                  const float* advantages, const uint8_t* mask_u8, const float* denom, float clip_lo,
                                  float clip_hi, float kl_coef, float entropy_coef, float* loss, float* terms,
                                  float* used_denom, float* row_stats, void* d_logits, float* partials,
                                  int32_t* bad_actions, void* stream);
/* d_logits: [M][K], every element (zeros on inactive rows), for the incoming gradient *grad of *loss. have_unit:
 * d_logits holds what the forward call put there, and stays as it is where *grad is 1. */
int32_t swarm_policy_loss_backward(int32_t dtype, int64_t M, int64_t K, const void* logits, int64_t row_stride,
                                   const int64_t* actions, float entropy_coef, const float* row_stats,
                                   const float* used_denom, const float* grad, int32_t have_unit, void* d_logits,
                                   void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SWARMSEQ_H */
