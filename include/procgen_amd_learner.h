/*
 * procgen_amd_learner.h -- the learner operators of libenv.so: what a policy gradient needs of a rollout window (T steps of N envs), computed where
 * the step and render kernels left the rollout, in HBM.  No handle: plain device pointers of the caller, on the caller's stream.
 *
 * Every entry point
 *   - runs on device `device` and enqueues on `stream` (a hipStream_t of that device) without synchronizing; the caller's current device is kept;
 *   - allocates nothing and keeps nothing between calls: outputs and workspaces are the caller's, so calls on several streams, host threads or in
 *     captured graphs do not meet (each needs a workspace of its own while it runs);
 *   - returns 0, -1 for arguments it does not take (nothing is enqueued), or the hipError_t of a launch that failed.  It never ends the process;
 *   - reads strides in ELEMENTS, 64 bits wide; element types are PROCGEN_AMD_F32 / F16 / BF16.  Sums, states and statistics are held in 32 bits
 *     or more; what is written to a 16-bit output is rounded once, to nearest even.
 */
#ifndef PROCGEN_AMD_LEARNER_H
#define PROCGEN_AMD_LEARNER_H

#include "libenv.h"

#ifdef __cplusplus
extern "C" {
#endif

enum procgen_amd_dtype { PROCGEN_AMD_F32 = 0, PROCGEN_AMD_F16 = 1, PROCGEN_AMD_BF16 = 2 };

/* a [T][N][D] array: element (t, n, d) is data[t * t_stride + n * n_stride + d * d_stride]; a stride of 0 repeats (inputs only) */
struct procgen_amd_array3 {
    void *data;
    long long t_stride, n_stride, d_stride;
};

/* Gated linear recurrence along t, every (n, d) a chain of its own:
 *     h[t] = keep[t] * gate[t] * h[t-1] + update[t],   keep[t] = (first[t][n] == 0),   h[-1] = state (zeros when NULL)
 * Where first is set the old state and the gate are not looked at, whatever they hold.  Products of neighbouring gates are formed on the way: where one
 * passes float's range, h behind it is not finite unless h before it is zero (or first is set in between); gradients alike, from the last step to the first.
 * state, state_out: float [N][D], contiguous; state_out may be state (updated in place), or NULL.  checkpoints: NULL, or float
 * [procgen_amd_recurrence_checkpoints(T)][N][D], which the backward pass reads (it does not read state).  workspace: memory of
 * procgen_amd_recurrence_workspace(T, N, D) bytes (NULL when that is 0). */
struct procgen_amd_recurrence {
    int dtype;                                    /* of gate, update, h and their gradients */
    int T, N, D;
    struct procgen_amd_array3 gate, update, h;
    const uint8_t *first;                         /* NULL: no episode begins inside the window */
    long long first_t_stride, first_n_stride;
    const float *state;
    float *state_out;
    float *checkpoints;
    void *workspace;
    /* backward only: d_h and d_state_out are read (NULL data: zeros), d_gate, d_update (NULL data: not wanted) and d_state are written */
    struct procgen_amd_array3 d_h, d_gate, d_update;
    const float *d_state_out;
    float *d_state;
};
LIBENV_API long long procgen_amd_recurrence_checkpoints(int T);
LIBENV_API long long procgen_amd_recurrence_workspace(int T, int N, int D);
LIBENV_API int procgen_amd_recurrence_forward(const struct procgen_amd_recurrence *args, int device, void *stream);
LIBENV_API int procgen_amd_recurrence_backward(const struct procgen_amd_recurrence *args, int device, void *stream);

/* Generalized advantages and returns of a rollout window:
 *     delta[t] = rew[t] + gamma * keep[t+1] * v[t+1] - v[t],   adv[t] = delta[t] + gamma * lam * keep[t+1] * adv[t+1],   ret[t] = adv[t] + v[t]
 * with keep[t] = (first[t] == 0).  rew: float [T][N]; values (dtype) and first: [T+1][N]; adv, ret: float [T][N] contiguous, either may be NULL.
 * Where first[t+1] is set, v[t+1] is not looked at.  workspace: procgen_amd_recurrence_workspace(T, N, 1) bytes. */
struct procgen_amd_advantage {
    int dtype;                                    /* of values */
    int T, N;
    const float *rew;
    long long rew_t_stride, rew_n_stride;
    const void *values;
    long long values_t_stride, values_n_stride;
    const uint8_t *first;
    long long first_t_stride, first_n_stride;
    float gamma, lam;
    float *adv, *ret;
    void *workspace;
};
LIBENV_API int procgen_amd_advantages(const struct procgen_amd_advantage *args, int device, void *stream);

/* Rows of logits, one column per action.  Row r = r0 * inner + r1 begins at logits + r0 * outer_stride + r1 * inner_stride; its columns are
 * contiguous.  A column of -inf is an action the policy cannot take.  A row without any finite column has no distribution: its log-prob is -inf,
 * its entropy and gradient 0.  An action outside [0, columns) has no log-prob: NaN (its row's gradient too). */
struct procgen_amd_rows {
    int dtype;
    long long rows, columns, inner;
    const void *logits;
    long long outer_stride, inner_stride;
    const void *actions;                          /* [rows] */
    int actions_are_64_bit;
    void *d_logits;                               /* [rows][columns] contiguous, dtype: written by the calls with a gradient */
    void *workspace;                              /* procgen_amd_rows_workspace(rows, columns) bytes */
};
LIBENV_API long long procgen_amd_rows_workspace(long long rows, long long columns);

/* log sum exp of a row = largest + log_sum, with log_sum = log sum exp(logit - largest).  In two parts: one float of the size of the logits would round
 * log_sum away.  largest = -inf: a row without any finite column. */
struct procgen_amd_lse {
    float largest, log_sum;
};
/* logp[r] = log p(actions[r]), entropy[r]: float [rows]; lse: [rows], read by the backward call, or NULL */
LIBENV_API int procgen_amd_action_logprobs(const struct procgen_amd_rows *rows, float *logp, float *entropy, struct procgen_amd_lse *lse, int device, void *stream);
/* d_logits of sum(d_logp * logp + d_entropy * entropy); d_logp, d_entropy: float [rows] or NULL (zeros).  A row whose two are zero gets zeros,
 * whatever its logits hold. */
LIBENV_API int procgen_amd_action_logprobs_backward(const struct procgen_amd_rows *rows, const struct procgen_amd_lse *lse, const float *entropy, const float *d_logp, const float *d_entropy, int device, void *stream);

/* Clipped policy loss with a KL term:
 *     ratio = exp(logp - old_logprobs);  objective = min(ratio * adv, clip(ratio, 1 - clip_low, 1 + clip_high) * adv)
 *     KL = sum p (log p - log q), q from ref_logits (laid out by ref_outer_stride / ref_inner_stride, dtype of logits);
 *       or its estimator exp(d) - d - 1, d = ref_logprobs - logp;  or 0 when neither is given
 *     loss = mean over the rows with valid != 0 of  -objective + kl_coef * KL - entropy_coef * entropy       (0 when there is none)
 * Rows with valid == 0 are not looked at and get a zero gradient.  stats: float [4], the means of -objective, KL, entropy and of (ratio outside
 * the clip range).  d_logits of the rows: NULL, or written with the gradient of scale * loss; scale: device float, NULL = 1.
 * resume: not 0 for a second call on the same rows and workspace, whose first one had scale = NULL and a d_logits: the workspace's count of valid rows
 * is used again, and bit 1 says that d_logits is the first call's own, so that nothing is to be done where *scale is 1. */
struct procgen_amd_policy {
    const float *old_logprobs, *adv;              /* [rows] */
    const uint8_t *valid;                         /* [rows] or NULL */
    const void *ref_logits;
    long long ref_outer_stride, ref_inner_stride;
    const float *ref_logprobs;
    float clip_low, clip_high, kl_coef, entropy_coef;
    const float *scale;
    float *loss, *stats;                          /* both NULL: only the gradient */
    int resume;                                   /* 0, 1, or 1 | 2 */
};
/* the graph capture that the stream is in: its id, 0 when there is none, -1 when the runtime cannot say.  (bit 1 of resume holds within one capture, or
 * for one call outside of any: a replay of the second call alone would find what its last run left in d_logits.) */
LIBENV_API long long procgen_amd_capture_id(void *stream);
LIBENV_API int procgen_amd_policy_loss(const struct procgen_amd_rows *rows, const struct procgen_amd_policy *policy, int device, void *stream);

#ifdef __cplusplus
}
#endif
#endif
