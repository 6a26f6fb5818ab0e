/*
 * gw_learn.h — C-ABI of the policy operators: what stands between a policy's
 * logits and the engine's action rows, and between a rollout's slabs
 * (gw_rollout) and the policy's gradient.
 *
 *   gw_policy_sample        logits -> action rows (what gw_step / gw_rollout
 *                           take), their log-probabilities, the entropy
 *   gw_policy_loss          the clipped policy loss with a KL term and an
 *                           entropy term, its gradient by the logits, or both
 *   gw_recurrence[_backward]  h[t] = gate[t] h[t-1] + x[t] over the steps of a
 *                           fragment (a policy's memory, discounted returns)
 *   gw_advantages           the recurrence over a rollout's slabs: generalized
 *                           advantages and value targets
 *   gw_fragment_marks       where the episodes of a rollout's slabs end
 *
 * No reference counterpart: the reference hands its dicts to RLlib, which does
 * this work on the host (train.py:10, trainers/base.py:82-192).
 *
 * Every pointer is a device buffer of the caller's on the current HIP device
 * unless it says "host"; the work is put on `stream` and nothing waits for it.
 * No call allocates, and none keeps anything for the next, so calls on several
 * streams and captured graphs need only workspaces of their own.  Counts are
 * rows or elements, never bytes, except where a name says bytes.
 * GW_E_INVALID: an argument that cannot be run; nothing was launched, and
 * gw_learn_last_error() (this thread's) says which.
 */
#ifndef GW_LEARN_H
#define GW_LEARN_H

#include <stdint.h>
#include "gw_engine.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define GW_T_F32  0
#define GW_T_F16  1
#define GW_T_BF16 2

#define GW_MAX_HEADS 256

/* The heads of a policy: head d is a softmax over sizes[d] choices, whose
   logits stand side by side in a row (n_choices = the sum of the sizes), and
   choice i of it is action value low[d] + i in column slots[d] of an action
   row of act_dim ints.  Columns that no head has are written 0.  Host
   arrays, read during the call.                                            */
typedef struct gw_policy_heads {
    int32_t n_heads;               /* 1..GW_MAX_HEADS                        */
    int32_t act_dim;               /* >= 1                                   */
    const int32_t* sizes;          /* >= 1 each                              */
    const int32_t* low;            /* low[d] + sizes[d] <= 2^31              */
    const int32_t* slots;          /* 0..act_dim-1, each at most once        */
} gw_policy_heads;

/* A choice exists unless choice_mask has 0 for it or its logit is -inf.  Row
   r uses mask row r % mask_rows (mask_rows divides n_rows: the lanes of an
   env, one row for all, or a row each).  What stands at masked places is never used
   (NaN and infinities included).  A head without a choice takes part in
   nothing: its action is low[d], its log-probability and entropy 0.        */

/* Per row and head the choice with the largest float(logit) + noise (noise
   NULL: the largest logit); ties go to the lowest choice.  With Gumbel noise
   that draws from the softmax.
     logits   [n_rows][n_choices] of dtype, rows ld elements apart
     noise    float [n_rows][n_choices], rows side by side, or NULL
     actions  int32 [n_rows][act_dim]
     logp     float [n_rows]: the sum over the heads of the choices'
              log-probabilities; entropy float [n_rows] (both may be NULL)   */
gw_status gw_policy_sample(const gw_policy_heads* heads, int32_t dtype, int64_t n_rows,
                           const void* logits, int64_t ld, const float* noise,
                           const uint8_t* choice_mask, int64_t mask_rows,
                           int32_t* actions, float* logp, float* entropy, void* stream);

/* With p, q the softmax of logits and ref, L the log-probability of the row's
   action under p (sums over the heads), ratio = exp(L - old_logp):
     loss = 1/M sum over valid rows of
            - min(ratio A, clamp(ratio, 1 - clip_low, 1 + clip_high) A)
            + kl_coef KL(q || p) - entropy_coef H(p)
     loss     float [1];  stats  float [5]: the means over valid rows of the
              policy term, KL, entropy and clipped rows, and M.  Both or
              neither NULL
     logp     float [n_rows]: L (0 for rows not valid); NULL: not wanted
     grad     [n_rows][n_choices] of dtype, rows side by side: dloss/dlogits
              times grad_scale (and times *upstream); 0 for rows not valid
              and choices that do not exist; NULL: not wanted
     M        = denominator if that is > 0, else *denominator_at if not NULL,
              else the number of valid rows; with M = 0 everything is 0
     ref      NULL: no KL term.  valid: NULL: every row
   An action outside its head, or whose choice does not exist, has
   probability 0: L = -inf, ratio 0, no gradient from the policy term.
   What stands in rows not valid is never used (NaN, infinities and any action
   included), but it may be read.  The sums over rows are made in double in a
   fixed order: the same inputs give the same bits.
   workspace: gw_policy_loss_workspace(n_rows) bytes, 8-byte aligned, free
   for other use once the call's work is done.                              */
int64_t   gw_policy_loss_workspace(int64_t n_rows);
gw_status gw_policy_loss(const gw_policy_heads* heads, int32_t dtype, int64_t n_rows,
                         const void* logits, int64_t ld, const void* ref, int64_t ld_ref,
                         const int32_t* actions, const float* advantage, const float* old_logp,
                         const uint8_t* valid, const uint8_t* choice_mask, int64_t mask_rows,
                         float clip_low, float clip_high, float kl_coef, float entropy_coef,
                         float denominator, const float* denominator_at,
                         float grad_scale, const float* upstream,
                         float* loss, float* stats, float* logp, void* grad,
                         void* workspace, int64_t workspace_bytes, void* stream);

/* h[t] = (cut[t] ? 0 : gate[t] h[t-1]) + x[t] for t = 0..n_steps-1, h[-1] =
   state; reverse != 0: t runs from the last step to the first, h[t+1] in the
   place of h[t-1], state before the last step.  Sums are held in float.
     x, h     [n_steps][n] of dtype
     gate     [n_steps][n / gate_span] of gate_dtype (dtype or GW_T_F32): channel
              c uses gate c / gate_span; NULL: gate_value everywhere
     cut      uint8 [n_steps][n / cut_span] or NULL: set where an episode begins.  (Of a
              fragment's marks, below: not where END stands but a step behind it, or, where
              the env is reset by a step of its own, behind RESET)
     state    float [n] or NULL (zeros);  last  float [n]: h after the last
              step done, or NULL
     carry    float [ceil(n_steps / GW_RECURRENCE_SEGMENT)][n] or NULL: h
              before each segment of steps (in the order of the recurrence),
              which gw_recurrence_backward takes
   gate_span and cut_span divide n.
   workspace: gw_recurrence_workspace(...) bytes, 8-byte aligned (may be 0). */
#define GW_RECURRENCE_SEGMENT 16
int64_t   gw_recurrence_workspace(int64_t n_steps, int64_t n);
gw_status gw_recurrence(int32_t dtype, int32_t gate_dtype, int64_t n_steps, int64_t n,
                        const void* x, const void* gate, int64_t gate_span, float gate_value,
                        const uint8_t* cut, int64_t cut_span, const float* state, int32_t reverse,
                        void* h, float* last, float* carry,
                        void* workspace, int64_t workspace_bytes, void* stream);

/* Gradients of gw_recurrence by x, gate and state, from those of h (dh, of
   dtype) and last (dlast); either may be NULL (zeros).  dgate: of gate_dtype,
   summed over the channels that share a gate (in a fixed order), 0 where cut;
   dgate and dstate may be NULL.                                            */
int64_t   gw_recurrence_backward_workspace(int64_t n_steps, int64_t n, int64_t gate_span);
gw_status gw_recurrence_backward(int32_t dtype, int32_t gate_dtype, int64_t n_steps, int64_t n,
                                 const void* x, const void* gate, int64_t gate_span, float gate_value,
                                 const uint8_t* cut, int64_t cut_span, const float* carry, int32_t reverse,
                                 const void* dh, const float* dlast,
                                 void* dx, void* dgate, float* dstate,
                                 void* workspace, int64_t workspace_bytes, void* stream);

/* What a step of an env was, in a fragment (gw_rollout) */
#define GW_MARK_END       1  /* the episode ended with it, nothing follows    */
#define GW_MARK_TRUNCATED 2  /* the horizon ended it: its observation is real */
#define GW_MARK_RESET     4  /* no step: the env was reset (NEXT_STEP)        */
#define GW_MARK_SKIP      8  /* the env raised somewhere in the fragment      */

/* marks uint8 [n_steps][n_envs] from a rollout's all_done slab, the '__all__'
   before it (all_done_in uint8 [n_envs]; NULL: none set), each env's steps
   before it (gw_get_state; int32 [n_envs]; NULL: zeros), the horizon (0:
   none) and the auto-reset mode (1 SAME_STEP, 2 NEXT_STEP, as gw_rollout).  With SAME_STEP the observation behind a horizon
   is the next episode's, so it is marked GW_MARK_END.  err (uint32 [n_envs], the flags that
   the rollout set, or NULL): envs with flags, whose reward and done rows are not all written, get
   GW_MARK_SKIP in every step.                                               */
gw_status gw_fragment_marks(int64_t n_steps, int64_t n_envs, const uint8_t* all_done,
                            const uint8_t* all_done_in, const int32_t* steps, const uint32_t* err,
                            int32_t horizon, int32_t autoreset, uint8_t* marks, void* stream);

/* Generalized advantages over a rollout's slabs ([n_steps][n_envs][n_lanes]):
   a lane acted in a step if it was not done before it (live uint8
   [n_envs][n_lanes] before step 0; afterwards done of the step before, or
   the episode just begun), acts[lane] != 0 (NULL: all) and the step is not marked
   RESET or SKIP; valid uint8 says so.  For such steps
     delta = reward + (done or END ? 0 : gamma value[t+1]) - value[t]
     advantage = delta + gamma lam (done, END or TRUNCATED ? 0 : advantage[t+1])
     target = advantage + value[t]
   and 0, 0 for the others.
     reward   double or float [n_steps][E][A] (reward_f64)
     value    [n_steps + 1][E][A] of dtype: of the observations before each
              step, and after the last
     done uint8 [n_steps][E][A], marks uint8 [n_steps][E]
     advantage, target float, valid uint8, all [n_steps][E][A]
   workspace as gw_recurrence_workspace(n_steps, n_envs * n_lanes).          */
gw_status gw_advantages(int32_t dtype, int32_t reward_f64, int64_t n_steps, int64_t n_envs, int64_t n_lanes,
                        const void* reward, const void* value, const uint8_t* done, const uint8_t* marks,
                        const uint8_t* live, const uint8_t* acts, float gamma, float lam,
                        float* advantage, float* target, uint8_t* valid,
                        void* workspace, int64_t workspace_bytes, void* stream);

const char* gw_learn_last_error(void);
int32_t     gw_learn_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* GW_LEARN_H */
