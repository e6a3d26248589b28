/*
 * b3_policy.h - what a policy's update needs next to the environments' step,
 * on the device buffers that the environments fill (b3_hover.h).
 *
 *   log probabilities   of the taken actions under rows of logits, with the
 *                       rows' entropies, their best alternatives, and the
 *                       gradient
 *   advantages          of a rollout's rewards, values and terminals
 *   AdamW               one step over all of a policy's tensors, moments in
 *                       32 or 8 bits, with the clip of the gradients' norm
 *
 * The reference leaves these to the trainer (docs/RL_LIBRARY.md).
 * Conventions are the engine's (b3_engine.h): hipError_t returns, no abort;
 * hipErrorInvalidValue for bad arguments with nothing launched; no work is a
 * successful no-op; the *_gpu functions enqueue on `stream` without
 * allocating or synchronising, on the current device, whose memory every
 * pointer is.  b3_adamw_create alone allocates.  Arrays need the alignment
 * of their elements and no more (8-bit moments none), workspaces that of 8
 * bytes.  Results do not depend on the order in which workgroups run.
 */
#ifndef PUFFYSICS_AMD_B3_POLICY_H
#define PUFFYSICS_AMD_B3_POLICY_H

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Types of array elements. */
#define B3_F32 0
#define B3_F16 1
#define B3_BF16 2
#define B3_U8 3

/* ---- log probabilities ---- */

#define B3_MAX_TOP 32

/* Rows of logits x.  A row's elements are contiguous; `row_stride` (in
 * elements, at least `actions`) is between rows.  `mask` is NULL or one byte
 * for each action, nonzero where it is allowed; its rows lie
 * `mask_row_stride` bytes apart (0: one row for all).  An action that is not
 * allowed has probability 0, whatever its logit holds. */
typedef struct B3Logits {
    const void* data;
    int type;                    /* B3_F32, B3_F16 or B3_BF16 */
    int64_t rows;
    int64_t actions;             /* 1 .. 2^21 */
    int64_t row_stride;
    const unsigned char* mask;
    int64_t mask_row_stride;
} B3Logits;

/* Bytes of workspace that b3_log_probs_gpu needs (0 for most sizes). */
size_t b3_log_probs_workspace(int64_t rows, int64_t actions, int top);

/* Per row: log_prob = log p(taken), entropy = -sum p log p, and in `stats`
 * (two floats a row, NULL if no gradient will be asked for) the largest
 * logit and the log of the sum of exp(x - largest).  With top > 0 the `top`
 * largest log probabilities in `top_log_prob` and their actions in
 * `top_action`, each `top` a row, in descending order; ties go to the lowest
 * action, NaN comes first.
 *   taken < 0         padding: log_prob is 0
 *   taken >= actions  log_prob is NaN
 *   no action left    log_prob is -inf, entropy 0, the alternatives -inf
 *   a NaN or +inf among the allowed: all of the row's results are NaN
 * Statistics are kept in 32 bits. */
hipError_t b3_log_probs_gpu(B3Logits logits, const int64_t* taken, float* log_prob, float* entropy, float* stats,
    int top, float* top_log_prob, int64_t* top_action, void* workspace, size_t workspace_bytes, hipStream_t stream);

/* The gradient of the logits, in their type, rows `d_row_stride` elements
 * apart:
 *   d_log_prob * ([j = taken] - p_j) - d_entropy * p_j (log p_j + entropy)
 * 0 where an action is not allowed, and in rows that allow none; a padding
 * row has no first term.  `d_log_prob` and `d_entropy` may be NULL (zero);
 * their elements lie d_*_stride apart (0: one for all rows).  d_logits may
 * be the logits themselves. */
hipError_t b3_log_probs_backward_gpu(B3Logits logits, const int64_t* taken, const float* stats, const float* entropy,
    const float* d_log_prob, int64_t d_log_prob_stride, const float* d_entropy, int64_t d_entropy_stride,
    void* d_logits, int64_t d_row_stride, hipStream_t stream);

/* ---- advantages ---- */

/* A rollout of `steps` steps of `envs` environments.  Each array is given
 * with its strides, in elements, from step to step and from environment to
 * environment. */
typedef struct B3Rollout {
    int64_t steps, envs;
    const float* rewards;
    int64_t rewards_stride[2];
    const void* values;          /* V of the observations before each step */
    int values_type;             /* B3_F32, B3_F16 or B3_BF16 */
    int64_t values_stride[2];
    const void* last_values;     /* V after the last step, of values_type */
    int64_t last_values_stride;
    const void* terminals;       /* nonzero where the step ended an episode */
    int terminals_type;          /* B3_F32 or B3_U8 */
    int64_t terminals_stride[2];
    float* advantages;           /* A */
    float* returns;              /* A + V */
    int64_t out_stride[2];       /* of both; no two elements share a place */
} B3Rollout;

size_t b3_advantages_workspace(int64_t steps, int64_t envs);

/* A_t = r_t + gamma V_{t+1} - V_t + gamma lambda A_{t+1}, where a terminal
 * at t drops the terms of t + 1 (they are not multiplied by 0: a NaN of the
 * next episode stays there).  0 <= gamma, lambda <= 1. */
hipError_t b3_advantages_gpu(const B3Rollout* rollout, double gamma, double lambda, void* workspace,
    size_t workspace_bytes, hipStream_t stream);

/* ---- AdamW ---- */

/* A tensor's weights: `numel` contiguous elements. */
typedef struct B3AdamWTensor {
    void* param;
    int type;                    /* B3_F32, B3_F16 or B3_BF16 */
    int64_t numel;
    double weight_decay;
} B3AdamWTensor;

/* Moments of all tensors lie in flat arrays of b3_adamw_size() elements, in
 * the tensors' order, each from the next multiple of B3_ADAMW_SEGMENT on.
 *   state_bits 32   exp_avg and exp_avg_sq: float
 *   state_bits 8    exp_avg and root_avg_sq (the square root of the second
 *                   moment): OCP e4m3 bytes, with the exponent byte b of a
 *                   scale 2^(b - 127) for every 32 of them
 * `master` holds the 32-bit copies that 16-bit weights are rounded from; NULL
 * keeps none, and the weights are then rounded to the nearest every step.  A
 * weight that is not what its copy rounds to (to the nearest) has been written
 * since, and the next step goes on from the weight. */
#define B3_ADAMW_SEGMENT 256
typedef struct B3AdamWState {
    int bits;
    void* exp_avg;
    void* exp_avg_sq;
    unsigned char* exp_avg_scale;
    unsigned char* exp_avg_sq_scale;
    float* master;
} B3AdamWState;

typedef struct B3AdamWConfig {
    double beta1, beta2, eps;    /* 0 <= beta < 1, eps >= 0 */
    uint32_t seed;               /* of the 8-bit moments' rounding */
} B3AdamWConfig;

typedef struct B3AdamW B3AdamW;

/* Elements of a flat array of the tensors' moments; -1 for bad arguments. */
int64_t b3_adamw_size(const B3AdamWTensor* tensors, int count);

/* The weights and the state stay the caller's, and stay where they are.  No
 * two tensors overlap (hipErrorInvalidValue), nor do weights, state and
 * gradients.  Allocates; synchronises. */
hipError_t b3_adamw_create(B3AdamW** out, const B3AdamWTensor* tensors, int count, B3AdamWState state,
    B3AdamWConfig config);

/* One step of the tensors that have a gradient (grads[i] != NULL), `numel`
 * contiguous elements of the weights' type or, where grad_types[i] says so,
 * of B3_F32:
 *   g' = g min(1, max_norm / (norm + 1e-6))  (max_norm 0: g' = g)
 *   m = beta1 m + (1 - beta1) g'             v = beta2 v + (1 - beta2) g'^2
 *   w = w (1 - lr decay) - lr m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps)
 * norm is the 2-norm of all gradients, written to *norm (device memory; NULL
 * where max_norm is 0).  t counts a tensor's own steps, on the host: a
 * captured step replays the corrections of the step that was captured.
 * 8-bit moments are rounded to one of their two neighbours by random bits
 * that seed, t and place give, and in a captured step the count of the
 * optimizer's captured steps that have run (one that 8 bits hold as it is may
 * fall a step of the grid, by one in 2^16 of the bits); a root over 0 stays
 * over 0.  Steps of one
 * optimizer must follow one another on the device. */
hipError_t b3_adamw_step_gpu(B3AdamW* optimizer, const void* const* grads, const int* grad_types, double lr,
    double max_norm, float* norm, hipStream_t stream);

/* Steps taken by tensor i; -1 for bad arguments. */
int64_t b3_adamw_steps(const B3AdamW* optimizer, int tensor);
hipError_t b3_adamw_set_steps(B3AdamW* optimizer, int tensor, int64_t steps);

/* 8-bit moments as the values they stand for, in bf16 (exact but for what lies
 * below its range): flat arrays of b3_adamw_size() elements. */
hipError_t b3_adamw_moments_gpu(const B3AdamW* optimizer, void* exp_avg, void* exp_avg_sq, hipStream_t stream);

/* float moments (flat arrays) to the 8-bit state, each to the nearest. */
hipError_t b3_adamw_load_moments_gpu(B3AdamW* optimizer, const float* exp_avg, const float* exp_avg_sq,
    hipStream_t stream);

/* Waits for the device; the weights and the state are left.  NULL is a no-op. */
hipError_t b3_adamw_destroy(B3AdamW* optimizer);

#ifdef __cplusplus
}
#endif
#endif
