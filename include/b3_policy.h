/*
 * b3_policy.h - what a policy needs next to the environments' step, on the
 * device buffers that the environments fill (b3_hover.h).
 *
 *   log probabilities   of the taken actions under rows of logits, with the
 *                       rows' entropies, their best alternatives, and the
 *                       gradient
 *   advantages          of a rollout's rewards, values and terminals
 *   AdamW               one step over all of a policy's tensors, moments in
 *                       32 or 8 bits, with the clip of the gradients' norm
 *   linear attention    a memory over a rollout's steps that decays and ends
 *                       with the episode, its gradient, and one step of it
 *   norm                root mean square, with the residual's addition, its
 *                       gradient, and an output in 8 bits
 *   Muon                one step over a policy's matrices, orthogonalised
 *
 * The reference leaves these to the trainer (docs/RL_LIBRARY.md).
 * Conventions are the engine's (b3_engine.h): hipError_t returns, no abort;
 * hipErrorInvalidValue for bad arguments with nothing launched; no work is a
 * successful no-op; the *_gpu functions enqueue on `stream` without
 * allocating or synchronising, on the current device, whose memory every
 * pointer is.  b3_adamw_create and b3_muon_create alone allocate.  Arrays need the alignment
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

/* ---- linear attention ---- */

#define B3_MAX_HEAD 128
#define B3_MAX_SEQUENCES (1 << 22)

/* q and k [steps, envs, heads, key], v [steps, envs, heads, value]: strides
 * in elements from step to step, environment to environment and head to
 * head; a head's elements are contiguous.  q, k and v may be NULL for no steps.
 * `decay` [heads] is in [0, 1] (a state becomes NaN by others).  `starts` is NULL
 * or [steps, envs], nonzero where a step begins an episode: what lies before is
 * dropped (not multiplied by 0: its NaN stay there).  `state` [envs, heads, key,
 * value], contiguous, is what the first step finds; NULL: zeros. */
typedef struct B3Attention {
    int64_t steps, envs, heads;  /* envs * heads at most B3_MAX_SEQUENCES */
    int key, value;              /* 1 .. B3_MAX_HEAD */
    int type;                    /* of q, k, v, the result and gradients */
    const void *q, *k, *v;
    int64_t q_stride[3], k_stride[3], v_stride[3];
    const float* decay;
    const void* starts;
    int starts_type;             /* B3_F32 or B3_U8 */
    int64_t starts_stride[2];
    const float* state;
    double scale;
} B3Attention;

/* Bytes of workspace of either direction (0 for many sequences or few steps). */
size_t b3_linear_attention_workspace(const B3Attention* attention, int backward);

/*   S_t = decay S_{t-1} + k_t^T v_t (without the first term where an episode
 *   starts), out_t = scale q_t S_t
 * out [steps, envs, heads, value], contiguous; last_state (NULL: not wanted)
 * like `state`, and apart from it: S after the last step.  States and sums are
 * in 32 bits; with bfloat16 the products q_t k_s of steps of a chunk, and the
 * state, are read to 16 bits where they give out.  Such products overflow past
 * 2^127, also where v is small; what an infinity comes to may be NaN. */
hipError_t b3_linear_attention_gpu(const B3Attention* attention, void* out, float* last_state, void* workspace,
    size_t workspace_bytes, hipStream_t stream);

/* Gradients from those of out (strides as q's) and, unless NULL, of
 * last_state (contiguous); d_q, d_k and d_v are contiguous, d_state is like
 * `state`.  NULL results are not wanted. */
hipError_t b3_linear_attention_backward_gpu(const B3Attention* attention, const void* d_out,
    const int64_t d_out_stride[3], const float* d_last_state, void* d_q, void* d_k, void* d_v, float* d_state,
    void* workspace, size_t workspace_bytes, hipStream_t stream);

/* One step of every environment (steps is 1), attention->state in place.
 * out [envs, heads, value], contiguous. */
hipError_t b3_linear_attention_step_gpu(const B3Attention* attention, float* state, void* out, hipStream_t stream);

/* ---- norm ---- */

/* Rows of `width` contiguous elements, each array's rows its stride apart (in
 * elements, at least `width`).  h = x + residual (NULL: none), in 32 bits, and
 * so are the squares: those of elements past 2^63 overflow. */
typedef struct B3Norm {
    int64_t rows, width;         /* width 1 .. 2^21 */
    int type;                    /* of x, residual and what comes of them */
    const void* x;
    int64_t x_stride;
    const void* residual;
    int64_t residual_stride;
    const void* weight;          /* [width], NULL: ones */
    int weight_type;             /* `type`, or B3_F32 */
    double eps;                  /* at least 0 */
} B3Norm;

/* out = weight h / sqrt(mean of h^2 + eps); with a residual, sum = h; root
 * [rows] = 1 / sqrt(mean of h^2 + eps).  out and sum are contiguous; sum
 * and root may be NULL. */
hipError_t b3_rms_norm_gpu(const B3Norm* norm, void* out, void* sum, float* root, hipStream_t stream);

/* The same, out as OCP e4m3 numbers, rounded to the nearest, with the exponent
 * byte b of a scale 2^(b - 127) for every 32 of a row: the least power with
 * which none passes 448.  out [rows, width] and scale [rows, ceil(width / 32)]
 * are contiguous.  What is not finite becomes NaN. */
hipError_t b3_rms_norm_8bit_gpu(const B3Norm* norm, unsigned char* out, unsigned char* scale, void* sum,
    hipStream_t stream);

/* The values that such numbers stand for, in `type`. */
hipError_t b3_values_of_8bit_gpu(int64_t rows, int64_t width, const unsigned char* in, const unsigned char* scale,
    void* out, int type, hipStream_t stream);

/* Gradients: d_x (also the residual's) and d_weight, of weight_type (NULL: not
 * wanted), from those of out and sum (NULL: zero).  `norm` is the forward
 * pass's; where the sum is in 32 bits, x may be it, without a residual. */
size_t b3_rms_norm_backward_workspace(int64_t rows, int64_t width);
hipError_t b3_rms_norm_backward_gpu(const B3Norm* norm, const float* root, const void* d_out, int64_t d_out_stride,
    const void* d_sum, int64_t d_sum_stride, void* d_x, void* d_weight, void* workspace, size_t workspace_bytes,
    hipStream_t stream);

/* ---- Muon ---- */

/* A matrix's weights: rows x columns contiguous elements. */
typedef struct B3MuonMatrix {
    void* param;
    int type;                    /* B3_F32, B3_F16 or B3_BF16 */
    int64_t rows, columns;
    double weight_decay;
} B3MuonMatrix;

/* Flat arrays of b3_muon_size() elements, laid out as AdamW's: `momentum`, and
 * `master`, the 32-bit copies of 16-bit weights (NULL keeps none), with the
 * same meaning. */
typedef struct B3MuonState {
    float* momentum;
    float* master;
} B3MuonState;

typedef struct B3MuonConfig {
    double momentum;             /* in [0, 1) */
    int nesterov;
    int newton_schulz;           /* steps, 1 .. 16 */
    double eps;                  /* over 0 */
} B3MuonConfig;

typedef struct B3Muon B3Muon;

int64_t b3_muon_size(const B3MuonMatrix* matrices, int count);

/* As b3_adamw_create.  Allocates what a step works in too. */
hipError_t b3_muon_create(B3Muon** out, const B3MuonMatrix* matrices, int count, B3MuonState state,
    B3MuonConfig config);

/* One step of the matrices that have a gradient, given as b3_adamw_step_gpu's:
 *   m = momentum m + g          u = g + momentum m with nesterov, else m
 *   x = u / (|u| + eps), its transpose where rows > columns
 *   newton_schulz times: a = x x^T, x = 3.4445 x + (-4.775 a + 2.0315 a a) x
 *   w = w (1 - lr decay) - lr sqrt(max(1, rows / columns)) x
 * Numbers of a product are kept to 22 bits (to 32 where a matrix is at most 64 x
 * 256), its sums are in 32.  Steps of one optimizer must follow one another on
 * the device. */
hipError_t b3_muon_step_gpu(B3Muon* optimizer, const void* const* grads, const int* grad_types, double lr,
    hipStream_t stream);

/* Waits for the device; the weights and the state are left.  NULL is a no-op. */
hipError_t b3_muon_destroy(B3Muon* optimizer);

#ifdef __cplusplus
}
#endif
#endif
