/*
 * b3_log_probs.hip - log probabilities, entropies and best alternatives of
 * rows of logits, and their gradient (include/b3_policy.h).
 *
 * With m = max x, z = x - m and S = sum exp(z):
 *   log p_j = z_j - log S          H = log S - (sum z exp(z)) / S
 *   dx_j = dlp ([j = taken] - p_j) - dH p_j (log p_j + H)
 */
#include "policy_common.h"

namespace b3p {
namespace {

constexpr int kThreads = 256;

/* A logit, -inf where its action is not allowed. */
template <typename T>
__device__ float logit(const T* row, const unsigned char* mask, int64_t j) {
    return mask && !mask[j] ? -INFINITY : to_float(row[j]);
}

/* Whole numbers in the order of the logits: NaN above +inf, -0 as 0; never 0
 * or 2^32 - 1, so that a key of order and action is neither all zeros nor all
 * ones. */
__device__ uint32_t order_of(float x) {
    if (x != x) return 0xfffffffeu;
    uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename V, typename F>
__device__ V block_reduce(V v, V* lds, F f) {
    lds[threadIdx.x] = v;
    __syncthreads();
    for (int half = kThreads / 2; half > 0; half /= 2) {
        if ((int)threadIdx.x < half) lds[threadIdx.x] = f(lds[threadIdx.x], lds[threadIdx.x + half]);
        __syncthreads();
    }
    v = lds[0];
    __syncthreads();
    return v;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void lp_rows(B3Logits g, const int64_t* taken, float* log_prob, float* entropy,
    float* stats, int top, float* top_log_prob, int64_t* top_action) {
    using T = typename Element<TYPE>::type;
    __shared__ float lds[kThreads];
    __shared__ uint64_t keys[kThreads];
    const int64_t r = blockIdx.x;
    const T* row = (const T*)g.data + r * g.row_stride;
    const unsigned char* mask = g.mask ? g.mask + r * g.mask_row_stride : NULL;
    float most = -INFINITY;
    for (int64_t j = threadIdx.x; j < g.actions; j += kThreads) most = fmaxf(most, logit(row, mask, j));
    most = block_reduce(most, lds, [](float a, float b) { return fmaxf(a, b); });
    const bool none = most == -INFINITY;
    const float m = none ? 0.0f : most;
    float sum = 0, dot = 0;
    for (int64_t j = threadIdx.x; j < g.actions; j += kThreads) {
        float z = logit(row, mask, j) - m, e = expf(z);
        sum += e;
        dot += e == 0.0f ? 0.0f : z * e;
    }
    auto add = [](float a, float b) { return a + b; };
    sum = block_reduce(sum, lds, add);
    dot = block_reduce(dot, lds, add);
    const float log_sum = logf(sum);
    /* a row of NaN alone has no largest logit: its sum is NaN */
    const bool empty = none && sum == 0.0f;
    if (threadIdx.x == 0) {
        int64_t a = taken[r];
        float lp = a < 0 ? 0.0f : a >= g.actions ? NAN : empty ? -INFINITY : logit(row, mask, a) - m - log_sum;
        log_prob[r] = lp;
        entropy[r] = empty ? 0.0f : log_sum - dot / sum;
        if (stats) {
            stats[2 * r] = m;
            stats[2 * r + 1] = log_sum;
        }
    }
    uint64_t below = ~0ull;
    for (int k = 0; k < top; k++) {
        uint64_t best = 0;
        for (int64_t j = threadIdx.x; j < g.actions; j += kThreads) {
            uint64_t key = (uint64_t)order_of(logit(row, mask, j)) << 32 | (uint32_t)~j;
            if (key < below && key > best) best = key;
        }
        best = block_reduce(best, keys, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        below = best;
        if (threadIdx.x == 0) {
            int64_t j = (uint32_t)~(uint32_t)best;
            top_action[r * top + k] = j;
            top_log_prob[r * top + k] = empty ? -INFINITY : logit(row, mask, j) - m - log_sum;
        }
    }
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void lp_backward(B3Logits g, const int64_t* taken, const float* stats,
    const float* entropy, const float* d_log_prob, int64_t dl_stride, const float* d_entropy, int64_t dh_stride,
    void* d_logits, int64_t d_row_stride) {
    using T = typename Element<TYPE>::type;
    const int64_t r = blockIdx.x;
    const T* row = (const T*)g.data + r * g.row_stride;
    const unsigned char* mask = g.mask ? g.mask + r * g.mask_row_stride : NULL;
    T* out = (T*)d_logits + r * d_row_stride;
    const int64_t a = taken[r];
    const float m = stats[2 * r], log_sum = stats[2 * r + 1], h = entropy[r];
    float dl = d_log_prob && a >= 0 ? d_log_prob[r * dl_stride] : 0.0f;
    if (a >= g.actions) dl *= NAN;
    const float dh = d_entropy ? d_entropy[r * dh_stride] : 0.0f;
    const bool empty = log_sum == -INFINITY;
    for (int64_t j = threadIdx.x; j < g.actions; j += kThreads) {
        float x = logit(row, mask, j), lp = x - m - log_sum, p = expf(lp);
        float d = (j == a ? dl : 0.0f) - p * (p == 0.0f ? 0.0f : dl + dh * (lp + h));
        out[j] = (T)(empty || x == -INFINITY ? 0.0f : d);
    }
}

bool valid(const B3Logits& g, const int64_t* taken) {
    return is_float_type(g.type) && g.rows >= 0 && g.rows <= 0x7fffffff && g.actions >= 1 && g.actions <= 1 << 30
        && g.row_stride >= g.actions && (!g.mask || g.mask_row_stride == 0 || g.mask_row_stride >= g.actions)
        && (g.rows == 0 || (g.data && taken));
}

}  // namespace
}  // namespace b3p

using namespace b3p;

extern "C" {

size_t b3_log_probs_workspace(int64_t, int64_t, int) { return 0; }

hipError_t b3_log_probs_gpu(B3Logits g, const int64_t* taken, float* log_prob, float* entropy, float* stats, int top,
        float* top_log_prob, int64_t* top_action, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!valid(g, taken) || top < 0 || top > B3_MAX_TOP || top > g.actions) return hipErrorInvalidValue;
    if (workspace_bytes < b3_log_probs_workspace(g.rows, g.actions, top)) return hipErrorInvalidValue;
    if (g.rows == 0) return hipSuccess;
    if (!log_prob || !entropy || (top && (!top_log_prob || !top_action))) return hipErrorInvalidValue;
    (void)workspace;
    dim3 grid((unsigned)g.rows);
    if (g.type == B3_F32)
        lp_rows<B3_F32><<<grid, kThreads, 0, stream>>>(g, taken, log_prob, entropy, stats, top, top_log_prob, top_action);
    else if (g.type == B3_F16)
        lp_rows<B3_F16><<<grid, kThreads, 0, stream>>>(g, taken, log_prob, entropy, stats, top, top_log_prob, top_action);
    else
        lp_rows<B3_BF16><<<grid, kThreads, 0, stream>>>(g, taken, log_prob, entropy, stats, top, top_log_prob, top_action);
    return hipGetLastError();
}

hipError_t b3_log_probs_backward_gpu(B3Logits g, const int64_t* taken, const float* stats, const float* entropy,
        const float* d_log_prob, int64_t dl_stride, const float* d_entropy, int64_t dh_stride, void* d_logits,
        int64_t d_row_stride, hipStream_t stream) {
    if (!valid(g, taken) || d_row_stride < g.actions || dl_stride < 0 || dh_stride < 0) return hipErrorInvalidValue;
    if (g.rows == 0) return hipSuccess;
    if (!stats || !entropy || !d_logits) return hipErrorInvalidValue;
    dim3 grid((unsigned)g.rows);
    if (g.type == B3_F32)
        lp_backward<B3_F32><<<grid, kThreads, 0, stream>>>(g, taken, stats, entropy, d_log_prob, dl_stride, d_entropy,
            dh_stride, d_logits, d_row_stride);
    else if (g.type == B3_F16)
        lp_backward<B3_F16><<<grid, kThreads, 0, stream>>>(g, taken, stats, entropy, d_log_prob, dl_stride, d_entropy,
            dh_stride, d_logits, d_row_stride);
    else
        lp_backward<B3_BF16><<<grid, kThreads, 0, stream>>>(g, taken, stats, entropy, d_log_prob, dl_stride, d_entropy,
            dh_stride, d_logits, d_row_stride);
    return hipGetLastError();
}

}  // extern "C"
