/*
 * b3_advantages.hip - generalised advantage estimates of a rollout
 * (include/b3_policy.h).
 *
 *   A_t = d_t + a_t A_{t+1},  d_t = r_t + gamma V_{t+1} - V_t,
 *   a_t = gamma lambda; a terminal at t drops the terms of t + 1.
 */
#include "policy_common.h"

namespace b3p {
namespace {

constexpr int kThreads = 256;

template <typename V, typename D>
__global__ __launch_bounds__(kThreads) void adv_columns(B3Rollout g, float gamma, float decay) {
    const int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (n >= g.envs) return;
    const float* rewards = g.rewards + n * g.rewards_stride[1];
    const V* values = (const V*)g.values + n * g.values_stride[1];
    const D* terminals = (const D*)g.terminals + n * g.terminals_stride[1];
    float after = to_float(((const V*)g.last_values)[n * g.last_values_stride]), adv = 0;
    for (int64_t t = g.steps - 1; t >= 0; t--) {
        float v = to_float(values[t * g.values_stride[0]]);
        float r = rewards[t * g.rewards_stride[0]];
        adv = terminals[t * g.terminals_stride[0]] != 0 ? r - v : r + gamma * after - v + decay * adv;
        g.advantages[n * g.out_stride[1] + t * g.out_stride[0]] = adv;
        g.returns[n * g.out_stride[1] + t * g.out_stride[0]] = adv + v;
        after = v;
    }
}

bool valid(const B3Rollout& g) {
    if (g.steps < 0 || g.envs < 0 || !is_float_type(g.values_type)) return false;
    if (g.terminals_type != B3_F32 && g.terminals_type != B3_U8) return false;
    if (g.steps == 0 || g.envs == 0) return true;
    return g.envs <= INT64_MAX / g.steps && g.rewards && g.values && g.last_values && g.terminals && g.advantages
        && g.returns && g.envs <= (int64_t)kThreads * 0x7fffffff;
}

template <typename V>
void launch(const B3Rollout& g, float gamma, float decay, hipStream_t stream) {
    unsigned grid = (unsigned)ceil_div(g.envs, kThreads);
    if (g.terminals_type == B3_F32)
        adv_columns<V, float><<<grid, kThreads, 0, stream>>>(g, gamma, decay);
    else
        adv_columns<V, uint8_t><<<grid, kThreads, 0, stream>>>(g, gamma, decay);
}

}  // namespace
}  // namespace b3p

using namespace b3p;

extern "C" {

size_t b3_advantages_workspace(int64_t, int64_t) { return 0; }

hipError_t b3_advantages_gpu(const B3Rollout* g, double gamma, double lambda, void* workspace, size_t workspace_bytes,
        hipStream_t stream) {
    if (!g || !valid(*g) || !(gamma >= 0 && gamma <= 1) || !(lambda >= 0 && lambda <= 1)
            || workspace_bytes < b3_advantages_workspace(g->steps, g->envs))
        return hipErrorInvalidValue;
    if (g->steps == 0 || g->envs == 0) return hipSuccess;
    (void)workspace;
    if (g->values_type == B3_F32)
        launch<float>(*g, (float)gamma, (float)(gamma * lambda), stream);
    else if (g->values_type == B3_F16)
        launch<_Float16>(*g, (float)gamma, (float)(gamma * lambda), stream);
    else
        launch<__bf16>(*g, (float)gamma, (float)(gamma * lambda), stream);
    return hipGetLastError();
}

}  // extern "C"
