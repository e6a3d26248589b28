/*
 * b3_linear_attention.hip - linear attention with a decay for each head, cut
 * where episodes start, its gradient, and one step of it
 * (include/b3_policy.h).
 *
 *   S_t = decay S_{t-1} + k_t^T v_t, or k_t^T v_t where an episode starts
 *   out_t = scale q_t S_t
 *
 * With G_t = scale q_t^T do_t + decay G_{t+1} (nothing of t + 1 where an
 * episode starts there) the gradients are dq_t = scale do_t S_t^T,
 * dk_t = v_t G_t^T and dv_t = k_t G_t: each a sum of the same form over the
 * earlier or the later steps, with the arrays in other places.  One kernel
 * does all four.
 */
#include "policy_common.h"

namespace b3p {
namespace {

constexpr int kThreads = 256;

/* out_p = `reach` q_p (decay^p E + sums over p' <= p of the episode of
 * `update` decay^(p - p') k_p'^T v_p'), and the state that is left,
 * decay^steps E + sums of `update` decay^(steps - p') k_p'^T v_p'.  Places p
 * follow the steps, or go from the last one back. */
struct Mix {
    const void *q, *k, *v;
    void* out;
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];   // place, environment, head
    int key, value;
    float reach, update;
    const char* starts;                          // of place 0 (which has none where `back`), or NULL
    int64_t starts_stride[2];                    // in bytes
    const float* enter;                          // E, NULL: zeros
    float* leave;                                // NULL: not wanted
    int64_t state_row, state_col;                // of both, in elements
    bool enter_early;                            // E is a step earlier: decayed before place 0
    bool leave_early;                            // the state is left a step earlier: not decayed after the last place
    const char* leave_starts;                    // [environments], dropped where nonzero; or NULL
    int64_t leave_starts_stride;
};

constexpr int kRoles = 3;
struct Job {
    Mix mix[kRoles];
    int64_t steps, envs, heads;
    const float* decay;
    int starts_type;
};

__device__ __forceinline__ bool started(const char* p, int type) {
    return type == B3_F32 ? *(const float*)p != 0.0f : *(const unsigned char*)p != 0;
}

/* A head's decay: NaN outside of [0, 1]. */
__device__ __forceinline__ float decay_of(const float* decay, int64_t head) {
    const float d = decay[head];
    return d >= 0.0f && d <= 1.0f ? d : NAN;
}

/* A workgroup to a sequence, place after place: thread t holds column t % 128
 * of one half of the state's rows. */
template <typename T>
__global__ __launch_bounds__(kThreads) void la_places(Job j) {
    constexpr int kRows = B3_MAX_HEAD / 2;
    __shared__ float q[B3_MAX_HEAD], k[B3_MAX_HEAD], v[B3_MAX_HEAD], half[B3_MAX_HEAD];
    const Mix& m = j.mix[blockIdx.y];
    const int64_t env = blockIdx.x / j.heads, head = blockIdx.x % j.heads;
    const int col = threadIdx.x % B3_MAX_HEAD, top = threadIdx.x / B3_MAX_HEAD * kRows;
    const float decay = decay_of(j.decay, head);
    const int64_t state = (env * j.heads + head) * m.key * m.value;
    float s[kRows];
#pragma unroll
    for (int r = 0; r < kRows; r++) {
        const bool in = top + r < m.key && col < m.value;
        s[r] = in && m.enter ? m.enter[state + (top + r) * m.state_row + col * m.state_col] : 0.0f;
        if (m.enter_early) s[r] *= decay;
    }
    for (int64_t p = 0; p < j.steps; p++) {
        const bool start = m.starts && (p || m.enter_early)
            && started(m.starts + p * m.starts_stride[0] + env * m.starts_stride[1], j.starts_type);
        __syncthreads();
        if ((int)threadIdx.x < B3_MAX_HEAD) {
            const int c = threadIdx.x;
            q[c] = c < m.key ? to_float(((const T*)m.q)[p * m.q_stride[0] + env * m.q_stride[1] + head * m.q_stride[2] + c]) : 0;
            k[c] = c < m.key ? m.update * to_float(((const T*)m.k)[p * m.k_stride[0] + env * m.k_stride[1] + head * m.k_stride[2] + c]) : 0;
            v[c] = c < m.value ? to_float(((const T*)m.v)[p * m.v_stride[0] + env * m.v_stride[1] + head * m.v_stride[2] + c]) : 0;
        }
        __syncthreads();
        float o = 0;
#pragma unroll
        for (int r = 0; r < kRows; r++) {
            s[r] = (start ? 0.0f : s[r]) + k[top + r] * v[col];
            o += q[top + r] * s[r];
            if (p + 1 < j.steps || !m.leave_early) s[r] *= decay;
        }
        if (top) half[col] = o;
        __syncthreads();
        if (!top && col < m.value && m.out)
            ((T*)m.out)[p * m.out_stride[0] + env * m.out_stride[1] + head * m.out_stride[2] + col] = (T)(m.reach * (o + half[col]));
    }
    if (!m.leave) return;
    const bool drop = m.leave_starts && started(m.leave_starts + env * m.leave_starts_stride, j.starts_type);
#pragma unroll
    for (int r = 0; r < kRows; r++)
        if (top + r < m.key && col < m.value)
            m.leave[state + (top + r) * m.state_row + col * m.state_col] = drop ? 0.0f : s[r];
}

/* ---- one step ---- */

struct StepJob {
    B3Attention g;
    float scale;
    float* state;
    void* out;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void la_step(StepJob j) {
    constexpr int kRows = B3_MAX_HEAD / 2;
    __shared__ float half[B3_MAX_HEAD];
    const B3Attention& g = j.g;
    const int64_t env = blockIdx.x / g.heads, head = blockIdx.x % g.heads;
    const int col = threadIdx.x % B3_MAX_HEAD, top = threadIdx.x / B3_MAX_HEAD * kRows;
    const float decay = decay_of(g.decay, head);
    const bool start = g.starts
        && started((const char*)g.starts + env * g.starts_stride[1] * (g.starts_type == B3_F32 ? 4 : 1), g.starts_type);
    float* s = j.state + (env * g.heads + head) * g.key * g.value + col;
    const T* q = (const T*)g.q + env * g.q_stride[1] + head * g.q_stride[2];
    const T* k = (const T*)g.k + env * g.k_stride[1] + head * g.k_stride[2];
    const float v = col < g.value ? to_float(((const T*)g.v)[env * g.v_stride[1] + head * g.v_stride[2] + col]) : 0.0f;
    float o = 0;
    for (int r = top; r < top + kRows && r < g.key && col < g.value; r++) {
        const float x = (start ? 0.0f : decay * s[r * g.value]) + to_float(k[r]) * v;
        s[r * g.value] = x;
        o += to_float(q[r]) * x;
    }
    if (top) half[col] = o;
    __syncthreads();
    if (!top && col < g.value) ((T*)j.out)[(env * g.heads + head) * g.value + col] = (T)(j.scale * (o + half[col]));
}

/* ---- launches ---- */

bool valid(const B3Attention* g) {
    if (!g || !is_float_type(g->type) || g->steps < 0 || g->envs < 0 || g->heads < 0 || g->key < 1 || g->key > B3_MAX_HEAD
            || g->value < 1 || g->value > B3_MAX_HEAD || !(g->scale == g->scale))
        return false;
    if (g->starts && g->starts_type != B3_F32 && g->starts_type != B3_U8) return false;
    if (g->envs == 0 || g->heads == 0) return true;
    if (g->envs > 0x7fffffff || g->heads > 0x7fffffff || g->steps > 0x7fffffff || g->envs * g->heads > kMostBlocks) return false;
    return g->steps == 0 || (g->q && g->k && g->v && g->decay);
}

int64_t size_of(int type) { return type == B3_F32 ? 4 : 2; }

void copy3(int64_t to[3], const int64_t from[3]) {
    for (int i = 0; i < 3; i++) to[i] = from[i];
}

void contiguous(int64_t to[3], const B3Attention& g, int dims) {
    to[2] = dims;
    to[1] = g.heads * dims;
    to[0] = g.envs * to[1];
}

/* The arrays of places from the last step back. */
template <typename P>
void turn(P*& p, int64_t stride[3], const B3Attention& g) {
    if (p) p = (P*)((char*)p + (g.steps - 1) * stride[0] * size_of(g.type));
    stride[0] = -stride[0];
}

void backwards_arrays(Mix& m, const B3Attention& g) {
    turn(m.q, m.q_stride, g);
    turn(m.k, m.k_stride, g);
    turn(m.v, m.v_stride, g);
    turn(m.out, m.out_stride, g);
}

Job job_of(const B3Attention& g) {
    Job j = {};
    j.steps = g.steps;
    j.envs = g.envs;
    j.heads = g.heads;
    j.decay = g.decay;
    j.starts_type = g.starts_type;
    return j;
}

Mix forwards(const B3Attention& g) {
    Mix m = {};
    const int64_t size = g.starts_type == B3_F32 ? 4 : 1;
    m.reach = (float)g.scale;
    m.update = 1;
    m.starts = (const char*)g.starts;
    m.starts_stride[0] = g.starts_stride[0] * size;
    m.starts_stride[1] = g.starts_stride[1] * size;
    m.enter = g.state;
    m.enter_early = m.leave_early = g.steps > 0;
    return m;
}

/* Before place p of the way back an episode starts where step steps - p's does. */
Mix backwards(const B3Attention& g, const float* d_last) {
    Mix m = forwards(g);
    m.reach = 1;
    m.update = (float)g.scale;
    if (m.starts && g.steps) {
        m.leave_starts = m.starts;
        m.leave_starts_stride = m.starts_stride[1];
        m.starts += g.steps * m.starts_stride[0];
        m.starts_stride[0] = -m.starts_stride[0];
    }
    m.enter = d_last;
    m.enter_early = m.leave_early = false;
    return m;
}

template <typename T>
hipError_t launch(const Job& j, int roles, hipStream_t stream) {
    la_places<T><<<dim3((unsigned)(j.envs * j.heads), roles), kThreads, 0, stream>>>(j);
    return hipGetLastError();
}

hipError_t launch(const Job& j, int roles, int type, hipStream_t stream) {
    return type == B3_F32 ? launch<float>(j, roles, stream) : type == B3_F16 ? launch<_Float16>(j, roles, stream)
                                                                            : launch<__bf16>(j, roles, stream);
}

}  // namespace
}  // namespace b3p

using namespace b3p;

extern "C" {

size_t b3_linear_attention_workspace(const B3Attention* g, int backward) { return 0; }

hipError_t b3_linear_attention_gpu(const B3Attention* g, void* out, float* last_state, void* workspace,
        size_t workspace_bytes, hipStream_t stream) {
    if (!valid(g)) return hipErrorInvalidValue;
    if (g->envs == 0 || g->heads == 0 || (g->steps == 0 && !last_state)) return hipSuccess;
    if (g->steps && !out) return hipErrorInvalidValue;
    Job j = job_of(*g);
    Mix m = forwards(*g);
    m.q = g->q;
    m.k = g->k;
    m.v = g->v;
    m.out = out;
    copy3(m.q_stride, g->q_stride);
    copy3(m.k_stride, g->k_stride);
    copy3(m.v_stride, g->v_stride);
    contiguous(m.out_stride, *g, g->value);
    m.key = g->key;
    m.value = g->value;
    m.leave = last_state;
    m.state_row = g->value;
    m.state_col = 1;
    j.mix[0] = m;
    return launch(j, 1, g->type, stream);
}

hipError_t b3_linear_attention_backward_gpu(const B3Attention* g, const void* d_out, const int64_t d_out_stride[3],
        const float* d_last_state, void* d_q, void* d_k, void* d_v, float* d_state, void* workspace,
        size_t workspace_bytes, hipStream_t stream) {
    if (!valid(g)) return hipErrorInvalidValue;
    if (g->envs == 0 || g->heads == 0) return hipSuccess;
    if (g->steps && (!d_out || !d_out_stride)) return hipErrorInvalidValue;
    Job j = job_of(*g);
    Mix a = forwards(*g);                        // d_q: S^T, of d_out, v and k
    a.q = d_out;
    a.k = g->v;
    a.v = g->k;
    if (d_out_stride) copy3(a.q_stride, d_out_stride);
    copy3(a.k_stride, g->v_stride);
    copy3(a.v_stride, g->k_stride);
    a.key = g->value;
    a.value = g->key;
    a.out = d_q;
    contiguous(a.out_stride, *g, g->key);
    a.state_row = 1;
    a.state_col = g->value;
    Mix b = backwards(*g, d_last_state);         // d_k: G^T, of v, d_out and q
    b.q = g->v;
    b.k = d_out;
    b.v = g->q;
    copy3(b.q_stride, g->v_stride);
    if (d_out_stride) copy3(b.k_stride, d_out_stride);
    copy3(b.v_stride, g->q_stride);
    b.key = g->value;
    b.value = g->key;
    b.out = d_k;
    contiguous(b.out_stride, *g, g->key);
    b.state_row = 1;
    b.state_col = g->value;
    Mix c = backwards(*g, d_last_state);         // d_v: G, of k, q and d_out
    c.q = g->k;
    c.k = g->q;
    c.v = d_out;
    copy3(c.q_stride, g->k_stride);
    copy3(c.k_stride, g->q_stride);
    if (d_out_stride) copy3(c.v_stride, d_out_stride);
    c.key = g->key;
    c.value = g->value;
    c.out = d_v;
    contiguous(c.out_stride, *g, g->value);
    c.state_row = g->value;
    c.state_col = 1;
    c.leave = d_state;
    if (g->steps) {
        backwards_arrays(b, *g);
        backwards_arrays(c, *g);
    }
    int roles = 0;
    if (d_q && g->steps) j.mix[roles++] = a;
    if (d_k && g->steps) j.mix[roles++] = b;
    if (d_v || d_state) j.mix[roles++] = c;
    return roles ? launch(j, roles, g->type, stream) : hipSuccess;
}

hipError_t b3_linear_attention_step_gpu(const B3Attention* g, float* state, void* out, hipStream_t stream) {
    if (!valid(g) || g->steps != 1) return hipErrorInvalidValue;
    if (g->envs == 0 || g->heads == 0) return hipSuccess;
    if (!state || !out) return hipErrorInvalidValue;
    const StepJob j = {*g, (float)g->scale, state, out};
    const unsigned blocks = (unsigned)(g->envs * g->heads);
    if (g->type == B3_F32) la_step<float><<<blocks, kThreads, 0, stream>>>(j);
    else if (g->type == B3_F16) la_step<_Float16><<<blocks, kThreads, 0, stream>>>(j);
    else la_step<__bf16><<<blocks, kThreads, 0, stream>>>(j);
    return hipGetLastError();
}

}  // extern "C"
