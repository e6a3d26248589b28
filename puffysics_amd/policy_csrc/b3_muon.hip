/*
 * b3_muon.hip - Muon's step over a policy's matrices (include/b3_policy.h).
 *
 *   m = momentum m + g, u = g + momentum m, x = u / (|u| + eps)
 *   x = a x + (b y + c y y) x, y = x x^T, some times; then w moves by x
 *
 * A matrix is worked on with its shorter side first, so that y is as small as
 * it can be.
 */
#include "policy_common.h"

#include <stdlib.h>

namespace b3p {

constexpr int kThreads = 256;
constexpr int kTile = 32;
constexpr int kSumBlocks = 256;
constexpr double kA = 3.4445, kB = -4.7750, kC = 2.0315;

}  // namespace b3p

struct B3Muon {
    int device, count;
    B3MuonConfig config;
    B3MuonState state;
    B3MuonMatrix* given;                         // host
    int64_t* at;                                 // host: of each in the flat arrays
    float* work;                                 // device: x and its next, y and its polynomial
    double* partial;                             // device
    int64_t most, side;                          // elements of the largest matrix, of its y
};

namespace b3p {
namespace {

template <typename T>
__device__ __forceinline__ float element(const void* p, int64_t i) { return to_float(((const T*)p)[i]); }

__device__ __forceinline__ float element(const void* p, int type, int64_t i) {
    return type == B3_F32 ? element<float>(p, i) : type == B3_F16 ? element<_Float16>(p, i) : element<__bf16>(p, i);
}

__global__ __launch_bounds__(kThreads) void mu_momentum(const void* grad, int type, float* momentum, int64_t rows,
    int64_t columns, float keep, int nesterov, float* x, double* partial) {
    __shared__ double lds[kThreads];
    const bool turned = rows > columns;
    double sum = 0;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * columns; i += (int64_t)gridDim.x * kThreads) {
        const float g = element(grad, type, i), m = keep * momentum[i] + g, u = nesterov ? g + keep * m : m;
        momentum[i] = m;
        x[turned ? i % columns * rows + i / columns : i] = u;
        sum += (double)u * u;
    }
    lds[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < kThreads; i++) sum += lds[i];
    partial[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kThreads) void mu_scale(float* x, int64_t n, const double* partial, int partials, float eps) {
    double sum = 0;
    for (int i = 0; i < partials; i++) sum += partial[i];
    const float size = (float)sqrt(sum) + eps;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) x[i] /= size;
}

/* out[m][n] = p add + q left[m][k] right, where right is [k][n], or [n][k] with TURNED. */
template <bool TURNED>
__global__ __launch_bounds__(kThreads) void mu_product(const float* left, const float* right, const float* add, float* out,
    int64_t m, int64_t n, int64_t k, float p, float q) {
    __shared__ float a[kTile][kTile + 1], b[kTile][kTile + 1];
    const int col = threadIdx.x % kTile, row = threadIdx.x / kTile;
    constexpr int kRows = kThreads / kTile;
    const int64_t j0 = (int64_t)blockIdx.x * kTile, i0 = (int64_t)blockIdx.y * kTile;
    float sum[kTile / kRows] = {};
    for (int64_t k0 = 0; k0 < k; k0 += kTile) {
        for (int r = row; r < kTile; r += kRows) {
            a[r][col] = i0 + r < m && k0 + col < k ? left[(i0 + r) * k + k0 + col] : 0.0f;
            if (TURNED)
                b[col][r] = j0 + r < n && k0 + col < k ? right[(j0 + r) * k + k0 + col] : 0.0f;
            else
                b[r][col] = k0 + r < k && j0 + col < n ? right[(k0 + r) * n + j0 + col] : 0.0f;
        }
        __syncthreads();
        for (int i = 0; i < kTile; i++)
#pragma unroll
            for (int r = 0; r < kTile / kRows; r++) sum[r] = __builtin_fmaf(a[row + r * kRows][i], b[i][col], sum[r]);
        __syncthreads();
    }
    for (int r = 0; r < kTile / kRows; r++) {
        const int64_t i = i0 + row + r * kRows, j = j0 + col;
        if (i < m && j < n) out[i * n + j] = q * sum[r] + (add ? p * add[i * n + j] : 0.0f);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void mu_update(T* param, float* master, const float* x, int64_t rows,
    int64_t columns, float keep, float rate) {
    const bool turned = rows > columns;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * columns; i += (int64_t)gridDim.x * kThreads) {
        const T old = param[i];
        float w = to_float(old);
        if (master && to_float((T)master[i]) == w) w = master[i];
        w = w * keep - rate * x[turned ? i % columns * rows + i / columns : i];
        if (master) master[i] = w;
        param[i] = (T)w;
    }
}

bool valid(const B3MuonMatrix* matrices, int count) {
    if (count < 0 || (count && !matrices)) return false;
    int64_t total = 0;
    for (int i = 0; i < count; i++) {
        const B3MuonMatrix& t = matrices[i];
        if (!is_float_type(t.type) || t.rows < 0 || t.columns < 0 || t.rows > 0x7fffffff || t.columns > 0x7fffffff
                || (t.rows && t.columns > ((int64_t)1 << 40) / t.rows) || (t.rows * t.columns && !t.param)
                || !(t.weight_decay >= 0))
            return false;
        total += t.rows * t.columns;
        if (total > (int64_t)1 << 40) return false;
    }
    return true;
}

int by_address(const void* a, const void* b) {
    const uintptr_t x = (uintptr_t)((const B3MuonMatrix*)a)->param, y = (uintptr_t)((const B3MuonMatrix*)b)->param;
    return (x > y) - (x < y);
}

/* Whether two of the matrices that have elements overlap; `sorted` has room for all. */
bool overlap(const B3MuonMatrix* matrices, int count, B3MuonMatrix* sorted) {
    int n = 0;
    for (int i = 0; i < count; i++)
        if (matrices[i].rows * matrices[i].columns) sorted[n++] = matrices[i];
    qsort(sorted, (size_t)n, sizeof(B3MuonMatrix), by_address);
    for (int i = 1; i < n; i++) {
        const B3MuonMatrix& b = sorted[i - 1];
        if ((uintptr_t)b.param + (uintptr_t)(b.rows * b.columns) * (b.type == B3_F32 ? 4 : 2) > (uintptr_t)sorted[i].param)
            return true;
    }
    return false;
}

int64_t segment(int64_t numel) { return ceil_div(numel, B3_ADAMW_SEGMENT) * B3_ADAMW_SEGMENT; }

}  // namespace
}  // namespace b3p

using namespace b3p;

extern "C" {

int64_t b3_muon_size(const B3MuonMatrix* matrices, int count) {
    if (!valid(matrices, count)) return -1;
    int64_t size = 0;
    for (int i = 0; i < count; i++) size += segment(matrices[i].rows * matrices[i].columns);
    return size;
}

hipError_t b3_muon_destroy(B3Muon* o) {
    if (!o) return hipSuccess;
    hipError_t first = hipSuccess;
    void* bufs[2] = {o->work, o->partial};
    for (void* p : bufs) {
        hipError_t err = p ? hipFree(p) : hipSuccess;
        if (first == hipSuccess) first = err;
    }
    free(o->given);
    free(o->at);
    free(o);
    return first;
}

hipError_t b3_muon_create(B3Muon** out, const B3MuonMatrix* matrices, int count, B3MuonState state, B3MuonConfig config) {
    if (!out) return hipErrorInvalidValue;
    *out = NULL;
    const int64_t size = b3_muon_size(matrices, count);
    if (size < 0 || (size && !state.momentum) || !(config.momentum >= 0 && config.momentum < 1) || !(config.eps > 0)
            || config.newton_schulz < 1 || config.newton_schulz > 16)
        return hipErrorInvalidValue;
    B3Muon* o = (B3Muon*)calloc(1, sizeof(B3Muon));
    if (!o) return hipErrorOutOfMemory;
    o->count = count;
    o->config = config;
    o->state = state;
    o->given = (B3MuonMatrix*)calloc((size_t)count + 1, sizeof(B3MuonMatrix));
    o->at = (int64_t*)calloc((size_t)count + 1, sizeof(int64_t));
    hipError_t err = !(o->given && o->at) ? hipErrorOutOfMemory
        : overlap(matrices, count, o->given) ? hipErrorInvalidValue : hipGetDevice(&o->device);
    if (err == hipSuccess) {
        int64_t at = 0;
        for (int i = 0; i < count; i++) {
            const B3MuonMatrix& t = o->given[i] = matrices[i];
            const int64_t m = t.rows < t.columns ? t.rows : t.columns;
            o->at[i] = at;
            at += segment(t.rows * t.columns);
            if (t.rows * t.columns > o->most) o->most = t.rows * t.columns;
            if (m * m > o->side) o->side = m * m;
        }
        err = hipMalloc((void**)&o->work, (size_t)(2 * (o->most + o->side) + 1) * sizeof(float));
    }
    if (err == hipSuccess) err = hipMalloc((void**)&o->partial, kSumBlocks * sizeof(double));
    if (err != hipSuccess) {
        (void)b3_muon_destroy(o);
        return err;
    }
    *out = o;
    return hipSuccess;
}

hipError_t b3_muon_step_gpu(B3Muon* o, const void* const* grads, const int* grad_types, double lr, hipStream_t stream) {
    if (!o || (o->count && !grads) || !(lr >= 0)) return hipErrorInvalidValue;
    for (int i = 0; grad_types && i < o->count; i++)
        if (grads[i] && grad_types[i] != o->given[i].type && grad_types[i] != B3_F32) return hipErrorInvalidValue;
    int device;
    hipError_t err = hipGetDevice(&device);
    if (err != hipSuccess || device != o->device) return err != hipSuccess ? err : hipErrorInvalidDevice;
    for (int i = 0; i < o->count; i++) {
        const B3MuonMatrix& t = o->given[i];
        const int64_t numel = t.rows * t.columns, m = t.rows < t.columns ? t.rows : t.columns, n = numel ? numel / m : 0;
        if (!grads[i] || !numel) continue;
        float *x = o->work, *next = x + o->most, *y = next + o->most, *poly = y + o->side;
        const int blocks = (int)(ceil_div(numel, kThreads) < kSumBlocks ? ceil_div(numel, kThreads) : kSumBlocks);
        mu_momentum<<<blocks, kThreads, 0, stream>>>(grads[i], grad_types ? grad_types[i] : t.type,
            o->state.momentum + o->at[i], t.rows, t.columns, (float)o->config.momentum, o->config.nesterov, x, o->partial);
        mu_scale<<<blocks, kThreads, 0, stream>>>(x, numel, o->partial, blocks, (float)o->config.eps);
        const unsigned gm = (unsigned)ceil_div(m, kTile), gn = (unsigned)ceil_div(n, kTile);
        for (int s = 0; s < o->config.newton_schulz; s++) {
            mu_product<true><<<dim3(gm, gm), kThreads, 0, stream>>>(x, x, NULL, y, m, m, n, 0, 1);
            mu_product<false><<<dim3(gm, gm), kThreads, 0, stream>>>(y, y, y, poly, m, m, m, (float)kB, (float)kC);
            mu_product<false><<<dim3(gn, gm), kThreads, 0, stream>>>(poly, x, x, next, m, n, m, (float)kA, 1);
            float* swap = x;
            x = next;
            next = swap;
        }
        const float keep = (float)(1 - lr * t.weight_decay);
        const float rate = (float)(lr * sqrt(t.rows > t.columns ? (double)t.rows / (double)t.columns : 1.0));
        float* master = o->state.master ? o->state.master + o->at[i] : NULL;
        if (t.type == B3_F32)
            mu_update<float><<<blocks, kThreads, 0, stream>>>((float*)t.param, NULL, x, t.rows, t.columns, keep, rate);
        else if (t.type == B3_F16)
            mu_update<_Float16><<<blocks, kThreads, 0, stream>>>((_Float16*)t.param, master, x, t.rows, t.columns, keep, rate);
        else
            mu_update<__bf16><<<blocks, kThreads, 0, stream>>>((__bf16*)t.param, master, x, t.rows, t.columns, keep, rate);
        if ((err = hipGetLastError()) != hipSuccess) return err;
    }
    return hipSuccess;
}

}  // extern "C"
