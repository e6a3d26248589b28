/*
 * b3_adamw.hip - AdamW over many tensors at once, moments in 32 or 8 bits,
 * with the clip of the gradients' norm (include/b3_policy.h).
 *
 * The tensors are cut into chunks of kChunk elements, a workgroup each; a
 * table of chunks made once says whose.  A launch takes the gradients of up
 * to kBatch tensors as kernel arguments, so a step copies nothing to the
 * device.  With a clip the norm is summed first: chunk by chunk, then all
 * chunks in one order.
 */
#include "policy_common.h"

#include <stdlib.h>
#include <string.h>

namespace b3p {

constexpr int kThreads = 256;
constexpr int kVector = 4;                       // elements a thread loads at once
constexpr int kChunk = 4096;
constexpr int kTurns = kChunk / (kThreads * kVector);
constexpr int kBatch = 160;                      // tensors to a launch: 4,000 bytes of arguments
constexpr int kGroup = 32;                       // 8-bit moments: elements to a scale
constexpr int kSumThreads = 1024;

/* A tensor of the table. */
struct Tensor {
    void* param;
    int64_t at;                                  // of its moments in the flat arrays
    int64_t numel;
    int type;
};

/* What a step says of each tensor of a launch. */
struct StepArgs {
    const void* grad[kBatch];                    // NULL: not stepped
    float size[kBatch];                          // lr / (1 - beta1^t)
    float root[kBatch];                          // 1 / sqrt(1 - beta2^t)
    float keep[kBatch];                          // 1 - lr weight_decay
    uint32_t key[kBatch];                        // of the 8-bit moments' rounding
    uint8_t grad_type[kBatch];
};
static_assert(sizeof(StepArgs) <= 4096 - 96, "kernel arguments");

struct Moments {
    void* exp_avg;
    void* exp_avg_sq;
    uint8_t* exp_avg_scale;
    uint8_t* exp_avg_sq_scale;
    float* master;
};

struct Rates {
    float beta1, beta2, rest1, rest2, eps;       // rest = 1 - beta, rounded once
};

}  // namespace b3p

struct B3AdamW {
    int device, count, bits;
    int64_t size, chunks;
    B3AdamWConfig config;
    b3p::Moments moments;
    b3p::Tensor* tensors;                        // device
    int2* chunk;                                 // device: tensor, chunk of it
    float* partial;                              // device: sums of squares of the chunks
    float* scale;                                // device: the clip's factor
    int64_t* first;                              // host: a tensor's first chunk; count + 1
    int64_t* steps;                              // host
    B3AdamWTensor* given;                        // host
};

namespace b3p {
namespace {

inline __host__ __device__ uint32_t mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x7feb352du;
    x ^= x >> 15;
    x *= 0x846ca68bu;
    return x ^ x >> 16;
}

template <typename T>
__device__ void load(const T* p, int64_t i, int64_t n, float x[kVector]) {
    if (i + kVector <= n) {
        Pack<T, kVector> v = *(const Pack<T, kVector>*)(p + i);
#pragma unroll
        for (int k = 0; k < kVector; k++) x[k] = to_float(v.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < kVector; k++) x[k] = i + k < n ? to_float(p[i + k]) : 0.0f;
    }
}

template <typename T>
__device__ void store(T* p, int64_t i, int64_t n, const float x[kVector]) {
    if (i + kVector <= n) {
        Pack<T, kVector> v;
#pragma unroll
        for (int k = 0; k < kVector; k++) v.v[k] = (T)x[k];
        *(Pack<T, kVector>*)(p + i) = v;
    } else {
#pragma unroll
        for (int k = 0; k < kVector; k++)
            if (i + k < n) p[i + k] = (T)x[k];
    }
}

/* ---- 8-bit moments: four e4m3 bytes of a thread, 8 threads to a scale ---- */

__device__ void unpack(uint32_t codes, uint8_t scale, float x[kVector]) {
    float s = __uint_as_float((uint32_t)scale << 23);
    x[0] = __builtin_amdgcn_cvt_f32_fp8(codes, 0) * s;
    x[1] = __builtin_amdgcn_cvt_f32_fp8(codes, 1) * s;
    x[2] = __builtin_amdgcn_cvt_f32_fp8(codes, 2) * s;
    x[3] = __builtin_amdgcn_cvt_f32_fp8(codes, 3) * s;
}

/* The exponent byte of the least power of two with which none of the group's
 * finite values passes 448 (7/8 of 2^9). */
__device__ uint32_t group_scale(const float x[kVector]) {
    float most = 0;
#pragma unroll
    for (int k = 0; k < kVector; k++) {
        float a = fabsf(x[k]);
        most = a <= 3.4028235e38f ? fmaxf(most, a) : most;
    }
    for (int d = 1; d < kGroup / kVector; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
    uint32_t b = __float_as_uint(most);
    int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u);
    return e < 1 ? 1 : e;
}

/* x on the group's scale as an e4m3 number, still in 32 bits: one of its two
 * neighbours by 16 random bits, or the nearest. */
template <bool RANDOM, bool ROOT>
__device__ float round_code(float x, float inverse, uint32_t random) {
    float y = fabsf(x) * inverse;
    if (RANDOM) {
        float low = y < 0.015625f ? 0.015625f : 0.0f;       // below 2^-6 the steps stay 2^-9
        uint32_t b = __float_as_uint(y + low) + (random << 4);
        float z = __uint_as_float(b & ~0xfffffu) - low;
        y = y <= 448.0f ? z : NAN;
    } else {
        y = y <= 448.0f ? y : NAN;
    }
    if (ROOT && y < 0.001953125f && x > 0.0f) y = 0.001953125f;
    return ROOT ? y : copysignf(y, x);
}

template <bool RANDOM, bool ROOT>
__device__ uint32_t pack(const float x[kVector], uint32_t scale, const uint32_t random[kVector]) {
    float inverse = __uint_as_float((254u - scale) << 23);
    float y[kVector];
#pragma unroll
    for (int k = 0; k < kVector; k++)
        y[k] = round_code<RANDOM, ROOT>(x[k], inverse, ROOT ? random[k] >> 16 : random[k] & 0xffffu);
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
}

__device__ void store_codes(uint8_t* codes, uint8_t* scales, int64_t i, uint32_t code, uint32_t scale) {
    *(uint32_t*)(codes + i) = code;
    if (i % kGroup == 0) scales[i / kGroup] = (uint8_t)scale;
}

/* ---- the step ---- */

template <typename P, typename G, bool MASTER, int BITS>
__device__ void step_chunk(const Tensor& t, int64_t from, const G* grad, const Moments& mo, const Rates& k, float clip,
    float size, float root_scale, float keep, uint32_t key) {
    for (int turn = 0; turn < kTurns; turn++) {
        const int64_t i = from + (int64_t)(turn * kThreads + (int)threadIdx.x) * kVector;
        /* whole groups of 8-bit moments go on together */
        if (i / kGroup * kGroup >= t.numel) return;
        const int64_t at = t.at + i;
        float g[kVector], w[kVector], m[kVector], v[kVector];
        load(grad, i, t.numel, g);
        if (MASTER)
            load(mo.master + t.at, i, t.numel, w);
        else
            load((const P*)t.param, i, t.numel, w);
        if (BITS == 32) {
            load((const float*)mo.exp_avg + t.at, i, t.numel, m);
            load((const float*)mo.exp_avg_sq + t.at, i, t.numel, v);
        } else {
            unpack(*(const uint32_t*)((const uint8_t*)mo.exp_avg + at), mo.exp_avg_scale[at / kGroup], m);
            unpack(*(const uint32_t*)((const uint8_t*)mo.exp_avg_sq + at), mo.exp_avg_sq_scale[at / kGroup], v);
        }
        float root[kVector];
#pragma unroll
        for (int j = 0; j < kVector; j++) {
            float gc = g[j] * clip;
            float old = BITS == 32 ? v[j] : v[j] * v[j];
            m[j] = m[j] * k.beta1 + gc * k.rest1;
            v[j] = old * k.beta2 + gc * gc * k.rest2;
            root[j] = sqrtf(v[j]);
            w[j] = w[j] * keep - m[j] * size / (root[j] * root_scale + k.eps);
        }
        store((P*)t.param, i, t.numel, w);
        if (MASTER) store(mo.master + t.at, i, t.numel, w);
        if (BITS == 32) {
            store((float*)mo.exp_avg + t.at, i, t.numel, m);
            store((float*)mo.exp_avg_sq + t.at, i, t.numel, v);
        } else {
            uint32_t random[kVector];
#pragma unroll
            for (int j = 0; j < kVector; j++)
                random[j] = mix((uint32_t)(at + j) ^ key ^ mix((uint32_t)((at + j) >> 32)));
            uint32_t sm = group_scale(m), sr = group_scale(root);
            store_codes((uint8_t*)mo.exp_avg, mo.exp_avg_scale, at, pack<true, false>(m, sm, random), sm);
            store_codes((uint8_t*)mo.exp_avg_sq, mo.exp_avg_sq_scale, at, pack<true, true>(root, sr, random), sr);
        }
    }
}

template <typename P, bool MASTER, int BITS>
__device__ void step_typed(const Tensor& t, int64_t from, const void* grad, bool float_grad, const Moments& mo,
    const Rates& k, float clip, float size, float root_scale, float keep, uint32_t key) {
    if (float_grad)
        step_chunk<P, float, MASTER, BITS>(t, from, (const float*)grad, mo, k, clip, size, root_scale, keep, key);
    else
        step_chunk<P, P, MASTER, BITS>(t, from, (const P*)grad, mo, k, clip, size, root_scale, keep, key);
}

template <int BITS>
__global__ __launch_bounds__(kThreads) void aw_step(StepArgs a, int base, int64_t first, const int2* chunk,
    const Tensor* tensors, Moments mo, Rates k, const float* scale) {
    const int2 c = chunk[first + blockIdx.x];
    const int at = c.x - base;
    const void* grad = a.grad[at];
    if (!grad) return;
    const Tensor t = tensors[c.x];
    const int64_t from = (int64_t)c.y * kChunk;
    const float clip = scale ? *scale : 1.0f, size = a.size[at], root = a.root[at], keep = a.keep[at];
    const uint32_t key = a.key[at];
    const bool fg = a.grad_type[at] == B3_F32;
    if (t.type == B3_F32)
        step_chunk<float, float, false, BITS>(t, from, (const float*)grad, mo, k, clip, size, root, keep, key);
    else if (t.type == B3_BF16 && mo.master)
        step_typed<__bf16, true, BITS>(t, from, grad, fg, mo, k, clip, size, root, keep, key);
    else if (t.type == B3_BF16)
        step_typed<__bf16, false, BITS>(t, from, grad, fg, mo, k, clip, size, root, keep, key);
    else if (mo.master)
        step_typed<_Float16, true, BITS>(t, from, grad, fg, mo, k, clip, size, root, keep, key);
    else
        step_typed<_Float16, false, BITS>(t, from, grad, fg, mo, k, clip, size, root, keep, key);
}

/* ---- the norm ---- */

template <typename G>
__device__ float square_chunk(const G* grad, int64_t from, int64_t n) {
    float sum = 0;
#pragma unroll
    for (int turn = 0; turn < kTurns; turn++) {
        const int64_t i = from + (int64_t)(turn * kThreads + (int)threadIdx.x) * kVector;
        float g[kVector];
        load(grad, i, n, g);
#pragma unroll
        for (int j = 0; j < kVector; j++) sum += g[j] * g[j];
    }
    return sum;
}

__global__ __launch_bounds__(kThreads) void aw_squares(StepArgs a, int base, int64_t first, const int2* chunk,
    const Tensor* tensors, float* partial) {
    __shared__ float lds[kThreads / kWave];
    const int2 c = chunk[first + blockIdx.x];
    const int at = c.x - base;
    const void* grad = a.grad[at];
    float sum = 0;
    if (grad) {
        const int64_t n = tensors[c.x].numel, from = (int64_t)c.y * kChunk;
        const int type = a.grad_type[at];
        if (type == B3_F32)
            sum = square_chunk((const float*)grad, from, n);
        else if (type == B3_BF16)
            sum = square_chunk((const __bf16*)grad, from, n);
        else
            sum = square_chunk((const _Float16*)grad, from, n);
    }
    for (int d = kWave / 2; d > 0; d /= 2) sum += __shfl_xor(sum, d);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0;
        for (int w = 0; w < kThreads / kWave; w++) sum += lds[w];
        partial[first + blockIdx.x] = sum;
    }
}

/* The sums of the chunks, added in 64 bits: there may be 10^5 of them. */
__global__ __launch_bounds__(kSumThreads) void aw_norm(const float* partial, int64_t chunks, float max_norm, float* norm,
    float* scale) {
    __shared__ double lds[kSumThreads / kWave];
    double sum = 0;
    for (int64_t i = threadIdx.x; i < chunks; i += kSumThreads) sum += partial[i];
    for (int d = kWave / 2; d > 0; d /= 2) sum += __shfl_xor(sum, d);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0;
        for (int w = 0; w < kSumThreads / kWave; w++) sum += lds[w];
        float n = (float)sqrt(sum), s = max_norm / (n + 1e-6f);
        *norm = n;
        *scale = s > 1.0f ? 1.0f : s;            // a NaN norm stays one
    }
}

/* ---- 8-bit moments in and out: a thread to four elements ---- */

__global__ __launch_bounds__(kThreads) void aw_moments(Moments mo, int64_t size, __bf16* exp_avg, __bf16* exp_avg_sq) {
    const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kVector;
    if (i >= size) return;
    float m[kVector], r[kVector];
    unpack(*(const uint32_t*)((const uint8_t*)mo.exp_avg + i), mo.exp_avg_scale[i / kGroup], m);
    unpack(*(const uint32_t*)((const uint8_t*)mo.exp_avg_sq + i), mo.exp_avg_sq_scale[i / kGroup], r);
    for (int k = 0; k < kVector; k++) r[k] *= r[k];
    store(exp_avg, i, size, m);
    store(exp_avg_sq, i, size, r);
}

__global__ __launch_bounds__(kThreads) void aw_load(Moments mo, int64_t size, const float* exp_avg,
    const float* exp_avg_sq) {
    const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kVector;
    if (i >= size) return;                        // a multiple of 256: groups stay whole
    float m[kVector], r[kVector];
    load(exp_avg, i, size, m);
    load(exp_avg_sq, i, size, r);
    for (int k = 0; k < kVector; k++) r[k] = sqrtf(r[k]);
    const uint32_t none[kVector] = {0, 0, 0, 0};
    uint32_t sm = group_scale(m), sr = group_scale(r);
    store_codes((uint8_t*)mo.exp_avg, mo.exp_avg_scale, i, pack<false, false>(m, sm, none), sm);
    store_codes((uint8_t*)mo.exp_avg_sq, mo.exp_avg_sq_scale, i, pack<false, true>(r, sr, none), sr);
}

bool valid(const B3AdamWTensor* tensors, int count) {
    if (count < 0 || (count && !tensors)) return false;
    int64_t total = 0;
    for (int i = 0; i < count; i++) {
        const B3AdamWTensor& t = tensors[i];
        if (!is_float_type(t.type) || t.numel < 0 || t.numel > (int64_t)1 << 40 || (t.numel && !t.param)
                || !(t.weight_decay >= 0))
            return false;
        total += t.numel;
        if (total > (int64_t)1 << 40) return false;
    }
    return true;
}

int64_t segment(int64_t numel) { return ceil_div(numel, B3_ADAMW_SEGMENT) * B3_ADAMW_SEGMENT; }

hipError_t on_device(const B3AdamW* o) {
    int device;
    hipError_t err = hipGetDevice(&device);
    return err != hipSuccess ? err : device == o->device ? hipSuccess : hipErrorInvalidDevice;
}

}  // namespace
}  // namespace b3p

using namespace b3p;

extern "C" {

int64_t b3_adamw_size(const B3AdamWTensor* tensors, int count) {
    if (!valid(tensors, count)) return -1;
    int64_t size = 0;
    for (int i = 0; i < count; i++) size += segment(tensors[i].numel);
    return size;
}

hipError_t b3_adamw_destroy(B3AdamW* o) {
    if (!o) return hipSuccess;
    hipError_t first = hipSuccess;
    void* bufs[4] = {o->tensors, o->chunk, o->partial, o->scale};
    for (void* p : bufs) {
        hipError_t err = p ? hipFree(p) : hipSuccess;
        if (first == hipSuccess) first = err;
    }
    free(o->first);
    free(o->steps);
    free(o->given);
    free(o);
    return first;
}

hipError_t b3_adamw_create(B3AdamW** out, const B3AdamWTensor* tensors, int count, B3AdamWState state,
        B3AdamWConfig config) {
    if (!out) return hipErrorInvalidValue;
    *out = NULL;
    if (!valid(tensors, count) || (state.bits != 8 && state.bits != 32) || !(config.beta1 >= 0 && config.beta1 < 1)
            || !(config.beta2 >= 0 && config.beta2 < 1) || !(config.eps >= 0))
        return hipErrorInvalidValue;
    int64_t size = b3_adamw_size(tensors, count), chunks = 0;
    if (size && (!state.exp_avg || !state.exp_avg_sq
            || (state.bits == 8 && (!state.exp_avg_scale || !state.exp_avg_sq_scale))))
        return hipErrorInvalidValue;
    for (int i = 0; i < count; i++) chunks += ceil_div(tensors[i].numel, kChunk);
    if (chunks > 0x7fffffff) return hipErrorInvalidValue;
    B3AdamW* o = (B3AdamW*)calloc(1, sizeof(B3AdamW));
    if (!o) return hipErrorOutOfMemory;
    o->count = count;
    o->bits = state.bits;
    o->size = size;
    o->chunks = chunks;
    o->config = config;
    o->moments = Moments{state.exp_avg, state.exp_avg_sq, state.exp_avg_scale, state.exp_avg_sq_scale, state.master};
    o->first = (int64_t*)calloc((size_t)count + 1, sizeof(int64_t));
    o->steps = (int64_t*)calloc((size_t)count + 1, sizeof(int64_t));
    o->given = (B3AdamWTensor*)calloc((size_t)count + 1, sizeof(B3AdamWTensor));
    Tensor* table = (Tensor*)calloc((size_t)count + 1, sizeof(Tensor));
    int2* chunk = (int2*)calloc((size_t)chunks + 1, sizeof(int2));
    hipError_t err = o->first && o->steps && o->given && table && chunk ? hipGetDevice(&o->device) : hipErrorOutOfMemory;
    if (err == hipSuccess) {
        int64_t at = 0, c = 0;
        for (int i = 0; i < count; i++) {
            o->given[i] = tensors[i];
            table[i] = Tensor{tensors[i].param, at, tensors[i].numel, tensors[i].type};
            at += segment(tensors[i].numel);
            o->first[i] = c;
            for (int64_t j = 0; j < ceil_div(tensors[i].numel, kChunk); j++) chunk[c++] = make_int2(i, (int)j);
        }
        o->first[count] = c;
    }
    if (err == hipSuccess) err = hipMalloc((void**)&o->tensors, ((size_t)count + 1) * sizeof(Tensor));
    if (err == hipSuccess) err = hipMalloc((void**)&o->chunk, ((size_t)chunks + 1) * sizeof(int2));
    if (err == hipSuccess) err = hipMalloc((void**)&o->partial, ((size_t)chunks + 1) * sizeof(float));
    if (err == hipSuccess) err = hipMalloc((void**)&o->scale, sizeof(float));
    if (err == hipSuccess)
        err = hipMemcpy(o->tensors, table, ((size_t)count + 1) * sizeof(Tensor), hipMemcpyHostToDevice);
    if (err == hipSuccess) err = hipMemcpy(o->chunk, chunk, ((size_t)chunks + 1) * sizeof(int2), hipMemcpyHostToDevice);
    if (err == hipSuccess) err = hipDeviceSynchronize();
    free(table);
    free(chunk);
    if (err != hipSuccess) {
        (void)b3_adamw_destroy(o);
        return err;
    }
    *out = o;
    return hipSuccess;
}

hipError_t b3_adamw_step_gpu(B3AdamW* o, const void* const* grads, const int* grad_types, double lr, double max_norm,
        float* norm, hipStream_t stream) {
    if (!o || (o->count && !grads) || !(lr >= 0) || !(max_norm >= 0) || (max_norm > 0 && !norm))
        return hipErrorInvalidValue;
    for (int i = 0; grad_types && i < o->count; i++)
        if (grads[i] && grad_types[i] != o->given[i].type && grad_types[i] != B3_F32) return hipErrorInvalidValue;
    hipError_t err = on_device(o);
    if (err != hipSuccess) return err;
    const B3AdamWConfig& cf = o->config;
    const Rates rates = {(float)cf.beta1, (float)cf.beta2, (float)(1 - cf.beta1), (float)(1 - cf.beta2), (float)cf.eps};
    StepArgs a;
    for (int pass = max_norm > 0 ? 0 : 1; pass < 2; pass++) {
        int64_t t_last = -1;
        float size = 0, root = 0;
        for (int base = 0; base < o->count; base += kBatch) {
            const int n = o->count - base < kBatch ? o->count - base : kBatch;
            const int64_t first = o->first[base], blocks = o->first[base + n] - first;
            memset((void*)&a, 0, sizeof(a));
            for (int j = 0; j < n; j++) {
                const int i = base + j;
                a.grad[j] = grads[i];
                a.grad_type[j] = (uint8_t)(grad_types ? grad_types[i] : o->given[i].type);
                if (pass == 0 || !grads[i]) continue;
                const int64_t t = ++o->steps[i];
                if (t != t_last) {
                    size = (float)(lr / (1 - pow(cf.beta1, (double)t)));
                    root = (float)(1 / sqrt(1 - pow(cf.beta2, (double)t)));
                    t_last = t;
                }
                a.size[j] = size;
                a.root[j] = root;
                a.keep[j] = (float)(1 - lr * o->given[i].weight_decay);
                a.key[j] = mix((uint32_t)t * 0x9e3779b9u + cf.seed);
            }
            if (blocks == 0) continue;
            if (pass == 0)
                aw_squares<<<(unsigned)blocks, kThreads, 0, stream>>>(a, base, first, o->chunk, o->tensors, o->partial);
            else if (o->bits == 32)
                aw_step<32><<<(unsigned)blocks, kThreads, 0, stream>>>(a, base, first, o->chunk, o->tensors, o->moments,
                    rates, max_norm > 0 ? o->scale : NULL);
            else
                aw_step<8><<<(unsigned)blocks, kThreads, 0, stream>>>(a, base, first, o->chunk, o->tensors, o->moments,
                    rates, max_norm > 0 ? o->scale : NULL);
            if ((err = hipGetLastError()) != hipSuccess) return err;
        }
        if (pass == 0) {
            aw_norm<<<1, kSumThreads, 0, stream>>>(o->partial, o->chunks, (float)max_norm, norm, o->scale);
            if ((err = hipGetLastError()) != hipSuccess) return err;
        }
    }
    return hipSuccess;
}

int64_t b3_adamw_steps(const B3AdamW* o, int tensor) {
    return o && tensor >= 0 && tensor < o->count ? o->steps[tensor] : -1;
}

hipError_t b3_adamw_set_steps(B3AdamW* o, int tensor, int64_t steps) {
    if (!o || tensor < 0 || tensor >= o->count || steps < 0) return hipErrorInvalidValue;
    o->steps[tensor] = steps;
    return hipSuccess;
}

hipError_t b3_adamw_moments_gpu(const B3AdamW* o, void* exp_avg, void* exp_avg_sq, hipStream_t stream) {
    if (!o || o->bits != 8 || (o->size && (!exp_avg || !exp_avg_sq))) return hipErrorInvalidValue;
    hipError_t err = on_device(o);
    if (err != hipSuccess || o->size == 0) return err;
    aw_moments<<<(unsigned)ceil_div(o->size, kThreads * kVector), kThreads, 0, stream>>>(o->moments, o->size,
        (__bf16*)exp_avg, (__bf16*)exp_avg_sq);
    return hipGetLastError();
}

hipError_t b3_adamw_load_moments_gpu(B3AdamW* o, const float* exp_avg, const float* exp_avg_sq, hipStream_t stream) {
    if (!o || o->bits != 8 || (o->size && (!exp_avg || !exp_avg_sq))) return hipErrorInvalidValue;
    hipError_t err = on_device(o);
    if (err != hipSuccess || o->size == 0) return err;
    aw_load<<<(unsigned)ceil_div(o->size, kThreads * kVector), kThreads, 0, stream>>>(o->moments, o->size, exp_avg,
        exp_avg_sq);
    return hipGetLastError();
}

}  // extern "C"
