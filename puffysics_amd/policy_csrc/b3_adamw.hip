/*
 * b3_adamw.hip - AdamW over many tensors at once, moments in 32 or 8 bits,
 * with the clip of the gradients' norm (include/b3_policy.h).
 *
 * The tensors are cut into chunks of kChunk elements; a table of chunks made
 * once says whose each is.  A launch takes the gradients of up to kBatch
 * tensors as kernel arguments, so that a step copies nothing to the device.
 * The step is one pass: a thread's loads of a vector of everything are issued
 * before the first is used.  It is bound by memory (28 bytes a weight in 32
 * bits, 30 of 16-bit weights with copies), and what it moves goes past the
 * caches: 400 million weights in 32 bits take 1,953 us so (5.7 TB/s), and 2,098
 * through them.  With a clip the norm is summed first, by at most kSumBlocks
 * workgroups a launch over their chunks in turn, through the caches, which
 * keep gradients of a moderate size for the step (100 million in bf16 with the
 * clip: 520 us, 545 past them; 60 million in fp32: 290 to 296, 327); few partial
 * sums are added by the step itself, many by a launch of their own.  Sums go
 * in one order always.
 */
#include "policy_common.h"

#include <stdlib.h>

namespace b3p {

constexpr int kThreads = 256;
constexpr int kVector = 4;                       // elements a thread loads at once
constexpr int kChunk = 4096;
constexpr int kSumBlocks = 2048;
constexpr int kBatch = 156;                      // tensors to a launch, see StepLaunch
constexpr size_t kMostArguments = 4096;          // bytes of a launch
constexpr int kGroup = 32;                       // 8-bit moments: elements to a scale
constexpr int kSumThreads = 1024;
constexpr int kFewPartials = kThreads;

/* A tensor of the table. */
struct Tensor {
    void* param;
    int64_t at;                                  // of its moments in the flat arrays
    int64_t numel;
    int type;
};

/* The gradients of a launch's tensors. */
struct Gradients {
    const void* at[kBatch];                      // NULL: not stepped
    uint8_t type[kBatch];
};

/* What a step says of each tensor of a launch. */
struct StepArgs {
    float size[kBatch];                          // lr / (1 - beta1^t)
    float root[kBatch];                          // 1 / sqrt(1 - beta2^t)
    float keep[kBatch];                          // 1 - lr weight_decay
    uint32_t key[kBatch];                        // of the 8-bit moments' rounding
};

struct Moments {
    void* exp_avg;
    void* exp_avg_sq;
    uint8_t* exp_avg_scale;
    uint8_t* exp_avg_sq_scale;
    float* master;
};

/* Workgroups to a chunk: a thread has one vector.  400 million weights in 32
 * bits take 1,953 us, and 2,000 with one workgroup to a chunk whose threads go
 * on twice over two vectors; 30 million in bf16 148 and 160; 200 million with
 * 8-bit moments 541 and 567. */
constexpr int kParts = 4, kPart = kChunk / kParts;
static_assert(kPart == kThreads * kVector, "a vector to a thread");

struct Rates {
    float beta1, beta2, rest1, rest2, eps;       // rest = 1 - beta, rounded once
};

/* Where a step's clip comes from. */
struct Clip {
    const float* scale;                          // NULL: none, or
    const double* partial;                       // `partials` sums of squares (at most kFewPartials)
    int partials;
    float max_norm;
    float* norm;
};

/* All arguments of a launch of aw_step: the chunks from `first` on, of tensors
 * from `base` on. */
struct StepLaunch {
    Gradients g;
    StepArgs a;
    int base;
    int64_t first;
    const int2* chunk;
    const Tensor* tensors;
    Moments mo;
    Rates rates;
    const float* inverse;
    const uint32_t* replays;                     // of a captured step, else NULL
    Clip clip;
};
static_assert(sizeof(StepLaunch) <= kMostArguments, "kernel arguments");

/* All arguments of a launch of aw_squares: the chunks from `first` to `end`. */
struct SquaresLaunch {
    Gradients g;
    int base;
    int64_t first, end;
    const int2* chunk;
    const Tensor* tensors;
    double* partial;
};
static_assert(sizeof(SquaresLaunch) <= kMostArguments, "kernel arguments");

}  // namespace b3p

struct B3AdamW {
    int device, count, bits;
    int64_t size, chunks;
    B3AdamWConfig config;
    b3p::Moments moments;
    b3p::Tensor* tensors;                        // device
    int2* chunk;                                 // device: tensor, chunk of it
    int partials;                                // of a step with a clip
    double* partial;                             // device: sums of squares
    float* scale;                                // device: the clip's factor
    float* inverse;                              // device: see aw_inverse
    uint32_t* replays;                           // device: captured steps of 8-bit moments that have run
    int64_t* first;                              // host: a tensor's first chunk; count + 1
    int64_t* steps;                              // host
    B3AdamWTensor* given;                        // host
};

namespace b3p {
namespace {

/* 32 well mixed bits of 32: two rounds of shift, xor and multiply.  The shifts
 * and multipliers are those of a published search for the least biased (C.
 * Wellons, "Prospecting for Hash Functions", 2018). */
inline __host__ __device__ uint32_t mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x7feb352du;
    x ^= x >> 15;
    x *= 0x846ca68bu;
    return x ^ x >> 16;
}

/* FULL: no element passes the tensor's end.  ONCE: not to be read again. */
template <bool FULL, bool ONCE, typename T>
__device__ void load(const T* p, int64_t i, int64_t n, float x[kVector]) {
    if (FULL || i + kVector <= n) {
        Pack<T, kVector> v = ONCE ? Stream<T, kVector>::load(p + i) : *(const Pack<T, kVector>*)(p + i);
#pragma unroll
        for (int k = 0; k < kVector; k++) x[k] = to_float(v.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < kVector; k++) x[k] = i + k < n ? to_float(p[i + k]) : 0.0f;
    }
}

/* The same as they lie, not to be read again. */
template <bool FULL, typename T>
__device__ Pack<T, kVector> load_raw(const T* p, int64_t i, int64_t n) {
    if (FULL || i + kVector <= n) return Stream<T, kVector>::load(p + i);
    Pack<T, kVector> v = {};
#pragma unroll
    for (int k = 0; k < kVector; k++)
        if (i + k < n) v.v[k] = p[i + k];
    return v;
}

template <bool FULL, typename T>
__device__ void store(T* p, int64_t i, int64_t n, const float x[kVector]) {
    if (FULL || i + kVector <= n) {
        Pack<T, kVector> v;
#pragma unroll
        for (int k = 0; k < kVector; k++) v.v[k] = (T)x[k];
        Stream<T, kVector>::store(p + i, v);
    } else {
#pragma unroll
        for (int k = 0; k < kVector; k++)
            if (i + k < n) p[i + k] = (T)x[k];
    }
}

/* ---- 8-bit moments: four e4m3 bytes of a thread, 8 threads to a scale ---- */

/* 4 N codes; bytes lie anywhere. */
template <int N>
__device__ Bytes<uint32_t, N> load_codes(const uint8_t* codes) {
    return *(const Bytes<uint32_t, N>*)codes;
}

__device__ void unpack(uint32_t codes, uint8_t scale, float x[kVector]) {
    float s = __uint_as_float((uint32_t)scale << 23);
    x[0] = __builtin_amdgcn_cvt_f32_fp8(codes, 0) * s;
    x[1] = __builtin_amdgcn_cvt_f32_fp8(codes, 1) * s;
    x[2] = __builtin_amdgcn_cvt_f32_fp8(codes, 2) * s;
    x[3] = __builtin_amdgcn_cvt_f32_fp8(codes, 3) * s;
}

/* The largest over 8 neighbouring lanes, by lanes swapped in pairs, pairs
 * swapped, and the eight mirrored. */
__device__ uint32_t max_of_8_lanes(uint32_t x) {
    uint32_t y = __builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, true);
    x = x > y ? x : y;
    y = __builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, true);
    x = x > y ? x : y;
    y = __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true);
    return x > y ? x : y;
}
static_assert(kGroup / kVector == 8, "a scale's lanes");

/* The exponent byte of the least power of two with which none of the group's
 * finite values passes 448 (7/8 of 2^9). */
__device__ uint32_t group_scale(const float x[kVector]) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < kVector; k++) {
        uint32_t a = __float_as_uint(x[k]) & 0x7fffffffu;
        a = a < 0x7f800000u ? a : 0;
        most = most > a ? most : a;
    }
    most = max_of_8_lanes(most);
    int e = (int)(most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u);
    return e < 1 ? 1 : e;
}

/* inverse[b] = 2^(127 - b) as pow() gives it, a unit in the last place low
 * for 41 exponents: torch.ldexp multiplies by the same numbers, so that a
 * torch program that rounds by the same bits gets the same moments.  With the
 * exact powers 1.3 in a million roundings go the other way, as many as a unit
 * in the last place of the moment itself moves; a moment on the grid falls a
 * step by one in 65,536 random bits on those scales.  Never over the exact
 * power: a group's largest, where it is 448 on its scale, would pass the
 * greatest number.  b goes from 1 to 247. */
__global__ void aw_inverse(float* inverse) {
    const uint32_t b = threadIdx.x;
    inverse[b] = fminf(powf(2.0f, 127.0f - (float)b), __uint_as_float((b < 254 ? 254 - b : 0) << 23));
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
__device__ uint32_t pack(const float x[kVector], float inverse, const uint32_t random[kVector]) {
    float y[kVector];
#pragma unroll
    for (int k = 0; k < kVector; k++)
        y[k] = round_code<RANDOM, ROOT>(x[k], inverse, ROOT ? random[k] >> 16 : random[k] & 0xffffu);
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
}

__device__ void store_codes(uint8_t* codes, uint8_t* scales, int64_t i, uint32_t code, uint32_t scale) {
    *(Bytes<uint32_t, 1>*)(codes + i) = Bytes<uint32_t, 1>{{code}};
    if (i % kGroup == 0) scales[i / kGroup] = (uint8_t)scale;
}

/* ---- the step ---- */

/* What a step is to a chunk. */
struct Step {
    const Moments& mo;
    const Rates& rates;
    const float* inverse;
    float clip, size, root, keep;
    uint32_t key;
};

/* A weight's 32-bit copy, unless the weight is no longer what the copy rounds
 * to: it was written since the last step and is then what counts.  Reading
 * 16 bits more a weight (30 million in bf16: 155 us a step, 146 without) tells
 * it for each, in replayed graphs too, which no count of writes on the host
 * does.  As a rule all of a vector are what their copies round to. */
template <typename P>
__device__ __forceinline__ void copies_or_weights(float w[kVector], const Pack<P, kVector>& held) {
    Pack<P, kVector> rounded;
#pragma unroll
    for (int k = 0; k < kVector; k++) rounded.v[k] = (P)w[k];
    if (__builtin_bit_cast(uint64_t, rounded) == __builtin_bit_cast(uint64_t, held)) return;
#pragma unroll
    for (int k = 0; k < kVector; k++) {
        const bool same = __builtin_bit_cast(uint16_t, rounded.v[k]) == __builtin_bit_cast(uint16_t, held.v[k]);
        w[k] = same ? w[k] : to_float(held.v[k]);
    }
}

/* A thread's vector of the part from `from` on.  The square root is the
 * correctly rounded one, since what is kept of it is cut off by random bits
 * (the hardware's with its residuals' correction took as long, and gives 0 for
 * denormals); the division in the update is a reciprocal, good to two units. */
template <typename P, typename G, bool MASTER, int BITS, bool FULL>
__device__ __forceinline__ void step_vector(const Tensor& t, int64_t from, const G* grad, const Step& s) {
    float g[kVector], w[kVector], m[kVector], v[kVector];
    Pack<P, kVector> held;                       // MASTER: the weights themselves
    const int64_t n = t.numel, i = from + (int)threadIdx.x * kVector, at = t.at + i;
    /* whole groups of 8-bit moments go on together */
    if (!FULL && i / kGroup * kGroup >= n) return;
    load<FULL, true>(grad, i, n, g);
    if (MASTER) {
        load<FULL, true>(s.mo.master + t.at, i, n, w);
        held = load_raw<FULL>((const P*)t.param, i, n);
    } else {
        load<FULL, true>((const P*)t.param, i, n, w);
    }
    if (BITS == 32) {
        load<FULL, true>((const float*)s.mo.exp_avg + t.at, i, n, m);
        load<FULL, true>((const float*)s.mo.exp_avg_sq + t.at, i, n, v);
    } else {
        const uint32_t cm = load_codes<1>((const uint8_t*)s.mo.exp_avg + at).v[0];
        const uint32_t cv = load_codes<1>((const uint8_t*)s.mo.exp_avg_sq + at).v[0];
        unpack(cm, s.mo.exp_avg_scale[at / kGroup], m);
        unpack(cv, s.mo.exp_avg_sq_scale[at / kGroup], v);
    }
    if constexpr (MASTER) copies_or_weights(w, held);
    float root[kVector];
#pragma unroll
    for (int j = 0; j < kVector; j++) {
        const float gc = g[j] * s.clip, old = BITS == 32 ? v[j] : v[j] * v[j];
        m[j] = m[j] * s.rates.beta1 + gc * s.rates.rest1;
        v[j] = old * s.rates.beta2 + gc * gc * s.rates.rest2;
        root[j] = sqrtf(v[j]);
        w[j] = w[j] * s.keep - m[j] * s.size * __builtin_amdgcn_rcpf(root[j] * s.root + s.rates.eps);
    }
    store<FULL>((P*)t.param, i, n, w);
    if (MASTER) store<FULL>(s.mo.master + t.at, i, n, w);
    if (BITS == 32) {
        store<FULL>((float*)s.mo.exp_avg + t.at, i, n, m);
        store<FULL>((float*)s.mo.exp_avg_sq + t.at, i, n, v);
    } else {
        uint32_t random[kVector];
        const uint32_t key = s.key ^ mix((uint32_t)(at >> 32));
#pragma unroll
        for (int j = 0; j < kVector; j++) random[j] = mix((uint32_t)(at + j) ^ key);
        const uint32_t to_m = group_scale(m), to_v = group_scale(root);
        store_codes((uint8_t*)s.mo.exp_avg, s.mo.exp_avg_scale, at, pack<true, false>(m, s.inverse[to_m], random), to_m);
        store_codes((uint8_t*)s.mo.exp_avg_sq, s.mo.exp_avg_sq_scale, at, pack<true, true>(root, s.inverse[to_v], random), to_v);
    }
}

template <typename P, typename G, bool MASTER, int BITS>
__device__ __forceinline__ void step_part(const Tensor& t, int64_t from, const G* grad, const Step& s) {
    if (from + kPart <= t.numel)
        step_vector<P, G, MASTER, BITS, true>(t, from, grad, s);
    else
        step_vector<P, G, MASTER, BITS, false>(t, from, grad, s);
}

template <typename P, bool MASTER, int BITS>
__device__ __forceinline__ void step_typed(const Tensor& t, int64_t from, const void* grad, bool float_grad, const Step& s) {
    if (float_grad)
        step_part<P, float, MASTER, BITS>(t, from, (const float*)grad, s);
    else
        step_part<P, P, MASTER, BITS>(t, from, (const P*)grad, s);
}

/* The clip's factor; a NaN norm stays one. */
__device__ float clip_of(float norm, float max_norm) {
    const float s = max_norm / (norm + 1e-6f);
    return s > 1.0f ? 1.0f : s;
}

template <int THREADS>
__device__ double block_sum(double x) {
    __shared__ double lds[THREADS / kWave];
    for (int d = kWave / 2; d > 0; d /= 2) x += __shfl_xor(x, d);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < THREADS / kWave; w++) x += lds[w];
    return x;
}

/* The key of the nth run of a captured step.  With the captured step's own a
 * replay would round every moment as the one before it did, and moments that
 * change by little would stay where they are. */
__device__ uint32_t key_of_replay(uint32_t key, uint32_t n) { return n ? mix(key + n * 0x9e3779b9u) : key; }

template <int BITS>
__global__ __launch_bounds__(kThreads) void aw_step(StepLaunch l) {
    const Clip& clip = l.clip;
    /* fetched together: the sums of squares and whose chunk it is */
    const double part = clip.partial && (int)threadIdx.x < clip.partials ? clip.partial[threadIdx.x] : 0;
    const int2 c = l.chunk[l.first + blockIdx.x / kParts];
    const Tensor t = l.tensors[c.x];
    const int at = c.x - l.base;
    const void* grad = l.g.at[at];
    float scale = clip.scale ? *clip.scale : 1.0f;
    if (clip.partial) {
        const float norm = (float)sqrt(block_sum<kThreads>(part));
        if (l.first + blockIdx.x == 0 && threadIdx.x == 0) *clip.norm = norm;
        scale = clip_of(norm, clip.max_norm);
    }
    const int64_t from = (int64_t)c.y * kChunk + blockIdx.x % kParts * kPart;
    if (!grad || from >= t.numel) return;
    const uint32_t key = BITS == 8 && l.replays ? key_of_replay(l.a.key[at], *l.replays) : l.a.key[at];
    const Step s = {l.mo, l.rates, l.inverse, scale, l.a.size[at], l.a.root[at], l.a.keep[at], key};
    const bool fg = l.g.type[at] == B3_F32;
    if (t.type == B3_F32)
        step_part<float, float, false, BITS>(t, from, (const float*)grad, s);
    else if (t.type == B3_BF16 && l.mo.master)
        step_typed<__bf16, true, BITS>(t, from, grad, fg, s);
    else if (t.type == B3_BF16)
        step_typed<__bf16, false, BITS>(t, from, grad, fg, s);
    else if (l.mo.master)
        step_typed<_Float16, true, BITS>(t, from, grad, fg, s);
    else
        step_typed<_Float16, false, BITS>(t, from, grad, fg, s);
}

/* After a captured step. */
__global__ void aw_count(uint32_t* replays) { ++*replays; }

/* ---- the norm ---- */

/* A thread's squares of a chunk: at most 16 in 32 bits, the rest of the sum
 * in 64. */
template <bool FULL, typename G>
__device__ float squares(const G* grad, int64_t from, int64_t n) {
    float g[kChunk / (kThreads * kVector)][kVector], sum = 0;
#pragma unroll
    for (int u = 0; u < kChunk / (kThreads * kVector); u++)
        load<FULL, false>(grad, from + (int64_t)(u * kThreads + (int)threadIdx.x) * kVector, n, g[u]);
#pragma unroll
    for (int u = 0; u < kChunk / (kThreads * kVector); u++)
#pragma unroll
        for (int j = 0; j < kVector; j++) sum += g[u][j] * g[u][j];
    return sum;
}

template <typename G>
__device__ float square_chunk(const void* grad, int64_t from, int64_t n) {
    return from + kChunk <= n ? squares<true>((const G*)grad, from, n) : squares<false>((const G*)grad, from, n);
}

__global__ __launch_bounds__(kThreads) void aw_squares(SquaresLaunch l) {
    double sum = 0;
    for (int64_t i = l.first + blockIdx.x; i < l.end; i += gridDim.x) {
        const int2 c = l.chunk[i];
        const int at = c.x - l.base;
        const void* grad = l.g.at[at];
        if (!grad) continue;
        const int64_t n = l.tensors[c.x].numel, from = (int64_t)c.y * kChunk;
        const int type = l.g.type[at];
        sum += type == B3_F32 ? square_chunk<float>(grad, from, n)
            : type == B3_BF16 ? square_chunk<__bf16>(grad, from, n) : square_chunk<_Float16>(grad, from, n);
    }
    sum = block_sum<kThreads>(sum);
    if (threadIdx.x == 0) l.partial[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kSumThreads) void aw_norm(const double* partial, int partials, float max_norm, float* norm,
    float* scale) {
    double sum = 0;
    for (int i = threadIdx.x; i < partials; i += kSumThreads) sum += partial[i];
    sum = block_sum<kSumThreads>(sum);
    if (threadIdx.x == 0) {
        *norm = (float)sqrt(sum);
        *scale = clip_of((float)sqrt(sum), max_norm);
    }
}

/* ---- 8-bit moments in and out ---- */

/* Eight of one of the moments a thread, so that neighbouring threads write 16
 * neighbouring bytes each. */
constexpr int kMomentsOut = 8;

template <bool ROOT>
__device__ __forceinline__ void moments_of(const uint8_t* codes, const uint8_t* scales, int64_t i, __bf16* out) {
    const Bytes<uint32_t, 2> c = load_codes<2>(codes + i);
    const uint8_t scale = scales[i / kGroup];
    float x[kMomentsOut];
    unpack(c.v[0], scale, x);
    unpack(c.v[1], scale, x + kVector);
    Pack<__bf16, kMomentsOut> y;
#pragma unroll
    for (int k = 0; k < kMomentsOut; k++) y.v[k] = (__bf16)(ROOT ? x[k] * x[k] : x[k]);
    Stream<__bf16, kMomentsOut>::store(out + i, y);
}

/* Element i of the flat arrays, from `first` on, to a thread. */
__global__ __launch_bounds__(kThreads) void aw_moments(Moments mo, int64_t first, int64_t size, __bf16* exp_avg,
    __bf16* exp_avg_sq) {
    const int64_t i = first + ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kMomentsOut;
    if (i >= size) return;                        // a multiple of 256
    moments_of<false>((const uint8_t*)mo.exp_avg, mo.exp_avg_scale, i, exp_avg);
    moments_of<true>((const uint8_t*)mo.exp_avg_sq, mo.exp_avg_sq_scale, i, exp_avg_sq);
}

__global__ __launch_bounds__(kThreads) void aw_load(Moments mo, int64_t first, int64_t size, const float* inverse,
    const float* exp_avg, const float* exp_avg_sq) {
    const int64_t i = first + ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kVector;
    if (i >= size) return;                        // a multiple of 256: groups stay whole
    float m[kVector], r[kVector];
    load<true, true>(exp_avg, i, size, m);
    load<true, true>(exp_avg_sq, i, size, r);
    for (int k = 0; k < kVector; k++) r[k] = sqrtf(r[k]);
    const uint32_t none[kVector] = {0, 0, 0, 0};
    uint32_t sm = group_scale(m), sr = group_scale(r);
    store_codes((uint8_t*)mo.exp_avg, mo.exp_avg_scale, i, pack<false, false>(m, inverse[sm], none), sm);
    store_codes((uint8_t*)mo.exp_avg_sq, mo.exp_avg_sq_scale, i, pack<false, true>(r, inverse[sr], none), sr);
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

int by_address(const void* a, const void* b) {
    const uintptr_t x = (uintptr_t)((const B3AdamWTensor*)a)->param, y = (uintptr_t)((const B3AdamWTensor*)b)->param;
    return (x > y) - (x < y);
}

/* Whether two of the tensors that have elements overlap; `sorted` has room for
 * all.  Weights that belong to two would be written by two workgroups. */
bool overlap(const B3AdamWTensor* tensors, int count, B3AdamWTensor* sorted) {
    int n = 0;
    for (int i = 0; i < count; i++)
        if (tensors[i].numel) sorted[n++] = tensors[i];
    qsort(sorted, (size_t)n, sizeof(B3AdamWTensor), by_address);
    for (int i = 1; i < n; i++) {
        const B3AdamWTensor& before = sorted[i - 1];
        const uintptr_t end = (uintptr_t)before.param + (uintptr_t)before.numel * (before.type == B3_F32 ? 4 : 2);
        if (end > (uintptr_t)sorted[i].param) return true;
    }
    return false;
}

int64_t segment(int64_t numel) { return ceil_div(numel, B3_ADAMW_SEGMENT) * B3_ADAMW_SEGMENT; }

/* Tensors of the launch that begins with tensor `base`. */
int batch(const B3AdamW* o, int base) { return o->count - base < kBatch ? o->count - base : kBatch; }

int sum_blocks(const B3AdamW* o, int base) {
    const int64_t chunks = o->first[base + batch(o, base)] - o->first[base];
    return (int)(chunks < kSumBlocks ? chunks : kSumBlocks);
}

/* The chunks from l.first to `end`. */
template <int BITS>
void launch_step(StepLaunch& l, int64_t end, hipStream_t stream) {
    constexpr int64_t kMost = kMostBlocks / kParts;
    for (; l.first < end; l.first += kMost) {
        const int64_t chunks = end - l.first < kMost ? end - l.first : kMost;
        aw_step<BITS><<<(unsigned)(chunks * kParts), kThreads, 0, stream>>>(l);
    }
}

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
    void* bufs[6] = {o->tensors, o->chunk, o->partial, o->scale, o->inverse, o->replays};
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
    hipError_t err = !(o->first && o->steps && o->given && table && chunk) ? hipErrorOutOfMemory
        : overlap(tensors, count, o->given) ? hipErrorInvalidValue : hipGetDevice(&o->device);
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
        for (int base = 0; base < count; base += kBatch) o->partials += sum_blocks(o, base);
    }
    if (err == hipSuccess) err = hipMalloc((void**)&o->tensors, ((size_t)count + 1) * sizeof(Tensor));
    if (err == hipSuccess) err = hipMalloc((void**)&o->chunk, ((size_t)chunks + 1) * sizeof(int2));
    if (err == hipSuccess) err = hipMalloc((void**)&o->partial, ((size_t)o->partials + 1) * sizeof(double));
    if (err == hipSuccess) err = hipMalloc((void**)&o->scale, sizeof(float));
    if (err == hipSuccess) err = hipMalloc((void**)&o->inverse, 256 * sizeof(float));
    if (err == hipSuccess) err = hipMalloc((void**)&o->replays, sizeof(uint32_t));
    const uint32_t none = 0;
    if (err == hipSuccess) err = hipMemcpy(o->replays, &none, sizeof(none), hipMemcpyHostToDevice);
    if (err == hipSuccess) {
        aw_inverse<<<1, 256>>>(o->inverse);
        err = hipGetLastError();
    }
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
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (o->bits == 8 && (err = hipStreamIsCapturing(stream, &capture)) != hipSuccess) return err;
    uint32_t* const replays = capture == hipStreamCaptureStatusNone ? NULL : o->replays;
    const B3AdamWConfig& cf = o->config;
    const Rates rates = {(float)cf.beta1, (float)cf.beta2, (float)(1 - cf.beta1), (float)(1 - cf.beta2), (float)cf.eps};
    const bool few = o->partials > 0 && o->partials <= kFewPartials;
    Clip clip = {};
    if (max_norm > 0) clip = few ? Clip{NULL, o->partial, o->partials, (float)max_norm, norm} : Clip{o->scale, NULL, 0, 0, NULL};
    StepLaunch l = {};
    l.chunk = o->chunk;
    l.tensors = o->tensors;
    l.mo = o->moments;
    l.rates = rates;
    l.inverse = o->inverse;
    l.replays = replays;
    l.clip = clip;
    for (int pass = max_norm > 0 ? 0 : 1; pass < 2; pass++) {
        int64_t t_last = -1;
        float size = 0, root = 0;
        double* partial = o->partial;
        for (int base = 0; base < o->count; base += kBatch) {
            const int n = batch(o, base);
            const int64_t first = o->first[base], end = o->first[base + n];
            for (int j = 0; j < n; j++) {
                const int i = base + j;
                l.g.at[j] = grads[i];
                l.g.type[j] = (uint8_t)(grad_types ? grad_types[i] : o->given[i].type);
                if (pass == 0 || !grads[i]) continue;
                const int64_t t = ++o->steps[i];
                if (t != t_last) {
                    size = (float)(lr / (1 - pow(cf.beta1, (double)t)));
                    root = (float)(1 / sqrt(1 - pow(cf.beta2, (double)t)));
                    t_last = t;
                }
                l.a.size[j] = size;
                l.a.root[j] = root;
                l.a.keep[j] = (float)(1 - lr * o->given[i].weight_decay);
                l.a.key[j] = mix((uint32_t)t * 0x9e3779b9u + cf.seed);
            }
            if (first == end) continue;
            if (pass == 0) {
                const int blocks = sum_blocks(o, base);
                aw_squares<<<blocks, kThreads, 0, stream>>>({l.g, base, first, end, o->chunk, o->tensors, partial});
                partial += blocks;
            } else {
                l.base = base;
                l.first = first;
                if (o->bits == 32)
                    launch_step<32>(l, end, stream);
                else
                    launch_step<8>(l, end, stream);
            }
            if ((err = hipGetLastError()) != hipSuccess) return err;
        }
        if (pass == 0 && !few) {
            aw_norm<<<1, kSumThreads, 0, stream>>>(o->partial, o->partials, (float)max_norm, norm, o->scale);
            if ((err = hipGetLastError()) != hipSuccess) return err;
        }
    }
    if (replays) {
        aw_count<<<1, 1, 0, stream>>>(replays);
        err = hipGetLastError();
    }
    return err;
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
    const int64_t most = kMostBlocks * kThreads * kMomentsOut;
    for (int64_t first = 0; first < o->size && err == hipSuccess; first += most) {
        const int64_t n = o->size - first < most ? o->size - first : most;
        aw_moments<<<(unsigned)ceil_div(n, kThreads * kMomentsOut), kThreads, 0, stream>>>(o->moments, first, o->size,
            (__bf16*)exp_avg, (__bf16*)exp_avg_sq);
        err = hipGetLastError();
    }
    return err;
}

hipError_t b3_adamw_load_moments_gpu(B3AdamW* o, const float* exp_avg, const float* exp_avg_sq, hipStream_t stream) {
    if (!o || o->bits != 8 || (o->size && (!exp_avg || !exp_avg_sq))) return hipErrorInvalidValue;
    hipError_t err = on_device(o);
    if (err != hipSuccess || o->size == 0) return err;
    const int64_t most = kMostBlocks * kThreads * kVector;
    for (int64_t first = 0; first < o->size && err == hipSuccess; first += most) {
        const int64_t n = o->size - first < most ? o->size - first : most;
        aw_load<<<(unsigned)ceil_div(n, kThreads * kVector), kThreads, 0, stream>>>(o->moments, first, o->size, o->inverse,
            exp_avg, exp_avg_sq);
        err = hipGetLastError();
    }
    return err;
}

}  // extern "C"
