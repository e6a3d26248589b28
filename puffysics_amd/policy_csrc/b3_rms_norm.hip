/*
 * b3_rms_norm.hip - the root-mean-square norm with the residual's addition, its
 * gradient, and an output in 8 bits (include/b3_policy.h).
 *
 *   h = x + r, s = 1 / sqrt(mean h^2 + eps), y = w h s
 *   dh = d_h + s (w dy - h s mean(w dy h s)), dw = sum over rows of dy h s
 *
 * Everything is read once and written once, so that memory bounds it.  G lanes
 * share a row and hold it in registers, one to four vectors of 8 neighbouring
 * elements each: 4 to 64 lanes of a wave, or a workgroup's 256 beyond 1,024
 * elements, 512 beyond 2,048 and, back, 1,024 beyond 8,192.
 * Rows of more than 16,384 are gone over twice.  A lane keeps its columns from
 * row to row: of the weights' gradient each workgroup writes the sums over its
 * rows, in one order always, and a second launch adds these.
 */
#include "policy_common.h"

namespace b3p {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;
constexpr int kWide = 1024;                      // lanes to the longest rows that registers hold
constexpr int kMostInRegisters = kWide * kVec * 2;
constexpr int64_t kMaxWidth = 1 << 21;
constexpr int64_t kForwardBlocks = 2048, kBackwardBlocks = 1024;
constexpr int64_t kAlone = 4;                    // turns of one workgroup over its rows
constexpr int64_t kMostSums = 1 << 25;           // of long rows: floats of the workgroups' sums
constexpr int kGroup = 32;                       // 8 bits: elements to a scale
constexpr int kSumColumns = 64, kSumSlices = 16;

struct Job {
    B3Norm g;
    float eps;
    void* out;
    unsigned char* scale;                        // of 8 bits
    void* sum;
    float* root;                                 // written by the forward pass, read by the backward
    const void* d_out;
    int64_t d_out_stride;
    const void* d_sum;
    int64_t d_sum_stride;
    float* partial;                              // [workgroups][width], or NULL
    void* d_weight;                              // of one workgroup, or NULL
    float* dot;                                  // [rows], of long rows
};

/* Eight elements of a row of `width` from column c on, zeros past its end.  Of
 * the last ones, fewer than eight, the eight that end the row are fetched and
 * moved down: by the same steps in all rows. */
template <typename T>
__device__ __forceinline__ void load8(const T* row, int64_t c, int64_t width, float x[kVec]) {
    const int64_t left = width - c;
    const int past = (int)(-width & (kVec - 1));
    if (left <= 0) {
#pragma unroll
        for (int k = 0; k < kVec; k++) x[k] = 0.0f;
    } else if (left >= kVec || width >= kVec) {
        const Pack<T, kVec> v = *(const Pack<T, kVec>*)(row + (left >= kVec ? c : width - kVec));
#pragma unroll
        for (int k = 0; k < kVec; k++) x[k] = to_float(v.v[k]);
        if (past && left < kVec) {
#pragma unroll
            for (int s = kVec / 2; s; s /= 2) {
#pragma unroll
                for (int k = 0; k < kVec; k++) x[k] = past & s ? (k + s < kVec ? x[k + s] : 0.0f) : x[k];
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < kVec; k++) x[k] = k < left ? to_float(row[c + k]) : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t left, const float x[kVec]) {
    if (left >= kVec) {
        Pack<T, kVec> v;
#pragma unroll
        for (int k = 0; k < kVec; k++) v.v[k] = (T)x[k];
        *(Pack<T, kVec>*)p = v;
    } else {
#pragma unroll
        for (int k = 0; k < kVec; k++)
            if (k < left) p[k] = (T)x[k];
    }
}

template <typename T>
__device__ __forceinline__ void load_weight(const B3Norm& g, int64_t c, float w[kVec]) {
    if (!g.weight) {
#pragma unroll
        for (int k = 0; k < kVec; k++) w[k] = 1.0f;
    } else if (g.weight_type == B3_F32) {
        load8((const float*)g.weight, c, g.width, w);
    } else {
        load8((const T*)g.weight, c, g.width, w);
    }
}

/* Over the G lanes of a row, each with the sum. */
template <int G>
__device__ __forceinline__ float row_sum(float x, float* lds) {
#pragma unroll
    for (int d = 1; d < (G < kWave ? G : kWave); d *= 2) x += __shfl_xor(x, d);
    if (G > kWave) {
        __syncthreads();
        if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = x;
        __syncthreads();
        x = 0;
#pragma unroll
        for (int w = 0; w < G / kWave; w++) x += lds[w];
    }
    return x;
}

/* h of eight elements. */
template <typename T>
__device__ __forceinline__ void load_h(const B3Norm& g, int64_t r, int64_t c, float h[kVec]) {
    load8((const T*)g.x + r * g.x_stride, c, g.width, h);
    if (g.residual) {
        float d[kVec];
        load8((const T*)g.residual + r * g.residual_stride, c, g.width, d);
#pragma unroll
        for (int k = 0; k < kVec; k++) h[k] += d[k];
    }
}

/* Codes of eight elements whose scale they share with those of four lanes in
 * all.  The power is that of the largest's least one; 2^-126 at the least, as
 * of zeros. */
__device__ __forceinline__ void store_codes(const Job& j, int64_t r, int64_t c, const float y[kVec]) {
    const int64_t left = j.g.width - c;
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < kVec; k++) {
        const uint32_t b = __float_as_uint(y[k]) & 0x7fffffffu;
        if (k < left && b > most) most = b;
    }
#pragma unroll
    for (int d = 1; d < kGroup / kVec; d *= 2) {
        const uint32_t other = (uint32_t)__shfl_xor((int)most, d);
        most = other > most ? other : most;
    }
    /* 2^e is over the largest, which is over 7/8 of it: the power is e - 9 or e - 8 */
    int power = (int)(most >> 23) - 126 - 9 + ((most & 0x7fffffu) > 0x600000u);
    power = power < -126 ? -126 : power;
    const float inverse = __uint_as_float((uint32_t)(127 - power) << 23);
    if (left <= 0) return;
    uint32_t code[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < kVec; k += 4) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(y[k] * inverse, y[k + 1] * inverse, 0, false);
        word = __builtin_amdgcn_cvt_pk_fp8_f32(y[k + 2] * inverse, y[k + 3] * inverse, word, true);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if ((__float_as_uint(y[k + i]) & 0x7f800000u) == 0x7f800000u) word = (word & ~(0xff << 8 * i)) | 0x7f << 8 * i;
        code[k / 4] = (uint32_t)word;
    }
    unsigned char* out = (unsigned char*)j.out + r * j.g.width + c;
    if (left >= kVec) {
        *(Bytes<uint32_t, 2>*)out = Bytes<uint32_t, 2>{code[0], code[1]};
    } else {
#pragma unroll
        for (int k = 0; k < kVec; k++)
            if (k < left) out[k] = (unsigned char)(code[k / 4] >> 8 * (k % 4));
    }
    if (c % kGroup == 0) j.scale[r * ceil_div(j.g.width, kGroup) + c / kGroup] = (unsigned char)(power + 127);
}

template <typename T, bool BITS8>
__device__ __forceinline__ void write_row(const Job& j, int64_t r, int64_t c, const float h[kVec], const float w[kVec],
    float s) {
    float y[kVec];
#pragma unroll
    for (int k = 0; k < kVec; k++) y[k] = h[k] * s * w[k];
    if (BITS8)
        store_codes(j, r, c, y);
    else
        store8((T*)j.out + r * j.g.width + c, j.g.width - c, y);
    if (j.sum) store8((T*)j.sum + r * j.g.width + c, j.g.width - c, h);
}

__device__ __forceinline__ float root_of(const Job& j, float squares) {
    return rsqrtf(squares / (float)j.g.width + j.eps);
}

/* Threads of a workgroup whose rows have G lanes. */
constexpr int threads_of(int g) { return g > kThreads ? g : kThreads; }

/* 262,144 rows of 256 in bf16 with a residual 90 us, 6.0 TB/s, in fp32, call after
 * call, 216 us, 5.0 TB/s; 16,384 rows of 4,096 with 8 bits out 97 us, 4.8 TB/s. */
template <typename T, int G, int NV, bool BITS8>
__global__ __launch_bounds__(threads_of(G)) void rn_forward(Job j) {
    constexpr int kGroups = threads_of(G) / G;
    __shared__ float lds[threads_of(G) / kWave];
    const int lane = threadIdx.x % G;
    float w[NV][kVec];
#pragma unroll
    for (int v = 0; v < NV; v++) load_weight<T>(j.g, (v * G + lane) * kVec, w[v]);
    for (int64_t r = (int64_t)blockIdx.x * kGroups + threadIdx.x / G; r < j.g.rows; r += (int64_t)gridDim.x * kGroups) {
        float h[NV][kVec], squares = 0;
#pragma unroll
        for (int v = 0; v < NV; v++) load_h<T>(j.g, r, (v * G + lane) * kVec, h[v]);
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int k = 0; k < kVec; k++) squares += h[v][k] * h[v][k];
        const float s = root_of(j, row_sum<G>(squares, lds));
#pragma unroll
        for (int v = 0; v < NV; v++) write_row<T, BITS8>(j, r, (v * G + lane) * kVec, h[v], w[v], s);
        if (j.root && lane == 0) j.root[r] = s;
    }
}

/* Rows that registers do not hold: a workgroup goes over each twice.  2,048 rows
 * of 40,000 in bf16 with a residual 214 us (3.1 TB/s of what has to be read and
 * written), back 325 (2.5), in fp32 426 and 446. */
template <typename T, bool BITS8>
__global__ __launch_bounds__(kThreads) void rn_forward_long(Job j) {
    __shared__ float lds[kThreads / kWave];
    const int64_t round = ceil_div(j.g.width, kThreads * kVec) * kThreads * kVec;
    for (int64_t r = blockIdx.x; r < j.g.rows; r += gridDim.x) {
        float squares = 0;
        for (int64_t c = threadIdx.x * kVec; c < j.g.width; c += kThreads * kVec) {
            float h[kVec], part = 0;
            load_h<T>(j.g, r, c, h);
#pragma unroll
            for (int k = 0; k < kVec; k++) part += h[k] * h[k];
            squares += part;
        }
        const float s = root_of(j, row_sum<kThreads>(squares, lds));
        /* lanes that share a scale go past the end together */
        for (int64_t c = threadIdx.x * kVec; c < round; c += kThreads * kVec) {
            float h[kVec], w[kVec];
            load_h<T>(j.g, r, c, h);
            load_weight<T>(j.g, c, w);
            write_row<T, BITS8>(j, r, c, h, w, s);
        }
        if (j.root && threadIdx.x == 0) j.root[r] = s;
    }
}

/* dh and the sums over rows for eight elements, from u = h s, g = w dy and the
 * mean of g u. */
template <typename T>
__device__ __forceinline__ void write_d(const Job& j, int64_t r, int64_t c, const float u[kVec], const float g[kVec],
    float s, float mean) {
    float d[kVec];
#pragma unroll
    for (int k = 0; k < kVec; k++) d[k] = s * (g[k] - u[k] * mean);
    if (j.d_sum) {
        float up[kVec];
        load8((const T*)j.d_sum + r * j.d_sum_stride, c, j.g.width, up);
#pragma unroll
        for (int k = 0; k < kVec; k++) d[k] += up[k];
    }
    store8((T*)j.out + r * j.g.width + c, j.g.width - c, d);
}

template <typename T>
__device__ __forceinline__ void load_d_out(const Job& j, int64_t r, int64_t c, float d[kVec]) {
    if (j.d_out) {
        load8((const T*)j.d_out + r * j.d_out_stride, c, j.g.width, d);
    } else {
#pragma unroll
        for (int k = 0; k < kVec; k++) d[k] = 0;
    }
}

__device__ __forceinline__ void store_weight(void* out, int type, int64_t c, float x) {
    if (type == B3_F32)
        ((float*)out)[c] = x;
    else if (type == B3_F16)
        ((_Float16*)out)[c] = (_Float16)x;
    else
        ((__bf16*)out)[c] = (__bf16)x;
}

/* It reads what the forward pass read, the gradients and writes one: 262,144 rows
 * of 256 in bf16 with a residual 138 us, 4.9 TB/s, in fp32, of the sum, 198 us, 5.4
 * TB/s. */
template <typename T, int G, int NV>
__global__ __launch_bounds__(threads_of(G)) void rn_backward(Job j) {
    constexpr int kGroups = threads_of(G) / G;
    __shared__ float lds[threads_of(G) / kWave];
    __shared__ float sums[kGroups > 1 ? kThreads * kVec * NV : 1];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    float w[NV][kVec], dw[NV][kVec];
#pragma unroll
    for (int v = 0; v < NV; v++) {
        load_weight<T>(j.g, (v * G + lane) * kVec, w[v]);
#pragma unroll
        for (int k = 0; k < kVec; k++) dw[v][k] = 0;
    }
    for (int64_t r = (int64_t)blockIdx.x * kGroups + group; r < j.g.rows; r += (int64_t)gridDim.x * kGroups) {
        float u[NV][kVec], g[NV][kVec], dot = 0;
        const float s = j.root[r];
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int64_t c = (v * G + lane) * kVec;
            load_h<T>(j.g, r, c, u[v]);
            load_d_out<T>(j, r, c, g[v]);
        }
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int k = 0; k < kVec; k++) {
                u[v][k] *= s;
                dw[v][k] += g[v][k] * u[v][k];
                g[v][k] *= w[v][k];
                dot += g[v][k] * u[v][k];
            }
        const float mean = row_sum<G>(dot, lds) / (float)j.g.width;
#pragma unroll
        for (int v = 0; v < NV; v++) write_d<T>(j, r, (v * G + lane) * kVec, u[v], g[v], s, mean);
    }
    if (!j.partial && !j.d_weight) return;
    float* to = j.partial + (int64_t)blockIdx.x * j.g.width;
    if (kGroups > 1) {
#pragma unroll
        for (int v = 0; v < NV; v++)
#pragma unroll
            for (int k = 0; k < kVec; k++) sums[(group * G * NV + v * G + lane) * kVec + k] = dw[v][k];
        __syncthreads();
        for (int c = threadIdx.x; c < j.g.width; c += kThreads) {
            float x = 0;
#pragma unroll
            for (int i = 0; i < kGroups; i++) x += sums[i * G * NV * kVec + c];
            if (j.d_weight) store_weight(j.d_weight, j.g.weight_type, c, x);
            else to[c] = x;
        }
    } else {
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int64_t c = (v * G + lane) * kVec, left = j.g.width - c;
            if (!j.d_weight) store8(to + c, left, dw[v]);
            else if (j.g.weight_type == B3_F32) store8((float*)j.d_weight + c, left, dw[v]);
            else store8((T*)j.d_weight + c, left, dw[v]);
        }
    }
}

/* Rows that registers do not hold: first each row's mean, ... */
template <typename T>
__global__ __launch_bounds__(kThreads) void rn_dot(Job j) {
    __shared__ float lds[kThreads / kWave];
    for (int64_t r = blockIdx.x; r < j.g.rows; r += gridDim.x) {
        float dot = 0;
        for (int64_t c = threadIdx.x * kVec; c < j.g.width; c += kThreads * kVec) {
            float h[kVec], d[kVec], w[kVec], part = 0;
            load_h<T>(j.g, r, c, h);
            load_d_out<T>(j, r, c, d);
            load_weight<T>(j.g, c, w);
#pragma unroll
            for (int k = 0; k < kVec; k++) part += d[k] * w[k] * (h[k] * j.root[r]);
            dot += part;
        }
        dot = row_sum<kThreads>(dot, lds);
        if (threadIdx.x == 0) j.dot[r] = dot / (float)j.g.width;
    }
}

/* ... then columns of a part of the rows. */
template <typename T>
__global__ __launch_bounds__(kThreads) void rn_backward_long(Job j) {
    const int64_t c = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kVec;
    if (c >= j.g.width) return;
    float w[kVec], dw[kVec] = {};
    load_weight<T>(j.g, c, w);
    for (int64_t r = blockIdx.y; r < j.g.rows; r += gridDim.y) {
        float u[kVec], g[kVec];
        const float s = j.root[r];
        load_h<T>(j.g, r, c, u);
        load_d_out<T>(j, r, c, g);
#pragma unroll
        for (int k = 0; k < kVec; k++) {
            u[k] *= s;
            dw[k] += g[k] * u[k];
            g[k] *= w[k];
        }
        write_d<T>(j, r, c, u, g, s, j.dot[r]);
    }
    if (j.partial) store8(j.partial + (int64_t)blockIdx.y * j.g.width + c, j.g.width - c, dw);
}

/* The sums over workgroups, 5 us of 1,024. */
__global__ __launch_bounds__(kSumColumns * kSumSlices) void rn_weight(const float* partial, int blocks, int64_t width,
    void* out, int type) {
    __shared__ float lds[kSumSlices][kSumColumns];
    const int col = threadIdx.x % kSumColumns, slice = threadIdx.x / kSumColumns;
    const int64_t c = (int64_t)blockIdx.x * kSumColumns + col;
    float x = 0;
    if (c < width) {
#pragma unroll 8
        for (int b = slice; b < blocks; b += kSumSlices) x += partial[b * width + c];
    }
    lds[slice][col] = x;
    __syncthreads();
    if (slice || c >= width) return;
    x = 0;
#pragma unroll
    for (int i = 0; i < kSumSlices; i++) x += lds[i][col];
    store_weight(out, type, c, x);
}

/* Eight values of a row to a thread: 16,384 rows of 4,096 to bf16 35 us, 5.8
 * TB/s. */
template <typename T>
__global__ __launch_bounds__(kThreads) void rn_values(int64_t rows, int64_t width, const unsigned char* in,
    const unsigned char* scale, T* out) {
    const int64_t vectors = ceil_div(width, kVec), total = rows * vectors;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t r = i / vectors, c = i % vectors * kVec, left = width - c;
        const unsigned char* p = in + r * width + c;
        uint32_t code[2] = {0, 0};
        if (left >= kVec) {
            const Bytes<uint32_t, 2> b = *(const Bytes<uint32_t, 2>*)p;
            code[0] = b.v[0];
            code[1] = b.v[1];
        } else {
            for (int k = 0; k < left; k++) code[k / 4] |= (uint32_t)p[k] << 8 * (k % 4);
        }
        /* 2^-127 is a denormal, 255 is NaN */
        const uint32_t e = scale[r * ceil_div(width, kGroup) + c / kGroup];
        const float s = e == 255 ? NAN : e == 0 ? 0x1p-127f : __uint_as_float(e << 23);
        float x[kVec];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            x[4 * k] = __builtin_amdgcn_cvt_f32_fp8(code[k], 0) * s;
            x[4 * k + 1] = __builtin_amdgcn_cvt_f32_fp8(code[k], 1) * s;
            x[4 * k + 2] = __builtin_amdgcn_cvt_f32_fp8(code[k], 2) * s;
            x[4 * k + 3] = __builtin_amdgcn_cvt_f32_fp8(code[k], 3) * s;
        }
        store8(out + r * width + c, left, x);
    }
}

/* ---- launches ---- */

enum Pass { FORWARD, FORWARD_8BIT, BACKWARD };

template <typename T, int G, int NV, Pass PASS>
void launch_row(const Job& j, unsigned blocks, hipStream_t stream) {
    if constexpr (PASS == BACKWARD)
        rn_backward<T, G, NV><<<blocks, threads_of(G), 0, stream>>>(j);
    else
        rn_forward<T, G, NV, PASS == FORWARD_8BIT><<<blocks, threads_of(G), 0, stream>>>(j);
}

/* Lanes to a row; 0 where registers do not hold it.  Two vectors to a lane of a
 * wave rather than four waves to a row of over 512: 65,536 rows of 768 in bf16
 * 37 us forward and 72 back, 47 and 127 with 256 lanes.  The fewest waves that
 * hold a row are best beyond as well, since all wait for the sum: 16,384 rows of
 * 4,096 in bf16 take 42 and 88 us with 512 lanes, 80 and 151 with 1,024; 8,192
 * rows of 8,192 43 and 92, 56 and 100 with 1,024. */
int lanes_of(int64_t width) {
    const int64_t v = ceil_div(width, kVec);
    return v <= 4 ? 4 : v <= 16 ? 16 : v <= 32 ? 32 : v <= 128 ? 64 : v <= 256 ? kThreads : v <= 1024 ? 2 * kThreads : width <= kMostInRegisters ? kWide : 0;
}

int64_t blocks_of(int64_t rows, int64_t width, bool backward) {
    const int lanes = lanes_of(width);
    int64_t most = backward ? kBackwardBlocks : kForwardBlocks;
    if (backward && !lanes && most > kMostSums / width) most = kMostSums / width;
    const int64_t need = ceil_div(rows, lanes && lanes < kThreads ? kThreads / lanes : 1);
    /* Few rows are one workgroup's, which has the weights' gradient without a second launch: 16 rows of 256 take
     * 4.1 us, 5.3 in two.  At four turns that is 0.3 to 2 us more on the device, and 4 less on the host. */
    if (backward && lanes && need <= kAlone) return 1;
    return need < most ? need : most;
}

template <typename T, Pass PASS>
void launch_typed(const Job& j, hipStream_t stream) {
    const int64_t width = j.g.width, v = ceil_div(width, kVec);
    const unsigned blocks = (unsigned)blocks_of(j.g.rows, width, PASS == BACKWARD);
    if (v <= 4) launch_row<T, 4, 1, PASS>(j, blocks, stream);
    else if (v <= 16) launch_row<T, 16, 1, PASS>(j, blocks, stream);
    else if (v <= 32) launch_row<T, 32, 1, PASS>(j, blocks, stream);
    else if (v <= 64) launch_row<T, 64, 1, PASS>(j, blocks, stream);
    else if (v <= 128) launch_row<T, 64, 2, PASS>(j, blocks, stream);
    else if (v <= 256) launch_row<T, kThreads, 1, PASS>(j, blocks, stream);
    else if (v <= 512) launch_row<T, 2 * kThreads, 1, PASS>(j, blocks, stream);
    else if (v <= 1024) launch_row<T, 2 * kThreads, 2, PASS>(j, blocks, stream);
    else if (v <= 2048) {
        /* 8,192 rows of 12,000 in bf16: 88 us forward and 230 back with four vectors to each of 512 lanes, 101 and 163
         * with two to 1,024 */
        if constexpr (PASS == BACKWARD) launch_row<T, kWide, 2, PASS>(j, blocks, stream);
        else launch_row<T, 2 * kThreads, 4, PASS>(j, blocks, stream);
    }
    else if (PASS != BACKWARD) rn_forward_long<T, PASS == FORWARD_8BIT><<<blocks, kThreads, 0, stream>>>(j);
    else {
        rn_dot<T><<<(unsigned)blocks_of(j.g.rows, width, false), kThreads, 0, stream>>>(j);
        rn_backward_long<T><<<dim3((unsigned)ceil_div(v, kThreads), blocks), kThreads, 0, stream>>>(j);
    }
}

template <Pass PASS>
hipError_t launch(const Job& j, hipStream_t stream) {
    if (j.g.type == B3_F32) launch_typed<float, PASS>(j, stream);
    else if (j.g.type == B3_F16) launch_typed<_Float16, PASS>(j, stream);
    else launch_typed<__bf16, PASS>(j, stream);
    return hipGetLastError();
}

bool valid(const B3Norm* g) {
    if (!g || !is_float_type(g->type) || g->rows < 0 || g->rows > 0x7fffffff || g->width < 1 || g->width > kMaxWidth
            || !(g->eps >= 0))
        return false;
    if (g->weight && g->weight_type != B3_F32 && g->weight_type != g->type) return false;
    if (g->rows == 0) return true;
    return g->x && (g->rows == 1 || (g->x_stride >= g->width && (!g->residual || g->residual_stride >= g->width)));
}

}  // namespace
}  // namespace b3p

using namespace b3p;

extern "C" {

hipError_t b3_rms_norm_gpu(const B3Norm* norm, void* out, void* sum, float* root, hipStream_t stream) {
    if (!valid(norm) || (norm->rows && !out) || (sum && !norm->residual)) return hipErrorInvalidValue;
    if (norm->rows == 0) return hipSuccess;
    Job j = {};
    j.g = *norm;
    j.eps = (float)norm->eps;
    j.out = out;
    j.sum = sum;
    j.root = root;
    return launch<FORWARD>(j, stream);
}

hipError_t b3_rms_norm_8bit_gpu(const B3Norm* norm, unsigned char* out, unsigned char* scale, void* sum,
        hipStream_t stream) {
    if (!valid(norm) || (norm->rows && (!out || !scale)) || (sum && !norm->residual)) return hipErrorInvalidValue;
    if (norm->rows == 0) return hipSuccess;
    Job j = {};
    j.g = *norm;
    j.eps = (float)norm->eps;
    j.out = out;
    j.scale = scale;
    j.sum = sum;
    return launch<FORWARD_8BIT>(j, stream);
}

hipError_t b3_values_of_8bit_gpu(int64_t rows, int64_t width, const unsigned char* in, const unsigned char* scale,
        void* out, int type, hipStream_t stream) {
    if (rows < 0 || rows > 0x7fffffff || width < 1 || width > kMaxWidth || !is_float_type(type)
            || (rows && (!in || !scale || !out)))
        return hipErrorInvalidValue;
    if (rows == 0) return hipSuccess;
    const int64_t need = ceil_div(rows * ceil_div(width, kVec), kThreads), most = 16 * kForwardBlocks;
    const unsigned blocks = (unsigned)(need < most ? need : most);
    if (type == B3_F32) rn_values<float><<<blocks, kThreads, 0, stream>>>(rows, width, in, scale, (float*)out);
    else if (type == B3_F16) rn_values<_Float16><<<blocks, kThreads, 0, stream>>>(rows, width, in, scale, (_Float16*)out);
    else rn_values<__bf16><<<blocks, kThreads, 0, stream>>>(rows, width, in, scale, (__bf16*)out);
    return hipGetLastError();
}

size_t b3_rms_norm_backward_workspace(int64_t rows, int64_t width) {
    if (rows <= 0 || width <= 0) return 0;
    const int64_t blocks = blocks_of(rows, width, true), sums = blocks == 1 && lanes_of(width) ? 0 : blocks * width;
    return (size_t)(sums + (lanes_of(width) ? 0 : rows)) * sizeof(float);
}

hipError_t b3_rms_norm_backward_gpu(const B3Norm* norm, const float* root, const void* d_out, int64_t d_out_stride,
        const void* d_sum, int64_t d_sum_stride, void* d_x, void* d_weight, void* workspace, size_t workspace_bytes,
        hipStream_t stream) {
    if (!valid(norm) || (d_weight && !norm->weight)) return hipErrorInvalidValue;
    if (norm->rows > 1 && ((d_out && d_out_stride < norm->width) || (d_sum && d_sum_stride < norm->width)))
        return hipErrorInvalidValue;
    if (norm->rows && (!root || !d_x)) return hipErrorInvalidValue;
    if (!holds(workspace, workspace_bytes, b3_rms_norm_backward_workspace(norm->rows, norm->width)))
        return hipErrorInvalidValue;
    Job j = {};
    j.g = *norm;
    j.out = d_x;
    j.root = (float*)root;
    j.d_out = d_out;
    j.d_out_stride = d_out_stride;
    j.d_sum = d_sum;
    j.d_sum_stride = d_sum_stride;
    const int64_t blocks = norm->rows ? blocks_of(norm->rows, norm->width, true) : 0;
    const bool alone = blocks == 1 && lanes_of(norm->width);
    j.partial = d_weight && !alone ? (float*)workspace : NULL;
    j.d_weight = alone ? d_weight : NULL;
    j.dot = (float*)workspace + blocks * norm->width;
    hipError_t err = norm->rows ? launch<BACKWARD>(j, stream) : hipSuccess;
    if (err != hipSuccess || !d_weight || alone) return err;
    rn_weight<<<(unsigned)ceil_div(norm->width, kSumColumns), kSumColumns * kSumSlices, 0, stream>>>((float*)workspace,
        (int)blocks, norm->width, d_weight, norm->weight_type);
    return hipGetLastError();
}

}  // extern "C"
