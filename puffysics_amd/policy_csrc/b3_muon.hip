/*
 * b3_muon.hip - Muon's step over a policy's matrices (include/b3_policy.h).
 *
 *   m = momentum m + g, u = g + momentum m, x = u / (|u| + eps)
 *   y = x x^T, z = a + b y + c y y, x = z x, some times; then w moves by x
 *
 * x is a matrix with its shorter side first, so that y and z are as small as
 * they can be; they are symmetric, and half of their tiles are computed, but for
 * small matrices, of which all are.
 *
 * Products of 32-bit numbers come of three on the 16-bit matrix units: a
 * number is kept as a half and the half of what is left, 22 bits in all, and
 * h h' + h l' + l h' leaves out 2^-22 of a term (S. Markidis and others,
 * "NVIDIA Tensor Core Programmability, Performance & Precision", 2018, has the
 * idea).  The range of halves is enough, since x, y and z are bounded: their
 * singular values stay under 1.21, 1.47 and 3.45, whatever the gradient, and
 * kScale brings their elements to where 2^-24, the least half, is 2^-37.
 * Accumulators are in 32 bits.
 *
 * Where x is much longer than wide, its steps are taken on the short side: with y
 * and z as above y becomes z y z, p = .. z z z collects the steps, and x becomes
 * p x after kGroup of them.  That is 3 m m n + (4 kGroup - 3) m^3 multiplications
 * rather than kGroup (3 m m n + m^3), half tiles taken for half.  y is then formed
 * anew from x, because its rounding, some 2^-22 of its norm, grows by up to
 * 3.4445^2 a step where y is all but 0: after 3 steps x is about as exact as by
 * products of 32 bits, after 5 it was off by 1e-3 of its norm for gradients of two
 * strong directions over others of a tenth, 512 x 1,024, where it is by 3e-6 (by
 * 1e-2 and 5e-5 for those two alone).  The 16 matrices of 2,048 x 512 and 512 x
 * 2,048 of a network's step pay for it with 116 of 1,022 us.  The rounding of many
 * rows is spread over as many directions; of few rows it is not, and x of one
 * tile's rows takes all its steps as above: 5 x 510 of that kind is off by 1.3e-6
 * so and was by 5e-5.
 *
 * A launch computes a product of all matrices, or those that need not wait for
 * each other, a workgroup to a tile of 128 x 128.  Matrices lie in blocks of 32
 * columns, halves and what is left side by side, 128 bytes to a row's block;
 * both sides are filled up with zeros to whole tiles.  Matrices of at most 64 x
 * 256 take all of their step in one workgroup's LDS.
 */
#include "policy_common.h"

#include <stdlib.h>

namespace b3p {

constexpr int kThreads = 256;
constexpr int kBatch = 200;                      // matrices to a launch that takes gradients
constexpr size_t kMostArguments = 4096;          // bytes of a launch
constexpr int kTile = 128, kStep = 32;           // of a product: rows and columns, and what is summed at once
constexpr int kSquare = 8;                       // tiles
constexpr int kCut = 64;                         // tile of the first x
constexpr int kMostParts = 256;                  // workgroups that a matrix' gradient is gone over by
/* Where row r of a side that is read across lies in LDS: the 32 bytes that 16
 * lanes fetch of each of four rows, and those of the rows 8 on, are in
 * different banks. */
constexpr int across_row(int r) { return r * (kTile * 4 + 32) + r / 8 * 128; }
constexpr int kSideLds = across_row(kStep), kProductLds = 4 * kSideLds;      // bytes: two of either side
constexpr int64_t kPart = 4096;                  // its elements at the least
constexpr double kA = 3.4445, kB = -4.7750, kC = 2.0315;
constexpr float kScale = 8192.0f, kCollected = 1024.0f;    // of x, y and z, and of p, whose singular values reach 3.4445^kGroup
constexpr int kGroup = 3;
/* x of more than a tile's rows that is twice as long as wide, and so much longer,
 * takes its steps on the short side, for launches more.  So or not, us a step: 16
 * matrices of 256 x 512 268 and 246, of 256 x 640 276 and 264, of 512 x 768 439
 * and 425, of 512 x 896 450 and 446, of 512 x 1,024 465 and 473, of 512 x 2,048 610
 * and 762; 4 of 1,024 x 1,408 665 and 653, of 1,024 x 2,048 704 and 752, of 2,048 x
 * 2,560 2,836 and 2,794, of 2,048 x 4,096 3,320 and 3,958. */
constexpr int64_t kLonger = 3 * kTile;
constexpr int kSmallSide = 64, kSmallLength = 256, kSmallThreads = 512;
constexpr int kSmallTiles = kSmallSide / 16 * kSmallLength / 16 / (kSmallThreads / kWave);      // of a wave

/* A matrix of the table.  x, next, y and z are in elements of `work`, of 4
 * bytes (both halves). */
struct Matrix {
    void* param;
    int64_t rows, columns, at;                   // at: in the flat arrays
    int64_t m, n;                                // x's sides, filled up
    int64_t x, next, y, z;
    int64_t between, collected[2];               // of long ones: z y, and p by turns
    int64_t part;                                // elements of a workgroup's part of the gradient
    int64_t partial;                             // its first sum
    double decay, factor;                        // of the rate, by shape
    int type, parts;
    bool is_long;
};

struct Place {
    int matrix, i, j;
};

/* The gradients of matrices from `base` on. */
struct Gradients {
    const void* at[kBatch];                      // NULL: not stepped
    uint8_t type[kBatch];
    int base;
};

struct Common {
    const Matrix* matrices;
    const Place* places;
    float* momentum;
    float* master;
    char* work;
    double* partial;
    int* live;                                   // [matrices]: has a gradient
    float keep;                                  // momentum
    int nesterov;
    double eps, lr;
    int64_t first;                               // place of the launch's first workgroup
};

struct GradientLaunch {
    Gradients g;
    Common c;
};
static_assert(sizeof(GradientLaunch) <= kMostArguments, "kernel arguments");

}  // namespace b3p

struct B3Muon {
    int device, count;
    B3MuonConfig config;
    B3MuonState state;
    B3MuonMatrix* given;                         // host
    b3p::Matrix* matrices;                       // device
    b3p::Place* places;                          // device: of parts, cuts, half of the tiles, tiles, small ones in turn
    int64_t* first_part;                         // host: by matrix; count + 1
    int64_t* first_cut;                          // host
    int64_t cuts, halves, tiles;                 // where those places begin, after the parts
    int64_t long_halves, long_tiles, end;        // those of long matrices come last
    int64_t smalls;
    int64_t* first_small;                        // host: by matrix, of the small ones; count + 1
    char* work;                                  // device
    double* partial;                             // device
    int* live;                                   // device
};

namespace b3p {
namespace {

typedef _Float16 H8 __attribute__((ext_vector_type(8)));
typedef _Float16 H4 __attribute__((ext_vector_type(4)));
typedef short S4 __attribute__((ext_vector_type(4)));
typedef float F4 __attribute__((ext_vector_type(4)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float element(const void* p, int type, int64_t i) {
    return type == B3_F32 ? ((const float*)p)[i] : type == B3_F16 ? to_float(((const _Float16*)p)[i])
                                                                  : to_float(((const __bf16*)p)[i]);
}

/* Of workgroups in turn to the 8 dies: each die's take neighbouring places. */
__device__ __forceinline__ unsigned by_die() {
    const unsigned die = blockIdx.x % 8, share = gridDim.x / 8, rest = gridDim.x % 8;
    return die * share + (die < rest ? die : rest) + blockIdx.x / 8;
}

__device__ double block_sum(double x) {
    __shared__ double lds[kThreads / kWave];
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) x += __shfl_xor(x, d);
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; w++) x += lds[w];
    return x;
}

__device__ __forceinline__ float direction(float g, float m, const Common& c) { return c.nesterov ? g + c.keep * m : m; }

/* Four neighbours of an array of `all`, zeros past its end.  WHOLE: all there;
 * without a branch many are in flight together. */
template <bool WHOLE, typename T>
__device__ __forceinline__ F4 load4(const T* p, int64_t i, int64_t all) {
    F4 x;
    if (WHOLE || i + 4 <= all) {
        const Pack<T, 4> v = *(const Pack<T, 4>*)(p + i);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = to_float(v.v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = i + k < all ? to_float(p[i + k]) : 0.0f;
    }
    return x;
}

template <bool WHOLE, typename T>
__device__ __forceinline__ void store4(T* p, int64_t i, int64_t all, F4 x) {
    if (WHOLE || i + 4 <= all) {
        Pack<T, 4> v;
#pragma unroll
        for (int k = 0; k < 4; k++) v.v[k] = (T)x[k];
        *(Pack<T, 4>*)(p + i) = v;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (i + k < all) p[i + k] = (T)x[k];
    }
}

constexpr int kMomentumAhead = 4;

/* The momentum of a thread's elements from i0 on, the sum of squares of u. */
template <bool WHOLE, typename T>
__device__ __forceinline__ double momentum_step(const T* grad, float* momentum, int64_t i0, int64_t end, const Common& c) {
    F4 g[kMomentumAhead], m[kMomentumAhead];
    double sum = 0;
#pragma unroll
    for (int k = 0; k < kMomentumAhead; k++) {
        const int64_t i = i0 + k * kThreads * 4;
        g[k] = m[k] = F4{0, 0, 0, 0};
        if (WHOLE || i < end) {
            g[k] = load4<WHOLE>(grad, i, end);
            m[k] = load4<WHOLE>(momentum, i, end);
        }
    }
#pragma unroll
    for (int k = 0; k < kMomentumAhead; k++) {
        const int64_t i = i0 + k * kThreads * 4;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            m[k][e] = c.keep * m[k][e] + g[k][e];
            const float u = direction(g[k][e], m[k][e], c);
            sum += (double)u * u;
        }
        if (WHOLE || i < end) store4<WHOLE>(momentum, i, end, m[k]);
    }
    return sum;
}

/* Of elements from .. end - 1. */
template <typename T>
__device__ __forceinline__ double momentum_part(const T* grad, float* momentum, int64_t from, int64_t end, const Common& c) {
    constexpr int kTurn = kThreads * 4 * kMomentumAhead;
    double sum = 0;
    for (; from + kTurn <= end; from += kTurn) sum += momentum_step<true>(grad, momentum, from + threadIdx.x * 4, end, c);
    if (from < end) sum += momentum_step<false>(grad, momentum, from + threadIdx.x * 4, end, c);
    return sum;
}

/* The momentum, and a part's sum of squares of u.  Memory bounds it: 12 matrices
 * of 2,048 and 8,192 in fp32 210 us, 5.8 TB/s. */
__global__ __launch_bounds__(kThreads) void mu_momentum(GradientLaunch l) {
    const Place p = l.c.places[l.c.first + blockIdx.x];
    const Matrix& t = l.c.matrices[p.matrix];
    const void* grad = l.g.at[p.matrix - l.g.base];
    const int type = l.g.type[p.matrix - l.g.base];
    if (p.i == 0 && threadIdx.x == 0) l.c.live[p.matrix] = grad != NULL;
    if (!grad) return;
    float* momentum = l.c.momentum + t.at;
    const int64_t from = p.i * t.part, all = t.rows * t.columns, end = from + t.part < all ? from + t.part : all;
    double sum = type == B3_F32 ? momentum_part((const float*)grad, momentum, from, end, l.c)
        : type == B3_F16 ? momentum_part((const _Float16*)grad, momentum, from, end, l.c)
                         : momentum_part((const __bf16*)grad, momentum, from, end, l.c);
    sum = block_sum(sum);
    if (threadIdx.x == 0) l.c.partial[t.partial + p.i] = sum;
}

/* Where halves of row r, columns from 32 b on, lie: 32 of them, then what is
 * left of those. */
__device__ __forceinline__ _Float16* block_of(char* work, int64_t base, int64_t columns, int64_t r, int64_t b) {
    return (_Float16*)(work + base * 4 + (r * columns + b * kStep) * 4);
}

/* A square of u, scaled, turned as x lies. */
template <bool WHOLE, typename T>
__device__ __forceinline__ void first_square(float (*tile)[kCut + 1], const T* grad, const float* momentum, const Matrix& t,
    int64_t r0, int64_t c0, bool turned, const Common& c) {
    constexpr int kAcross = kCut / 4, kDown = kThreads / kAcross, kLoads = kCut / kDown;
    const int col = threadIdx.x % kAcross * 4, row = threadIdx.x / kAcross;
    F4 g[kLoads], m[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; k++) {
        const int64_t r = r0 + row + k * kDown, at = r * t.columns;
        g[k] = m[k] = F4{0, 0, 0, 0};
        if (WHOLE || (r < t.rows && c0 + col < t.columns)) {
            g[k] = load4<WHOLE>(grad + at, c0 + col, t.columns);
            m[k] = load4<WHOLE>(momentum + at, c0 + col, t.columns);
        }
    }
    /* what is fetched meanwhile waits for the norm */
    const double size = sqrt(block_sum((int)threadIdx.x < t.parts ? c.partial[t.partial + threadIdx.x] : 0.0));
    const double scale = kScale / (size + c.eps);
#pragma unroll
    for (int k = 0; k < kLoads; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float u = (float)(scale * direction(g[k][e], m[k][e], c));
            if (turned) tile[col + e][row + k * kDown] = u;
            else tile[row + k * kDown][col + e] = u;
        }
}

/* The first x, a square of it: u over its norm.  The same matrices 262 us, 4.6
 * TB/s. */
__global__ __launch_bounds__(kThreads) void mu_split(GradientLaunch l) {
    __shared__ float tile[kCut][kCut + 1];
    const Place p = l.c.places[l.c.first + blockIdx.x];
    const Matrix& t = l.c.matrices[p.matrix];
    const void* grad = l.g.at[p.matrix - l.g.base];
    const int type = l.g.type[p.matrix - l.g.base];
    if (!grad) return;
    const bool turned = t.rows > t.columns;
    const int64_t r0 = (int64_t)(turned ? p.j : p.i) * kCut, c0 = (int64_t)(turned ? p.i : p.j) * kCut;
    const float* momentum = l.c.momentum + t.at;
    auto fill = [&](const auto* g) {
        if (r0 + kCut <= t.rows && c0 + kCut <= t.columns) first_square<true>(tile, g, momentum, t, r0, c0, turned, l.c);
        else first_square<false>(tile, g, momentum, t, r0, c0, turned, l.c);
    };
    if (type == B3_F32) fill((const float*)grad);
    else if (type == B3_F16) fill((const _Float16*)grad);
    else fill((const __bf16*)grad);
    __syncthreads();
    /* a row's block of 32 to four threads of eight */
    for (int k = threadIdx.x; k < kCut * kCut / 8; k += kThreads) {
        const int r = k / (kCut / 8), b = k % (kCut / 8) / 4, o = k % 4 * 8;
        H8 h, rest;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float x = tile[r][b * kStep + o + e];
            h[e] = (_Float16)x;
            rest[e] = (_Float16)(x - (float)h[e]);
        }
        _Float16* to = block_of(l.c.work, t.x, t.n, (int64_t)p.i * kCut + r, (int64_t)p.j * (kCut / kStep) + b) + o;
        *(H8*)to = h;
        *(H8*)(to + kStep) = rest;
    }
}

enum Product { GRAM, POLYNOMIAL, MIDDLE, NEXT, LAST };

/* What a launch of mu_product does: y = x x^T (of long matrices within a
 * group z y z, from z y), z = a + b y + c y y, z y and z p of long matrices, or
 * x = z x, p x (LAST: and the weights move by it). */
struct ProductLaunch {
    Common c;
    bool swapped, swapped_long;                  // x is in `next`
    int step;                                    // of a group
    int middle;                                  // 0: z y, 1: z p; the first that the launch forms
    int64_t middles;                             // workgroups that form one of them
    int64_t before;                              // workgroups of the launches before
};

/* Where z of a long matrix' step is (the first one is p), and p after a step. */
__device__ __forceinline__ int64_t step_of(const Matrix& t, int step) { return step ? t.z : t.collected[0]; }
__device__ __forceinline__ int64_t collected_of(const Matrix& t, int step) { return t.collected[step % 2]; }

/* A weight after the step.  A copy that the weight is not rounded from has been
 * overtaken by what was written to the weight. */
template <typename T>
__device__ __forceinline__ float moved(T old, float copy, bool copied, float x, float keep, float rate) {
    float w = to_float(old);
    if (copied && to_float((T)copy) == w) w = copy;
    return w * keep - rate * x;
}

template <typename T>
__device__ __forceinline__ void move(const Common& c, const Matrix& t, int64_t i, float x, float keep, float rate) {
    T* param = (T*)t.param + i;
    float* copy = c.master && sizeof(T) == 2 ? c.master + t.at + i : NULL;
    const float w = moved(*param, copy ? *copy : 0.0f, copy != NULL, x, keep, rate);
    if (copy) *copy = w;
    *param = (T)w;
}

constexpr int kMoveRow = kTile + 4;
static_assert(kTile * kMoveRow * 4 <= kProductLds, "a tile of x");

/* The weights from row r0 and column c0 on, by a tile of x that lies as they
 * do, which `put` writes to LDS: what is fetched is on its way before. */
template <bool WHOLE, typename T, typename F>
__device__ __forceinline__ void move_tile(const Common& c, const Matrix& t, const float* tile, int64_t r0, int64_t c0, F put) {
    constexpr int kAcross = kTile / 4, kDown = kThreads / kAcross, kLoads = kTile / kDown;
    const float keep = (float)(1 - c.lr * t.decay), rate = (float)(c.lr * t.factor);
    const int col = threadIdx.x % kAcross * 4, row = threadIdx.x / kAcross;
    const bool copied = c.master && sizeof(T) == 2, in = c0 + col < t.columns;
    F4 w[kLoads], copy[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; k++) {
        const int64_t r = r0 + k * kDown + row, at = r * t.columns;
        w[k] = copy[k] = F4{0, 0, 0, 0};
        if (WHOLE || (in && r < t.rows)) {
            w[k] = load4<WHOLE>((const T*)t.param + at, c0 + col, t.columns);
            if (copied) copy[k] = load4<WHOLE>(c.master + t.at + at, c0 + col, t.columns);
        }
    }
    put();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kLoads; k++) {
        const int64_t r = r0 + k * kDown + row, at = r * t.columns;
        if (!WHOLE && (!in || r >= t.rows)) continue;
        const F4 x = *(const F4*)(tile + (k * kDown + row) * kMoveRow + col);
#pragma unroll
        for (int e = 0; e < 4; e++) w[k][e] = moved((T)w[k][e], copy[k][e], copied, x[e], keep, rate);
        if (copied) store4<WHOLE>(c.master + t.at + at, c0 + col, t.columns, w[k]);
        store4<WHOLE>((T*)t.param + at, c0 + col, t.columns, w[k]);
    }
}

/* Writes a tile's rows from r0 and blocks of columns from b0 on, a row's line of
 * 128 bytes by four threads. */
__device__ __forceinline__ void store_tile(char* work, int64_t base, int64_t columns, int64_t r0, int64_t b0,
    const uint32_t* tile) {
#pragma unroll 4
    for (int k = threadIdx.x; k < kTile * kTile / 8; k += kThreads) {
        const int row = k / (kTile / 8), o = k % (kTile / 8) * 8;
        const U4 a = *(const U4*)(tile + row * kMoveRow + o), b = *(const U4*)(tile + row * kMoveRow + o + 4);
        U4 h, rest;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            h[e] = (a[2 * e] & 0xffffu) | a[2 * e + 1] << 16;
            h[e + 2] = (b[2 * e] & 0xffffu) | b[2 * e + 1] << 16;
            rest[e] = a[2 * e] >> 16 | (a[2 * e + 1] & 0xffff0000u);
            rest[e + 2] = b[2 * e] >> 16 | (b[2 * e + 1] & 0xffff0000u);
        }
        _Float16* to = block_of(work, base, columns, r0 + row, b0 + o / kStep) + o % kStep;
        *(U4*)to = h;
        *(U4*)(to + kStep) = rest;
    }
}

/* Where the 16 bytes k of a row of 128 bytes lie: two rows to all banks, turned
 * so that 16 rows' same bytes, and neighbouring ones, lie in different banks. */
__device__ __forceinline__ int in_row(int row, int k) { return row / 2 * 256 + (row % 2 * 8 + (k ^ row / 2 % 8)) * 16; }

/* Four waves, each with 64 x 64 of the tile.  A step of 32 of what is summed
 * is fetched into registers while the two before are worked on, since one takes
 * less time than memory does, and goes to the other half of LDS.  z of 12
 * matrices of 2,048 and 8,192 takes 356 us, 923 TFLOP/s of 16-bit products (a
 * large library product reaches 1,111), z of 50 matrices of 512 wide 39 us, 620
 * TFLOP/s: of 16 steps the beginnings and ends of tiles take the most, and what
 * a launch reads and writes (130 MB, 3.3 TB/s).  The last product, with the
 * weights, takes 1,233 and 151 us (3.3 TB/s). */
template <Product KIND>
__device__ __forceinline__ void product(const ProductLaunch& l, const Place& p, bool collect) {
    constexpr bool kAcross = KIND == NEXT || KIND == LAST;      // the right side's rows are what is summed over
    constexpr int kRow = kStep * 4;                             // bytes of a row in LDS
    constexpr int kSide = kSideLds, kLoads = kTile * kStep * 4 / 16 / kThreads;
    static_assert(kTile * kRow <= kSide, "either side");
    extern __shared__ __attribute__((aligned(16))) char shared[];
    const Matrix& t = l.c.matrices[p.matrix];
    if (!l.c.live[p.matrix]) return;
    const bool swapped = t.is_long ? l.swapped_long : l.swapped;
    const int64_t x = swapped ? t.next : t.x, z = t.is_long ? step_of(t, l.step) : t.z;
    int64_t left, right, out, sum = t.m;                        // sum: a row of the left side
    float scale = 1.0f / kScale;                                // of the product
    if (KIND == GRAM) {
        const bool go_on = t.is_long && l.step;
        left = go_on ? t.between : x;
        right = go_on ? step_of(t, l.step - 1) : x;
        sum = go_on ? t.m : t.n;
        out = t.y;
    } else if (KIND == POLYNOMIAL) {
        left = right = t.y;
        out = z;
    } else if (KIND == MIDDLE) {
        left = z;
        right = collect ? collected_of(t, l.step - 1) : t.y;
        out = collect ? collected_of(t, l.step) : t.between;
        if (collect && l.step == 1) scale *= kCollected / kScale;        // p was the first z
    } else {
        left = t.is_long ? collected_of(t, l.step) : z;
        right = x;
        out = swapped ? t.x : t.next;
        if (t.is_long && l.step) scale = 1.0f / kCollected;
    }
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, g = lane / 16, c = lane % 16;
    const int wi = wave / 2 * 64, wj = wave % 2 * 64;
    const char* from_left = l.c.work + left * 4 + ((int64_t)p.i * kTile + tid / 8) * sum * 4 + tid % 8 * 16;
    const char* from_right = l.c.work + right * 4
        + (kAcross ? (int64_t)(tid / 32) * t.n * 4 + (int64_t)p.j * kTile * 4 + tid % 32 * 16
                   : ((int64_t)p.j * kTile + tid / 8) * sum * 4 + tid % 8 * 16);
    struct Fetched {
        U4 a[kLoads], b[kLoads];
    } even, odd;                                 // steps to come
    auto fetch = [&](Fetched& f, int64_t k) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            f.a[i] = *(const U4*)(from_left + i * 32 * sum * 4 + k * 4);
            f.b[i] = kAcross ? *(const U4*)(from_right + (k + i * 8) * t.n * 4) : *(const U4*)(from_right + i * 32 * sum * 4 + k * 4);
        }
    };
    auto put = [&](const Fetched& f, char* to) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            *(U4*)(to + in_row(tid / 8 + i * 32, tid % 8)) = f.a[i];
            if (kAcross) *(U4*)(to + kSide + across_row(tid / 32 + i * 8) + tid % 32 * 16) = f.b[i];
            else *(U4*)(to + kSide + in_row(tid / 8 + i * 32, tid % 8)) = f.b[i];
        }
    };
    /* eight of what is summed to a lane, from 8 g on; `rest` is 4 for those of what is left */
    auto row_of = [&](const char* at, int row, int rest) { return *(const H8*)(at + in_row(row, rest + g)); };
    /* the hardware turns four elements of 16 lanes: lane 4 r + k fetches those of row r from 4 k on */
    auto column_of = [&](const char* at) {
        typedef __attribute__((address_space(3))) S4* Lds;
        const char* q = at + across_row(8 * g + c / 4) + c % 4 * 8;
        const S4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)q);
        const S4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(q + across_row(4)));
        return __builtin_bit_cast(H8, __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    F4 d[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) d[i][j] = F4{0, 0, 0, 0};
    auto work = [&](const char* at) {
        H8 lh[4], ll[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            lh[i] = row_of(at, wi + 16 * i + c, 0);
            ll[i] = row_of(at, wi + 16 * i + c, 4);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            H8 rh, rl;
            if (kAcross) {
                const char* q = at + kSide + (wj + 16 * j) / kStep * kStep * 4 + 16 * j % kStep * 2;
                rh = column_of(q);
                rl = column_of(q + kStep * 2);
            } else {
                rh = row_of(at + kSide, wj + 16 * j + c, 0);
                rl = row_of(at + kSide, wj + 16 * j + c, 4);
            }
            /* rows of the tile along the right side's: a lane has four neighbouring columns of one row of out */
#pragma unroll
            for (int i = 0; i < 4; i++) d[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rl, lh[i], d[i][j], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) d[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rh, ll[i], d[i][j], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) d[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rh, lh[i], d[i][j], 0, 0, 0);
        }
    };
    fetch(even, 0);
    fetch(odd, kStep);
    put(even, shared);
    __syncthreads();
    /* (sums are of whole tiles: an even number of steps) */
#pragma unroll 1
    for (int64_t k = 0; k < sum; k += 2 * kStep) {
        const bool more = k + 2 * kStep < sum;
        if (more) fetch(even, k + 2 * kStep);
        work(shared);
        put(odd, shared + 2 * kSide);
        __syncthreads();
        if (more) fetch(odd, k + 3 * kStep);
        work(shared + 2 * kSide);
        if (more) put(even, shared);
        __syncthreads();
    }
    if (KIND == LAST) {
        /* to LDS as the weights lie, so that a row's neighbours are moved together */
        const bool turned = t.rows > t.columns;
        float* tile = (float*)shared;
        auto put_tile = [&]() {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int row = wi + 16 * i + c, col = wj + 16 * j + 4 * g;
                    F4 y;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        y[r] = d[i][j][r] * scale * (1.0f / kScale);
                        if (turned) tile[(col + r) * kMoveRow + row] = y[r];
                    }
                    if (!turned) *(F4*)(tile + row * kMoveRow + col) = y;
                }
        };
        const int64_t r0 = (int64_t)(turned ? p.j : p.i) * kTile, c0 = (int64_t)(turned ? p.i : p.j) * kTile;
        const bool whole = r0 + kTile <= t.rows && c0 + kTile <= t.columns;
        auto move_all = [&](auto none) {
            if (whole) move_tile<true, decltype(none)>(l.c, t, tile, r0, c0, put_tile);
            else move_tile<false, decltype(none)>(l.c, t, tile, r0, c0, put_tile);
        };
        if (t.type == B3_F32) move_all(0.0f);
        else if (t.type == B3_F16) move_all((_Float16)0.0f);
        else move_all((__bf16)0.0f);
        return;
    }
    const int64_t columns = KIND == NEXT ? t.n : t.m;
    uint32_t* tile = (uint32_t*)shared;          // halves, and what is left of them in the high bits
    U4 both[4][4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int row = wi + 16 * i + c, col = wj + 16 * j + 4 * g;
            F4 y;
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = d[i][j][r] * scale;
            if (KIND == POLYNOMIAL) {
                const int64_t at = (int64_t)p.j * kTile + col;
                const _Float16* own = block_of(l.c.work, t.y, columns, (int64_t)p.i * kTile + row, at / kStep) + at % kStep;
                const H4 h = *(const H4*)own, rest = *(const H4*)(own + kStep);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    y[r] = __builtin_fmaf((float)kC, y[r], (float)kB * ((float)h[r] + (float)rest[r]));
                    if (p.i == p.j && row == col + r) y[r] += (float)kA * kScale;
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const _Float16 h = (_Float16)y[r], rest = (_Float16)(y[r] - (float)h);
                both[i][j][r] = (uint32_t)__builtin_bit_cast(uint16_t, rest) << 16 | __builtin_bit_cast(uint16_t, h);
            }
            *(U4*)(tile + row * kMoveRow + col) = both[i][j];
        }
    __syncthreads();
    store_tile(l.c.work, out, columns, (int64_t)p.i * kTile, (int64_t)p.j * (kTile / kStep), tile);
    if (KIND == NEXT || p.i == p.j) return;
    /* and the tile across from it */
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) tile[(wj + 16 * j + 4 * g + r) * kMoveRow + wi + 16 * i + c] = both[i][j][r];
    __syncthreads();
    store_tile(l.c.work, out, columns, (int64_t)p.j * kTile, (int64_t)p.i * (kTile / kStep), tile);
}

template <Product KIND>
__global__ __launch_bounds__(kThreads, 2) void mu_product(ProductLaunch l) {
    product<KIND>(l, l.c.places[l.c.first + l.before + by_die()], false);
}

/* z y and z p of long matrices, as the launch has them, and z x of others, whose
 * places follow: neither needs the other, and together they fill the device
 * better.  Of 50 matrices of 512 wide 320 + 520 tiles take 61 us, 33 + 35 in two
 * launches, of 12 of 2,048 and 8,192 1,088 + 2,048 tiles 634, 257 + 408. */
__global__ __launch_bounds__(kThreads, 2) void mu_products(ProductLaunch l, int formed) {
    const int64_t i = l.before + by_die(), middles = l.middles * formed;
    if (i < middles) product<MIDDLE>(l, l.c.places[l.c.first + i % l.middles], l.middle + i / l.middles == 1);
    else product<NEXT>(l, l.c.places[l.c.first + l.middles + i - middles], false);
}

/* ---- small matrices ---- */

/* The quad of the sum's elements k .. k + 3 of row c, and of column c. */
__device__ __forceinline__ F4 small_row(const float* lds, int row, int stride, int k) {
    const int lane = threadIdx.x % kWave;
    return *(const F4*)(lds + (row + lane % 16) * stride + k + lane / 16 * 4);
}
__device__ __forceinline__ F4 small_column(const float* lds, int col, int stride, int k) {
    const int lane = threadIdx.x % kWave;
    const float* p = lds + (k + lane / 16 * 4) * stride + col + lane % 16;
    return F4{p[0], p[stride], p[2 * stride], p[3 * stride]};
}

__device__ __forceinline__ F4 multiply(F4 a, F4 b, F4 d) {
#pragma unroll
    for (int e = 0; e < 4; e++) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], d, 0, 0, 0);
    return d;
}

/* A matrix' whole step, in 32 bits: tiles of 16 x 16 of y and z to a wave each,
 * and of x up to kSmallTiles.  15 products that wait for each other bound it:
 * four of up to 64 x 64 32 us; 64 of 64 x 256 84 us and 512 of them 280, in
 * launches of products 194 and 451. */
__global__ __launch_bounds__(kSmallThreads) void mu_small(GradientLaunch l, int steps) {
    extern __shared__ __attribute__((aligned(16))) char shared[];
    __shared__ double sums[kSmallThreads / kWave];
    const int matrix = l.c.places[l.c.first + blockIdx.x].matrix;
    const Matrix& t = l.c.matrices[matrix];
    const void* grad = l.g.at[matrix - l.g.base];
    const int type = l.g.type[matrix - l.g.base];
    if (!grad) return;
    const bool turned = t.rows > t.columns;
    const int rows = (int)t.rows, columns = (int)t.columns, m = turned ? columns : rows, n = turned ? rows : columns;
    const int mb = (m + 15) / 16, nb = (n + 15) / 16, stride = nb * 16 + 4, side = mb * 16 + 4;
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, g = lane / 16, c = lane % 16;
    constexpr int kWaves = kSmallThreads / kWave;
    float* x = (float*)shared;
    float* y = x + mb * 16 * stride;
    float* z = y + mb * 16 * side;
    for (int i = tid; i < mb * 16 * stride; i += kSmallThreads) x[i] = 0.0f;
    __syncthreads();
    float* momentum = l.c.momentum + t.at;
    double sum = 0;
    for (int i = tid; i < rows * columns; i += kSmallThreads) {
        const float gr = element(grad, type, i), mo = l.c.keep * momentum[i] + gr, u = direction(gr, mo, l.c);
        const int r = i / columns, k = i % columns;
        momentum[i] = mo;
        x[turned ? k * stride + r : r * stride + k] = u;
        sum += (double)u * u;
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < kWaves; w++) sum += sums[w];
    const double scale = 1.0 / (sqrt(sum) + l.c.eps);
    for (int i = tid; i < mb * 16 * stride; i += kSmallThreads) x[i] = (float)(scale * x[i]);
    __syncthreads();
    for (int s = 0; s < steps; s++) {
        for (int k = wave; k < mb * mb; k += kWaves) {
            const int i = k / mb * 16, j = k % mb * 16;
            F4 d = {0, 0, 0, 0};
#pragma unroll 4
            for (int at = 0; at < nb * 16; at += 16) d = multiply(small_row(x, j, stride, at), small_row(x, i, stride, at), d);
            *(F4*)(y + (i + c) * side + j + 4 * g) = d;          // symmetric: rows or columns
        }
        __syncthreads();
        for (int k = wave; k < mb * mb; k += kWaves) {
            const int i = k / mb * 16, j = k % mb * 16;
            F4 d = {0, 0, 0, 0};
#pragma unroll 4
            for (int at = 0; at < mb * 16; at += 16) d = multiply(small_row(y, j, side, at), small_row(y, i, side, at), d);
            const F4 own = *(const F4*)(y + (i + c) * side + j + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                d[r] = __builtin_fmaf((float)kC, d[r], (float)kB * own[r]);
                if (i + c == j + 4 * g + r) d[r] += (float)kA;
            }
            *(F4*)(z + (i + c) * side + j + 4 * g) = d;
        }
        __syncthreads();
        F4 next[kSmallTiles];
#pragma unroll
        for (int k = 0; k < kSmallTiles; k++) {
            const int tile = wave + k * kWaves, i = tile / nb * 16, j = tile % nb * 16;
            next[k] = F4{0, 0, 0, 0};
            if (tile >= mb * nb) break;
#pragma unroll 4
            for (int at = 0; at < mb * 16; at += 16)
                next[k] = multiply(small_column(x, j, stride, at), small_row(z, i, side, at), next[k]);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSmallTiles; k++) {
            const int tile = wave + k * kWaves, i = tile / nb * 16, j = tile % nb * 16;
            if (tile >= mb * nb) break;
            *(F4*)(x + (i + c) * stride + j + 4 * g) = next[k];
        }
        __syncthreads();
    }
    const float keep = (float)(1 - l.c.lr * t.decay), rate = (float)(l.c.lr * t.factor);
    for (int i = tid; i < rows * columns; i += kSmallThreads) {
        const int r = i / columns, k = i % columns;
        const float v = x[turned ? k * stride + r : r * stride + k];
        if (t.type == B3_F32) move<float>(l.c, t, i, v, keep, rate);
        else if (t.type == B3_F16) move<_Float16>(l.c, t, i, v, keep, rate);
        else move<__bf16>(l.c, t, i, v, keep, rate);
    }
}

/* Bytes of LDS for sides of at most m and n. */
constexpr int small_lds(int m, int n) {
    const int mb = (m + 15) / 16 * 16, nb = (n + 15) / 16 * 16;
    return (mb * (nb + 4) + 2 * mb * (mb + 4)) * 4;
}

/* ---- launches ---- */

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


/* Tiles of a matrix (`half`: on and under the diagonal), in squares of kSquare by
 * kSquare: those that a die works on at the same time share their sides in its
 * cache. */
Place* place_tiles(Place* to, int matrix, int64_t rows, int64_t columns, bool half) {
    for (int64_t r0 = 0; r0 < rows; r0 += kSquare)
        for (int64_t c0 = 0; c0 < (half ? r0 + 1 : columns); c0 += kSquare)
            for (int64_t r = r0; r < rows && r < r0 + kSquare; r++)
                for (int64_t c = c0; c < c0 + kSquare && c < (half ? r + 1 : columns); c++)
                    *to++ = Place{matrix, (int)r, (int)c};
    return to;
}

int batch(const B3Muon* o, int base) { return o->count - base < kBatch ? o->count - base : kBatch; }

int64_t filled(int64_t n) { return ceil_div(n, kTile) * kTile; }

/* Launches over places from `first` to `end`, which may be more than one takes. */
template <typename F>
hipError_t over(int64_t first, int64_t end, F launch) {
    for (int64_t at = first; at < end; at += kMostBlocks)
        launch(at, (unsigned)(end - at < kMostBlocks ? end - at : kMostBlocks));
    return hipGetLastError();
}

template <Product KIND>
hipError_t launch_product(ProductLaunch l, int64_t first, int64_t end, hipStream_t stream) {
    l.c.first = first;
    return over(0, end - first, [&](int64_t at, unsigned blocks) {
        l.before = at;
        mu_product<KIND><<<blocks, kThreads, kProductLds, stream>>>(l);
    });
}

/* `formed` of z y and z p for the places from first to middle, then z x to end. */
hipError_t launch_products(ProductLaunch l, int64_t first, int64_t middle, int64_t end, int formed, hipStream_t stream) {
    l.c.first = first;
    l.middles = middle - first;
    return over(0, l.middles * formed + end - middle, [&](int64_t at, unsigned blocks) {
        l.before = at;
        mu_products<<<blocks, kThreads, kProductLds, stream>>>(l, formed);
    });
}

bool is_small(int64_t rows, int64_t columns) {
    const int64_t m = rows < columns ? rows : columns, n = rows < columns ? columns : rows;
    return m <= kSmallSide && n <= kSmallLength;
}

hipError_t allow_lds(const void* kernel) {
    return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kProductLds);
}

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
    void* bufs[5] = {o->matrices, o->places, o->work, o->partial, o->live};
    for (void* p : bufs) {
        hipError_t err = p ? hipFree(p) : hipSuccess;
        if (first == hipSuccess) first = err;
    }
    free(o->given);
    free(o->first_part);
    free(o->first_cut);
    free(o->first_small);
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
    o->first_part = (int64_t*)calloc((size_t)count + 1, sizeof(int64_t));
    o->first_cut = (int64_t*)calloc((size_t)count + 1, sizeof(int64_t));
    o->first_small = (int64_t*)calloc((size_t)count + 1, sizeof(int64_t));
    Matrix* table = (Matrix*)calloc((size_t)count + 1, sizeof(Matrix));
    Place* places = NULL;
    int64_t work = 0, partials = 0;
    hipError_t err = !(o->given && o->first_part && o->first_cut && o->first_small && table) ? hipErrorOutOfMemory
        : overlap(matrices, count, o->given) ? hipErrorInvalidValue : hipGetDevice(&o->device);
    if (err == hipSuccess) {
        int64_t at = 0, parts = 0, cuts = 0, small = 0, halves[2] = {0, 0}, tiles[2] = {0, 0};
        for (int i = 0; i < count; i++) {
            const B3MuonMatrix& g = o->given[i] = matrices[i];
            Matrix& t = table[i];
            const int64_t numel = g.rows * g.columns, m = g.rows < g.columns ? g.rows : g.columns;
            t.param = g.param;
            t.rows = g.rows;
            t.columns = g.columns;
            t.at = at;
            at += segment(numel);
            t.type = g.type;
            t.decay = g.weight_decay;
            t.factor = g.rows > g.columns && g.columns ? sqrt((double)g.rows / (double)g.columns) : 1.0;
            o->first_part[i] = parts;
            o->first_cut[i] = cuts;
            o->first_small[i] = small;
            if (!numel) continue;
            if (is_small(g.rows, g.columns)) {
                small++;
                continue;
            }
            t.m = filled(m);
            t.n = filled(numel / m);
            t.is_long = t.m > kTile && t.n >= 2 * t.m && t.n >= t.m + kLonger;
            int64_t* const squares[5] = {&t.y, &t.z, &t.between, &t.collected[0], &t.collected[1]};
            t.x = work;
            t.next = t.x + t.m * t.n;
            work = t.next + t.m * t.n;
            for (int k = 0; k < (t.is_long ? 5 : 2); k++) {
                *squares[k] = work;
                work += t.m * t.m;
            }
            t.part = ceil_div(numel, kMostParts);
            t.part = t.part < kPart ? kPart : t.part;
            t.parts = (int)ceil_div(numel, t.part);
            t.partial = partials;
            partials += t.parts;
            const int64_t mt = t.m / kTile, nt = t.n / kTile, per = kTile / kCut;
            parts += t.parts;
            cuts += mt * nt * per * per;
            halves[t.is_long] += mt * (mt + 1) / 2;
            tiles[t.is_long] += mt * nt;
        }
        o->first_part[count] = parts;
        o->first_cut[count] = cuts;
        o->first_small[count] = small;
        o->cuts = parts;
        o->halves = o->cuts + cuts;
        o->long_halves = o->halves + halves[0];
        o->tiles = o->long_halves + halves[1];
        o->long_tiles = o->tiles + tiles[0];
        o->end = o->long_tiles + tiles[1];
        places = (Place*)malloc((size_t)(o->end + small + 1) * sizeof(Place));
        if (!places) err = hipErrorOutOfMemory;
        Place* to = places;
        for (int i = 0; i < count && places; i++)
            for (int k = 0; k < table[i].parts; k++) *to++ = Place{i, k, 0};
        for (int i = 0; i < count && places; i++)
            for (int64_t r = 0; r < table[i].m / kCut; r++)
                for (int64_t c = 0; c < table[i].n / kCut; c++) *to++ = Place{i, (int)r, (int)c};
        for (int k = 0; k < 4 && places; k++)            // half of the tiles, then all, and of both long matrices last
            for (int i = 0; i < count; i++)
                if (table[i].is_long == k % 2) to = place_tiles(to, i, table[i].m / kTile, table[i].n / kTile, k < 2);
        for (int i = 0; i < count && places; i++)
            if (o->first_small[i + 1] > o->first_small[i]) *to++ = Place{i, 0, 0};
        o->smalls = small;
    }
    if (err == hipSuccess) err = hipMalloc((void**)&o->matrices, ((size_t)count + 1) * sizeof(Matrix));
    if (err == hipSuccess) err = hipMalloc((void**)&o->places, (size_t)(o->end + o->smalls + 1) * sizeof(Place));
    if (err == hipSuccess) err = hipMalloc((void**)&o->work, (size_t)(work + 1) * 4);
    if (err == hipSuccess) err = hipMalloc((void**)&o->partial, (size_t)(partials + 1) * sizeof(double));
    if (err == hipSuccess) err = hipMalloc((void**)&o->live, ((size_t)count + 1) * sizeof(int));
    if (err == hipSuccess) err = hipMemcpy(o->matrices, table, ((size_t)count + 1) * sizeof(Matrix), hipMemcpyHostToDevice);
    if (err == hipSuccess) err = hipMemcpy(o->places, places, (size_t)(o->end + o->smalls) * sizeof(Place), hipMemcpyHostToDevice);
    if (err == hipSuccess) err = allow_lds((const void*)mu_product<GRAM>);
    if (err == hipSuccess) err = allow_lds((const void*)mu_product<POLYNOMIAL>);
    if (err == hipSuccess) err = allow_lds((const void*)mu_products);
    if (err == hipSuccess) err = allow_lds((const void*)mu_product<NEXT>);
    if (err == hipSuccess) err = allow_lds((const void*)mu_product<LAST>);
    if (err == hipSuccess)
        err = hipFuncSetAttribute((const void*)mu_small, hipFuncAttributeMaxDynamicSharedMemorySize,
            small_lds(kSmallSide, kSmallLength));
    free(table);
    free(places);
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
    GradientLaunch l = {};
    l.c.matrices = o->matrices;
    l.c.places = o->places;
    l.c.momentum = o->state.momentum;
    l.c.master = o->state.master;
    l.c.work = o->work;
    l.c.partial = o->partial;
    l.c.live = o->live;
    l.c.keep = (float)o->config.momentum;
    l.c.nesterov = o->config.nesterov;
    l.c.eps = o->config.eps;
    l.c.lr = lr;
    for (int base = 0; base < o->count; base += kBatch) {
        const int n = batch(o, base);
        l.g.base = base;
        for (int j = 0; j < n; j++) {
            l.g.at[j] = grads[base + j];
            l.g.type[j] = (uint8_t)(grad_types ? grad_types[base + j] : o->given[base + j].type);
        }
        err = over(o->first_part[base], o->first_part[base + n], [&](int64_t at, unsigned blocks) {
            l.c.first = at;
            mu_momentum<<<blocks, kThreads, 0, stream>>>(l);
        });
        if (err != hipSuccess) return err;
        err = over(o->end + o->first_small[base], o->end + o->first_small[base + n], [&](int64_t at, unsigned blocks) {
            l.c.first = at;
            mu_small<<<blocks, kSmallThreads, small_lds(kSmallSide, kSmallLength), stream>>>(l, o->config.newton_schulz);
        });
        if (err != hipSuccess) return err;
        err = over(o->cuts + o->first_cut[base], o->cuts + o->first_cut[base + n], [&](int64_t at, unsigned blocks) {
            l.c.first = at;
            mu_split<<<blocks, kThreads, 0, stream>>>(l);
        });
        if (err != hipSuccess) return err;
    }
    const int steps = o->config.newton_schulz;
    ProductLaunch p = {l.c, false, false, 0, 0, 0, 0};
    for (int s = 0; s < steps && o->halves < o->end && err == hipSuccess; s++) {
        const bool last = s + 1 == steps, joined = last || p.step + 1 == kGroup;     // long x becomes its next
        err = launch_product<GRAM>(p, o->halves, o->tiles, stream);
        if (err == hipSuccess) err = launch_product<POLYNOMIAL>(p, o->halves, o->tiles, stream);
        p.middle = joined ? 1 : 0;
        const int formed = (joined ? 0 : 1) + (p.step ? 1 : 0);
        if (err == hipSuccess) err = launch_products(p, o->long_halves, o->tiles, last ? o->tiles : o->long_tiles, formed, stream);
        if (err == hipSuccess && last) err = launch_product<LAST>(p, o->tiles, o->end, stream);
        else if (err == hipSuccess && joined) err = launch_product<NEXT>(p, o->long_tiles, o->end, stream);
        p.swapped = !p.swapped;
        p.swapped_long ^= joined;
        p.step = joined ? 0 : p.step + 1;
    }
    return err;
}

}  // extern "C"
