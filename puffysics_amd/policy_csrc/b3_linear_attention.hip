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
 * does all four: a wave takes a sequence (an environment's head) and a part of
 * v's columns, holds the state in the accumulators of the matrix units, and
 * goes over chunks of 32 steps (16 in 32 bits), within which the steps are
 * products of matrices.  No wave waits for another.  Where sequences are few
 * their steps are cut into pieces: a first launch finds what state each leaves,
 * a second adds up, and the third goes over all pieces at once.
 */
#include "policy_common.h"

namespace b3p {
namespace {

constexpr int kThreads = 256;
constexpr int kRoles = 3;                        // of a launch
static_assert((int64_t)B3_MAX_SEQUENCES * kRoles * kThreads < (int64_t)1 << 32, "threads of a launch");
constexpr int64_t kAlone = 1024, kFull = 2048;   // waves with a SIMD to themselves, and two to each
constexpr float kHold = 256.0f;                  // a state is held as between itself and 1 / kHold of it

/* out_p = `reach` q_p (decay^p E + sums over p' <= p of the episode of
 * `update` decay^(p - p') k_p'^T v_p'), and the state that is left,
 * decay^steps E + sums of `update` decay^(steps - p') k_p'^T v_p'.  Places p
 * follow the steps, or go from the last one back.  Forwards E is a step
 * earlier (decayed before place 0), and the state is left a step earlier (not
 * decayed after the last place). */
struct Mix {
    const void *q, *k, *v;
    void* out;
    int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];   // place, environment, head
    int key, value;
    float reach, update;
    bool forward;
    const char* starts;                          // of place 0 (which has none on the way back), or NULL
    int64_t starts_stride[2];                    // in bytes
    const float* enter;                          // E, NULL: zeros
    float* leave;                                // NULL: not wanted
    int64_t state_row, state_col;                // of both and of the pieces', in elements
    const char* leave_starts;                    // [environments], dropped where nonzero; or NULL
    int64_t leave_starts_stride;
    float* pieces;                               // [pieces - 1][sequences][key value]: what each leaves
    float* carry;                                // [pieces - 1][sequences]: decay over it, < 0 where it drops what enters
};

struct Job {
    Mix mix[kRoles];
    int64_t steps, envs, heads;
    const float* decay;
    int starts_type;
    int roles, parts;                            // parts: of v's columns
    int64_t places, pieces;                      // places: of a piece
};

__device__ __forceinline__ bool started(const char* p, int type) {
    return type == B3_F32 ? *(const float*)p != 0.0f : *(const unsigned char*)p != 0;
}

/* A head's decay: NaN outside of [0, 1]. */
__device__ __forceinline__ float decay_of(const float* decay, int64_t head) {
    const float d = decay[head];
    return d >= 0.0f && d <= 1.0f ? d : NAN;
}

/* ---- a wave's work on a sequence ---- */

typedef float F4 __attribute__((ext_vector_type(4)));
typedef short S4 __attribute__((ext_vector_type(4)));
typedef short S8 __attribute__((ext_vector_type(8)));
typedef __bf16 B4 __attribute__((ext_vector_type(4)));
typedef __bf16 B8 __attribute__((ext_vector_type(8)));
typedef _Float16 H8 __attribute__((ext_vector_type(8)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));

/* What the arithmetic goes by.  Lane (g, c) = (lane / 16, lane % 16) holds of
 * 16 x 16 operands the four elements 4 g .. 4 g + 3 along the axis that is
 * summed, of row or column c: a quad.  A product's tile lies the same way, so
 * that it is an operand of the next without a move between lanes. */
template <typename T>
struct Math {                                    // 32-bit products: of float, and of halves, whose scores could overflow
    typedef float Lds;
    typedef F4 Quad;
    static constexpr int kPlaces = 16;           // of a chunk
};
template <>
struct Math<__bf16> {
    typedef __bf16 Lds;
    typedef S4 Quad;
    static constexpr int kPlaces = 32;
};

__device__ __forceinline__ S4 round4(F4 x) { return __builtin_bit_cast(S4, __builtin_convertvector(x, B4)); }
/* What rounding left out, and that rounded. */
__device__ __forceinline__ F4 left4(F4 x, S4 rounded) { return x - __builtin_convertvector(__builtin_bit_cast(B4, rounded), F4); }
__device__ __forceinline__ S4 rest4(F4 x, S4 rounded) { return round4(left4(x, rounded)); }

/* d += a b over two blocks of 16. */
__device__ __forceinline__ F4 multiply(S4 a0, S4 a1, S4 b0, S4 b1, F4 d) {
    const S8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
    const S8 b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), d, 0, 0, 0);
}

/* Over one block. */
__device__ __forceinline__ F4 multiply(F4 a, F4 b, F4 d) {
#pragma unroll
    for (int e = 0; e < 4; e++) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], d, 0, 0, 0);
    return d;
}

/* Keeps a wave's writes to LDS before the reads of its other lanes; the
 * hardware does them in order. */
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/* decay^n, 1 for n = 0. */
__device__ __forceinline__ float power(float log2_decay, int n) {
    return n == 0 ? 1.0f : __builtin_amdgcn_exp2f((float)n * log2_decay);
}

/* An array's part of a chunk: COLS columns of kPlaces rows, in vectors of 16
 * bytes, in registers until the chunk before is done and then in LDS, whose
 * rows are 16 bytes longer so that 16 rows' neighbouring columns lie in other
 * banks.  W waves share it, and each moves every W-th of its vectors. */
template <typename T, int COLS, int W>
struct Tile {
    typedef typename Math<T>::Lds Lds;
    static constexpr int kVec = 16 / sizeof(T), kRow = COLS + 16 / sizeof(Lds), kPlaces = Math<T>::kPlaces;
    static constexpr int kPerRow = COLS / kVec, kRows = kWave / kPerRow, kLoads = kPlaces / (kRows * W);
    static constexpr int kBytes = kPlaces * kRow * sizeof(Lds);
    static_assert(kWave % kPerRow == 0 && kPlaces % (kRows * W) == 0, "whole loads");
    U4 raw[kLoads];

    /* Vector l of a lane is of row(l), from col() on. */
    static __device__ __forceinline__ int row(int l) { return l * (kRows * W) + (int)threadIdx.x % (kWave * W) / kPerRow; }
    static __device__ __forceinline__ int col() { return (int)threadIdx.x % kPerRow * kVec; }

    /* Columns from p on, of which there are `cols`, and `places` rows (at least 1).
     * What lies beyond is not fetched, but no branch of a lane's is taken for it, so
     * that all loads are in flight together: a lane that has fewer columns left than
     * a vector, or none, fetches the row's last ones, rows beyond are the last one
     * again.  fit_columns() is for when they have come: sooner it would wait for them. */
    __device__ __forceinline__ void load(const T* p, int64_t stride, int places, int cols) {
        int first = col() + kVec <= cols ? col() : cols - kVec;
        if (cols >= kVec && places == kPlaces) {
            const T* at = p + row(0) * stride + first;
#pragma unroll
            for (int l = 0; l < kLoads; l++) raw[l] = __builtin_bit_cast(U4, *(const Pack<T, kVec>*)(at + l * (kRows * W * stride)));
        } else {
            /* (values of their own, so that nothing of this is formed ahead of the loop and held) */
            asm volatile("" : "+s"(stride), "+v"(first));
#pragma unroll
            for (int l = 0; l < kLoads; l++) {
                const T* at = p + (row(l) < places ? row(l) : places - 1) * stride;
                Pack<T, kVec> x;
                if (cols >= kVec) {
                    x = *(const Pack<T, kVec>*)(at + first);
                } else {
#pragma unroll
                    for (int i = 0; i < kVec; i++) x.v[i] = at[i < cols ? i : 0];
                }
                raw[l] = __builtin_bit_cast(U4, x);
            }
            rows_beyond(places);                 // (nothing follows such a chunk)
        }
    }

    /* Zeros for columns beyond; the last ones moved to where they belong. */
    __device__ __forceinline__ void fit_columns(int cols) {
        if (cols < COLS) {
            const int left = cols - col();       // of a lane
            if (cols % kVec) {
                const bool some = left > 0 && left < kVec;
                const int by = cols >= kVec ? (kVec - cols % kVec) * (int)sizeof(T) : 0;
#pragma unroll
                for (int l = 0; l < kLoads; l++) {
                    U4 x = raw[l];
                    if (by & 8) x = U4{x[2], x[3], 0, 0};
                    if (by & 4) x = U4{x[1], x[2], x[3], 0};
                    if (by & 2) x = U4{x[0] >> 16 | x[1] << 16, x[1] >> 16 | x[2] << 16, x[2] >> 16 | x[3] << 16, x[3] >> 16};
                    if (cols < kVec) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int n = cols * (int)sizeof(T) - 4 * i;      // bytes
                            x[i] = n >= 4 ? x[i] : n == 2 ? x[i] & 0xffffu : 0;
                        }
                    }
                    if (some) raw[l] = x;
                }
            }
#pragma unroll
            for (int l = 0; l < kLoads; l++)
                if (left <= 0) raw[l] = U4{0, 0, 0, 0};
        }
    }

    /* Zeros from row `places` on. */
    __device__ __forceinline__ void rows_beyond(int places) {
#pragma unroll
        for (int l = 0; l < kLoads; l++)
            if (row(l) >= places) raw[l] = U4{0, 0, 0, 0};
    }

    __device__ __forceinline__ void none() {
#pragma unroll
        for (int l = 0; l < kLoads; l++) raw[l] = U4{0, 0, 0, 0};
    }

    /* Adds to sums in turn what is NaN in some lane if any element of the chunk is
     * NaN or infinite, else 0: the elements' products with 0, which the matrix
     * units form as they lie. */
    __device__ __forceinline__ void times_0(F4 sum[4]) const {
#pragma unroll
        for (int l = 0; l < kLoads; l++) {
            if constexpr (__is_same(T, __bf16)) {
                sum[l % 4] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(B8, raw[l]), B8{}, sum[l % 4], 0, 0, 0);
            } else if constexpr (__is_same(T, _Float16)) {
                sum[l % 4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(H8, raw[l]), H8{}, sum[l % 4], 0, 0, 0);
            } else {
                sum[l % 4] = __builtin_elementwise_fma(__builtin_bit_cast(F4, raw[l]), F4{0, 0, 0, 0}, sum[l % 4]);
            }
        }
    }

    __device__ __forceinline__ void put(Lds* lds, int r, int c, U4 x) const {
        if (sizeof(T) == sizeof(Lds)) {
            *(U4*)(lds + r * kRow + c) = x;
        } else {
            const Pack<_Float16, 8> h = __builtin_bit_cast(Pack<_Float16, 8>, x);
            F4 a, b;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                a[i] = (float)h.v[i];
                b[i] = (float)h.v[i + 4];
            }
            *(F4*)(lds + r * kRow + c) = a;
            *(F4*)(lds + r * kRow + c + 4) = b;
        }
    }

    __device__ __forceinline__ void store(Lds* lds) const {
#pragma unroll
        for (int l = 0; l < kLoads; l++)
            put(lds, row(l), col(), raw[l]);
    }
};

/* The quad of row c of 16 from `row` on, columns from `col` on. */
template <int ROW>
__device__ __forceinline__ S4 along(const __bf16* lds, int row, int col) {
    const int lane = threadIdx.x % kWave;
    return *(const S4*)(lds + (row + lane % 16) * ROW + col + lane / 16 * 4);
}
template <int ROW>
__device__ __forceinline__ F4 along(const float* lds, int row, int col) {
    const int lane = threadIdx.x % kWave;
    return *(const F4*)(lds + (row + lane % 16) * ROW + col + lane / 16 * 4);
}

/* The quad of a column, rows from `row` on.  The column of c is first(c / 4) +
 * c % 4 with first(n) = col + STEP n.  In 16 bits the hardware turns the four
 * elements of 16 lanes: lane 4 a + b fetches those of row a, columns first(b)
 * on, and lane c gets the column of c. */
template <int ROW, int STEP>
__device__ __forceinline__ S4 across(const __bf16* lds, int row, int col) {
    const int lane = threadIdx.x % kWave, g = lane / 16, a = lane % 16 / 4, b = lane % 4;
    const __bf16* p = lds + (row + 4 * g + a) * ROW + col + STEP * b;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S4*)(p));
}
template <int ROW, int STEP>
__device__ __forceinline__ F4 across(const float* lds, int row, int col) {
    const int lane = threadIdx.x % kWave, g = lane / 16, c = lane % 16;
    const float* p = lds + (row + 4 * g) * ROW + col + STEP * (c / 4) + c % 4;
    return F4{p[0], p[ROW], p[2 * ROW], p[3 * ROW]};
}

/* Where a unit's work lies. */
struct Unit {
    int64_t env, head, piece;
    int role, first;                             // first: column of v
};

/* A wave goes over the places of a piece of a sequence, a chunk at a time, KD
 * the columns of q and k and VD those of its part of v, both filled up with
 * zeros; STATE: without out, to learn what state the piece leaves.  W waves, a
 * workgroup where W > 1, have parts of one sequence and share q and k.  With i
 * and j places of the chunk, E the state that enters it and P the scores q_i k_j
 * decay^(i - j) of an episode, j <= i:
 *   out = P v + decay^i q E,  E' = decay^places E + (decay^(places - j) k)^T v
 * PART: some columns are filled up.  Tiles of 16 that all are, are left out of
 * products, which in 32 bits are most of the time: 333 steps of 57 x 3 with heads
 * of 48 and 80 take 56 us forward and 98 back so, 70 and 140 without.  Where none
 * are, asking costs 2 to 7 % (fp32 and fp16 heads of 64 and of 128).
 * 64 steps of 4,096 environments with 4 heads of 64 in bf16 take 190 us forward
 * (4.3 TB/s, vector units 35 % busy, matrix units 10) and 402 back (3.0 TB/s, 43
 * and 13), two histories of 65,536 steps and 8 heads of 128 152 us for the
 * pieces' states and 361 for all (3.1 TB/s, 56 and 29): what bounds it is that
 * the registers hold but two waves of a SIMD, which wait for each other's
 * instructions more than for memory.  The same 64 steps, call after call, with the
 * last state, no episodes and none to enter with: bf16 222 and 310, fp16 262 and
 * 546, fp32 306 and 597, whose products bound them. */
template <typename T, int KD, int VD, int W, bool STATE, bool PART>
struct Walk {
    typedef typename Math<T>::Lds Lds;
    typedef typename Math<T>::Quad Quad;
    static constexpr bool kHalf = sizeof(Lds) == 2;
    static constexpr int kPlaces = Math<T>::kPlaces, R = kPlaces / 16, KB = KD / 16, VB = VD / 16;
    typedef Tile<T, KD, W> KeyTile;
    typedef Tile<T, VD, 1> ValueTile;
    static constexpr int kKeyRow = KeyTile::kRow, kValueRow = ValueTile::kRow;
    static constexpr int kBytes = (STATE ? 1 : 2) * KeyTile::kBytes + W * ValueTile::kBytes + (W > 1 ? 16 : 0);
    /* in 16 bits two tiles' columns are dealt out so that a lane has eight neighbours of them */
    static constexpr int kStep = kHalf ? 8 : 4;
    static __device__ __forceinline__ int value_col(int vb) { return kHalf ? vb / 2 * 32 + vb % 2 * 4 : vb * 16; }

    static __device__ __forceinline__ Quad with(F4 x) {
        if constexpr (kHalf) return round4(x);
        else return x;
    }

    static __device__ __forceinline__ void fence() {
        if (W == 1) wave_fence();
        else __syncthreads();
    }

    static __device__ __forceinline__ void run(const Job& j, const Mix& m, const Unit& u, int64_t from, int64_t places, const float* enter,
        bool early, float* leave, float* carry, char* shared) {
        const int lane = threadIdx.x % kWave, g = lane / 16, c = lane % 16;
        const int wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        Lds* lk = (Lds*)shared;
        Lds* lv = (Lds*)(shared + KeyTile::kBytes + wave * ValueTile::kBytes);
        Lds* lq = (Lds*)(shared + KeyTile::kBytes + W * ValueTile::kBytes);
        int* bad = (int*)(shared + kBytes - 16);                    // of each wave
        const float l2 = log2f(decay_of(j.decay, u.head));
        const T* q = (const T*)m.q + from * m.q_stride[0] + u.env * m.q_stride[1] + u.head * m.q_stride[2];
        const T* k = (const T*)m.k + from * m.k_stride[0] + u.env * m.k_stride[1] + u.head * m.k_stride[2];
        const T* v = (const T*)m.v + from * m.v_stride[0] + u.env * m.v_stride[1] + u.head * m.v_stride[2] + u.first;
        T* out = (T*)m.out + from * m.out_stride[0] + u.env * m.out_stride[1] + u.head * m.out_stride[2] + u.first;
        const int value = m.value - u.first < VD ? m.value - u.first : VD;
        const bool active = W == 1 || value > 0;                    // else it has q and k to move alone

        /* weights of scores (of the tiles i = j and i = j + 16), of the state for place i, and of places for the state */
        const float gain = m.reach * m.update;
        F4 near[R];
        float reach[R];
#pragma unroll
        for (int t = 0; t < R; t++) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int n = 16 * t + c - 4 * g - r;
                near[t][r] = n >= 0 ? gain * power(l2, n) : 0.0f;
            }
            reach[t] = m.reach * power(l2, 16 * t + c);
        }
        F4 keep[R];
        int weighted = -1;                       // places and the step less that keep is for

        KeyTile tk, tq;
        ValueTile tv;
        uint32_t flag = 0;
        bool dropped = false;
        /* of the state: top decay^held, from its one rounding to 32 bits (a chunk's power times itself would add up) */
        float scale, top = kHold;
        int held = 0;
        bool any = enter != NULL;                // state
        auto fetch = [&](int64_t p) {
            const int n = places - p < kPlaces ? (int)(places - p) : kPlaces;
            tk.load(k + p * m.k_stride[0], m.k_stride[0], n, m.key);
            if (active) tv.load(v + p * m.v_stride[0], m.v_stride[0], n, value);
            if (!STATE) tq.load(q + p * m.q_stride[0], m.q_stride[0], n, m.key);
            if (m.starts) {
                /* the first place on the way back has none: a later one's is fetched, and dropped */
                const int at = lane < n ? lane : n - 1, none = from + p == 0 && !m.forward ? 1 : 0;
                if (n > none)
                    flag = started(m.starts + (from + p + (at > none ? at : none)) * m.starts_stride[0] + u.env * m.starts_stride[1],
                        j.starts_type) && lane < n && lane >= none;
                else
                    flag = 0;
            }
        };
        if (W > 1) tv.none();
        if (places > 0) fetch(0);
        /* E, lane (g, c) of tile [kb][vb] rows 16 kb + 4 g + r and the column of c */
        F4 state[KB][VB];
        const int state_row = (int)m.state_row, state_col = (int)m.state_col;
        if (enter && active) {
            const float* at[VB];
#pragma unroll
            for (int vb = 0; vb < VB; vb++) {
                const int col = value_col(vb) + kStep * (c / 4) + c % 4;
                at[vb] = enter + (u.first + (col < value ? col : 0)) * state_col;
            }
            /* (a transposed state's four rows are neighbours) */
            if (state_row == 1 && m.key % 4 == 0) {
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) {
                        const int row = kb * 16 + 4 * g;
                        state[kb][vb] = __builtin_bit_cast(F4, *(const Pack<float, 4>*)(at[vb] + (row < m.key ? row : 0)));
                    }
            } else {
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int row = kb * 16 + 4 * g + r, offset = (row < m.key ? row : 0) * state_row;
#pragma unroll
                        for (int vb = 0; vb < VB; vb++) state[kb][vb][r] = at[vb][offset];
                    }
            }
            top = 1.0f;
            held = early ? 1 : 0;
            if (m.key < KD || value < VD) {
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int vb = 0; vb < VB; vb++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int row = kb * 16 + 4 * g + r, col = value_col(vb) + kStep * (c / 4) + c % 4;
                            if (row >= m.key || col >= value) state[kb][vb][r] = 0.0f;
                        }
            }
        } else {
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int vb = 0; vb < VB; vb++) state[kb][vb] = F4{0, 0, 0, 0};
        }

        scale = top * power(l2, held);
        int n;
#pragma unroll 1
        for (int64_t p = 0; p < places; p += n) {
            n = places - p < kPlaces ? (int)(places - p) : kPlaces;
            /* A product with a weight of 0 would carry what is not finite in k or v to other places:
             * such a place is a chunk by itself. */
            F4 zero[4] = {};
            if (PART) {
                tk.fit_columns(m.key);
                if (active) tv.fit_columns(value);
                if (!STATE) tq.fit_columns(m.key);
            }
            tk.times_0(zero);
            tv.times_0(zero);
            zero[0] = zero[0] + zero[1] + (zero[2] + zero[3]);
            const bool found = __ballot(zero[0][0] + zero[0][1] + (zero[0][2] + zero[0][3]) != 0.0f) != 0;
            auto alone = [&]() {
                n = 1;
                tk.rows_beyond(1);
                tv.rows_beyond(1);
                if (!STATE) tq.rows_beyond(1);
            };
            auto stage = [&]() {
                fence();
                tk.store(lk);
                tv.store(lv);
                if (!STATE) tq.store(lq);
                if (W > 1 && lane == 0) bad[wave] = found;
                fence();
            };
            if (W == 1 && found && n > 1) alone();
            stage();
            if (W > 1 && n > 1) {
                int any_found = 0;
#pragma unroll
                for (int w = 0; w < W; w++) any_found |= bad[w];
                if (any_found) {
                    alone();
                    stage();
                }
            }
            const uint32_t starts = (uint32_t)__ballot(flag != 0 && lane < n);
            const bool end = p + n >= places;
            if (!end) fetch(p + n);
            if (!active) {
                if (end) break;
                continue;
            }
            Quad vq[R][VB];
#pragma unroll
            for (int t = 0; t < R; t++)
#pragma unroll
                for (int vb = 0; vb < VB; vb++) vq[t][vb] = across<kValueRow, kStep>(lv, 16 * t, value_col(vb));

            if (!STATE) {
                Quad qq[R][KB];
#pragma unroll
                for (int t = 0; t < R; t++)
#pragma unroll
                    for (int kb = 0; kb < KB; kb++) qq[t][kb] = along<kKeyRow>(lq, 16 * t, 16 * kb);
                /* of place i = 16 t + c the last start at or before it */
                int since[R];
#pragma unroll
                for (int t = 0; t < R; t++) {
                    const uint32_t before = starts & (uint32_t)((2ull << (16 * t + c)) - 1);
                    since[t] = before ? 31 - __builtin_clz(before) : -1;
                }
                /* scores, rows j and columns i; they are what P v sums over as they lie, in 16 bits as two numbers */
                Quad score[R][R], rest[R][R];
#pragma unroll
                for (int s = 0; s < R; s++) {
                    Quad kq[KB];
#pragma unroll
                    for (int kb = 0; kb < KB; kb++) kq[kb] = along<kKeyRow>(lk, 16 * s, 16 * kb);
#pragma unroll
                    for (int t = s; t < R; t++) {
                        F4 x = {0, 0, 0, 0};
                        if constexpr (kHalf) {
#pragma unroll
                            for (int kb = 0; kb < KB; kb += 2) x = multiply(kq[kb], kq[kb + 1], qq[t][kb], qq[t][kb + 1], x);
                        } else {
#pragma unroll
                            for (int kb = 0; kb < KB; kb++) {
                                if (PART && 16 * kb >= m.key) break;
                                x = multiply(kq[kb], qq[t][kb], x);
                            }
                        }
                        x *= near[t - s];
                        if (t == s) {
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                if (4 * g + r > c) x[r] = 0.0f;
                        }
                        if (starts) {
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                if (16 * s + 4 * g + r < since[t]) x[r] = 0.0f;
                        }
                        score[t][s] = with(x);
                        if constexpr (kHalf) rest[t][s] = rest4(x, score[t][s]);
                    }
                }
                /* kTiles tiles of columns at a time, which a lane writes together */
                constexpr int kTiles = kHalf ? 2 : 1, kWide = 4 * kTiles;
#pragma unroll
                for (int v0 = 0; v0 < VB; v0 += kTiles) {
                    if (PART && 16 * v0 >= value) break;
                    F4 o[R][kTiles];
#pragma unroll
                    for (int t = 0; t < R; t++)
#pragma unroll
                        for (int i = 0; i < kTiles; i++) o[t][i] = F4{0, 0, 0, 0};
                    if (any) {
                        /* q E: in 16 bits E as two numbers */
#pragma unroll
                        for (int i = 0; i < kTiles; i++) {
                            const int vb = v0 + i;
                            if constexpr (kHalf) {
#pragma unroll
                                for (int kb = 0; kb < KB; kb += 2) {
                                    const S4 h0 = round4(state[kb][vb]), h1 = round4(state[kb + 1][vb]);
                                    const S4 l0 = rest4(state[kb][vb], h0), l1 = rest4(state[kb + 1][vb], h1);
#pragma unroll
                                    for (int t = 0; t < R; t++) o[t][i] = multiply(l0, l1, qq[t][kb], qq[t][kb + 1], o[t][i]);
#pragma unroll
                                    for (int t = 0; t < R; t++) o[t][i] = multiply(h0, h1, qq[t][kb], qq[t][kb + 1], o[t][i]);
                                }
                            } else {
#pragma unroll
                                for (int kb = 0; kb < KB; kb++) {
                                    if (PART && 16 * kb >= m.key) break;
#pragma unroll
                                    for (int t = 0; t < R; t++) o[t][i] = multiply(state[kb][vb], qq[t][kb], o[t][i]);
                                }
                            }
                        }
#pragma unroll
                        for (int t = 0; t < R; t++)
#pragma unroll
                            for (int i = 0; i < kTiles; i++) {
                                o[t][i] *= reach[t] * scale;
                                if (starts && since[t] >= 0) o[t][i] = F4{0, 0, 0, 0};
                            }
                    }
#pragma unroll
                    for (int t = 0; t < R; t++)
#pragma unroll
                        for (int i = 0; i < kTiles; i++) {
                            if constexpr (kHalf) {
                                o[t][i] = multiply(vq[0][v0 + i], vq[1][v0 + i], rest[t][0], t ? rest[1][1] : S4{0, 0, 0, 0}, o[t][i]);
                                o[t][i] = multiply(vq[0][v0 + i], vq[1][v0 + i], score[t][0], t ? score[1][1] : S4{0, 0, 0, 0}, o[t][i]);
                            } else {
                                o[t][i] = multiply(vq[0][v0 + i], score[0][0], o[t][i]);
                            }
                        }
                    /* lane (g, c): of place 16 t + c the columns 4 g + r of each tile */
                    const int col = value_col(v0) + kWide * g;
#pragma unroll
                    for (int t = 0; t < R; t++) {
                        const int at = 16 * t + c;
                        if (at >= n || !m.out) continue;
                        T* to = out + (p + at) * m.out_stride[0];
                        Pack<T, kWide> y;
#pragma unroll
                        for (int i = 0; i < kWide; i++) y.v[i] = (T)o[t][i / 4][i % 4];
                        if (col + kWide <= value) {
                            *(Pack<T, kWide>*)(to + col) = y;
                        } else {
#pragma unroll
                            for (int i = 0; i < kWide; i++)
                                if (col + i < value) to[col + i] = y.v[i];
                        }
                    }
                }
            }
            if (end && !leave) break;
            const int less = end && m.forward && from + places == j.steps ? 1 : 0;
            if (weighted != 2 * n + less) {
                weighted = 2 * n + less;
#pragma unroll
                for (int t = 0; t < R; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int at = 16 * t + 4 * g + r;
                        keep[t][r] = at < n ? m.update * power(l2, n - at - less) : 0.0f;
                    }
            }
            any = true;
            /* What is kept of the state, and of the places from the last start on.  The state is
             * held as E / scale, so that no chunk has to go over it: its decay goes into scale and,
             * before that is under 1, into the state.  So what is held is never larger than E, nor
             * than k v what is added to it: nothing overflows that E does not. */
            const int last = starts ? 31 - __builtin_clz(starts) : -1;
            held += n - less;
            const float next = top * power(l2, held);
            if (starts) {
                dropped = true;
                scale = top = kHold;
                held = 0;
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) state[kb][vb] = F4{0, 0, 0, 0};
            } else if (next >= 1.0f) {
                scale = next;
            } else {
                const float f = next * (1.0f / kHold);
                scale = top = kHold;
                held = 0;
#pragma unroll
                for (int kb = 0; kb < KB; kb++)
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) state[kb][vb] *= f;
            }
            const float over = 1.0f / scale;
            F4 weight[R];
#pragma unroll
            for (int t = 0; t < R; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) weight[t][r] = 16 * t + 4 * g + r >= last ? keep[t][r] * over : 0.0f;
            if constexpr (kHalf) {
                /* weighted v as three numbers, since the state is one of 32 bits */
                auto split = [&](int vb, S4 h[R], S4 rest[R], S4 third[R]) {
#pragma unroll
                    for (int t = 0; t < R; t++) {
                        const F4 x = weight[t] * __builtin_convertvector(__builtin_bit_cast(B4, vq[t][vb]), F4);
                        h[t] = round4(x);
                        const F4 y = left4(x, h[t]);
                        rest[t] = round4(y);
                        third[t] = rest4(y, rest[t]);
                    }
                };
                /* either of k's and v's operands are held while the others pass, those of the fewer columns */
                if constexpr (KB <= VB) {
                    S4 kq[KB][R];
#pragma unroll
                    for (int kb = 0; kb < KB; kb++)
#pragma unroll
                        for (int t = 0; t < R; t++) kq[kb][t] = across<kKeyRow, 4>(lk, 16 * t, 16 * kb);
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) {
                        S4 h[R], rest[R], third[R];
                        split(vb, h, rest, third);
#pragma unroll
                        for (int kb = 0; kb < KB; kb++) state[kb][vb] = multiply(kq[kb][0], kq[kb][1], third[0], third[1], state[kb][vb]);
#pragma unroll
                        for (int kb = 0; kb < KB; kb++) state[kb][vb] = multiply(kq[kb][0], kq[kb][1], rest[0], rest[1], state[kb][vb]);
#pragma unroll
                        for (int kb = 0; kb < KB; kb++) state[kb][vb] = multiply(kq[kb][0], kq[kb][1], h[0], h[1], state[kb][vb]);
                    }
                } else {
                    S4 h[VB][R], rest[VB][R], third[VB][R];
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) split(vb, h[vb], rest[vb], third[vb]);
#pragma unroll
                    for (int kb = 0; kb < KB; kb++) {
                        const S4 k0 = across<kKeyRow, 4>(lk, 0, 16 * kb), k1 = across<kKeyRow, 4>(lk, 16, 16 * kb);
#pragma unroll
                        for (int vb = 0; vb < VB; vb++) state[kb][vb] = multiply(k0, k1, third[vb][0], third[vb][1], state[kb][vb]);
#pragma unroll
                        for (int vb = 0; vb < VB; vb++) state[kb][vb] = multiply(k0, k1, rest[vb][0], rest[vb][1], state[kb][vb]);
#pragma unroll
                        for (int vb = 0; vb < VB; vb++) state[kb][vb] = multiply(k0, k1, h[vb][0], h[vb][1], state[kb][vb]);
                    }
                }
            } else {
#pragma unroll
                for (int vb = 0; vb < VB; vb++) vq[0][vb] *= weight[0];
#pragma unroll
                for (int kb = 0; kb < KB; kb++) {
                    if (PART && 16 * kb >= m.key) break;
                    const F4 x = across<kKeyRow, 4>(lk, 0, 16 * kb);
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) {
                        if (PART && 16 * vb >= value) break;
                        state[kb][vb] = multiply(x, vq[0][vb], state[kb][vb]);
                    }
                }
            }
        }
        if (carry && lane == 0 && u.first == 0)
            *carry = dropped ? -1.0f : __builtin_amdgcn_exp2f(places ? (float)places * l2 : 0.0f);
        if (!leave || !active) return;
        const bool gone = !STATE && m.leave_starts && started(m.leave_starts + u.env * m.leave_starts_stride, j.starts_type);
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int vb = 0; vb < VB; vb++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int row = kb * 16 + 4 * g + r, col = value_col(vb) + kStep * (c / 4) + c % 4;
                    if (row < m.key && col < value)
                        leave[row * m.state_row + (u.first + col) * m.state_col] = gone ? 0.0f : scale * state[kb][vb][r];
                }
    }
};

/* Waves of a workgroup: the parts of a sequence where they share, else
 * neighbours in memory (roles of a sequence, heads).  Workgroups go to the 8
 * dies in turn: each die's take neighbouring ones. */
template <typename T, int KD, int VD, int W, bool STATE, bool PART>
__global__ __launch_bounds__(kThreads, 2) void la_walk(Job j) {
    extern __shared__ __attribute__((aligned(16))) char shared[];
    typedef Walk<T, KD, VD, W, STATE, PART> Walker;
    const unsigned die = blockIdx.x % 8, share = gridDim.x / 8, rest = gridDim.x % 8;
    const unsigned block = die * share + (die < rest ? die : rest) + blockIdx.x / 8;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    int64_t id = W > 1 ? (int64_t)block : (int64_t)block * (blockDim.x / kWave) + wave;
    const int64_t pieces = STATE ? j.pieces - 1 : j.pieces;
    if (W == 1 && id >= j.envs * j.heads * pieces * j.roles * j.parts) return;
    Unit u;
    u.first = (W > 1 ? wave : (int)(id % j.parts)) * VD;
    id /= W > 1 ? 1 : j.parts;
    u.role = (int)(id % j.roles);
    id /= j.roles;
    u.head = id % j.heads;
    id /= j.heads;
    u.env = id % j.envs;
    u.piece = id / j.envs;
    const Mix& m = j.mix[u.role];
    if (W == 1 && u.first >= m.value) return;
    if (!m.forward) u.piece = pieces - 1 - u.piece;
    const int64_t sequences = j.envs * j.heads, sequence = u.env * j.heads + u.head, size = (int64_t)m.key * m.value;
    const int64_t from = u.piece * j.places, left = j.steps - from, places = left < j.places ? left : j.places;
    const float* enter = m.enter ? m.enter + sequence * size : NULL;
    float* leave = m.leave ? m.leave + sequence * size : NULL;
    float* carry = NULL;
    if (STATE) {
        if (u.piece) enter = NULL;
        leave = m.pieces + (u.piece * sequences + sequence) * size;
        carry = m.carry + u.piece * sequences + sequence;
    } else {
        if (u.piece) enter = m.pieces + ((u.piece - 1) * sequences + sequence) * size;
        if (u.piece + 1 < pieces) leave = NULL;
    }
    Walker::run(j, m, u, from, places, enter, m.forward && u.piece == 0 && j.steps, leave, carry,
        shared + (W > 1 ? 0 : wave * Walker::kBytes));
}

/* What enters each piece, over what the pieces left by themselves; kAhead of
 * them are on their way at a time.  Of few sequences that is what it takes, else
 * memory: 31 pieces of 16 states of 128 x 128 12 us, 5.2 TB/s. */
__global__ __launch_bounds__(kThreads) void la_join(Job j) {
    constexpr int kAhead = 8;
    const Mix& m = j.mix[blockIdx.y];
    const int64_t sequences = j.envs * j.heads, size = (int64_t)m.key * m.value, all = sequences * size;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x, end = j.pieces - 1;
    if (i >= all) return;
    const float* carry = m.carry + i / size;
    float x = m.pieces[i];
    for (int64_t p = 1; p < end; p += kAhead) {
        float f[kAhead], own[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; a++) {
            if (p + a >= end) break;
            f[a] = carry[(p + a) * sequences];
            own[a] = m.pieces[(p + a) * all + i];
        }
#pragma unroll
        for (int a = 0; a < kAhead; a++) {
            if (p + a >= end) break;
            x = f[a] < 0 ? own[a] : f[a] * x + own[a];
            m.pieces[(p + a) * all + i] = x;
        }
    }
}

/* ---- one step ---- */

struct StepJob {
    B3Attention g;
    float scale;
    float* state;
    void* out;
};

/* A wave to a sequence: L lanes with four neighbouring columns each to a row
 * of the state, 64 / L rows at once.  The state, read and written, is all but
 * all that there is to move: 16,384 states of 64 x 64 102 us, 5.3 TB/s. */
template <typename T, int L>
__global__ __launch_bounds__(kThreads) void la_step(StepJob j) {
    constexpr int kRows = kWave / L, kAhead = 8;
    const B3Attention& g = j.g;
    const int64_t id = (int64_t)blockIdx.x * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (id >= g.envs * g.heads) return;
    const int64_t env = id / g.heads, head = id % g.heads;
    const int lane = threadIdx.x % kWave, col = lane % L * 4, row = lane / L, left = g.value - col;
    const float decay = decay_of(g.decay, head);
    const bool start = g.starts
        && started((const char*)g.starts + env * g.starts_stride[1] * (g.starts_type == B3_F32 ? 4 : 1), g.starts_type);
    float* s = j.state + id * g.key * g.value + col;
    const T* q = (const T*)g.q + env * g.q_stride[1] + head * g.q_stride[2];
    const T* k = (const T*)g.k + env * g.k_stride[1] + head * g.k_stride[2];
    const T* pv = (const T*)g.v + env * g.v_stride[1] + head * g.v_stride[2] + col;
    float v[4], o[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = i < left ? to_float(pv[i]) : 0.0f;
    for (int r0 = 0; r0 < g.key; r0 += kRows * kAhead) {
        Pack<float, 4> x[kAhead];
        float kr[kAhead], qr[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; a++) {
            const int r = r0 + a * kRows + row;
            const bool in = r < g.key;
            x[a] = Pack<float, 4>{0, 0, 0, 0};
            if (in && !start && left >= 4) {
                x[a] = *(const Pack<float, 4>*)(s + (int64_t)r * g.value);
            } else if (in && !start) {
                for (int i = 0; i < 3; i++)
                    if (i < left) x[a].v[i] = s[(int64_t)r * g.value + i];
            }
            kr[a] = in ? to_float(k[r]) : 0.0f;
            qr[a] = in ? to_float(q[r]) : 0.0f;
        }
#pragma unroll
        for (int a = 0; a < kAhead; a++) {
            const int r = r0 + a * kRows + row;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[a].v[i] = (start ? 0.0f : decay * x[a].v[i]) + kr[a] * v[i];
                if (r < g.key) o[i] += qr[a] * x[a].v[i];
            }
            if (r < g.key && left >= 4) {
                *(Pack<float, 4>*)(s + (int64_t)r * g.value) = x[a];
            } else if (r < g.key) {
                for (int i = 0; i < 3; i++)
                    if (i < left) s[(int64_t)r * g.value + i] = x[a].v[i];
            }
        }
    }
#pragma unroll
    for (int d = L; d < kWave; d *= 2)
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] += __shfl_xor(o[i], d);
    if (row) return;
    T* out = (T*)j.out + id * g.value + col;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < left) out[i] = (T)(j.scale * o[i]);
}

/* ---- launches ---- */

bool valid(const B3Attention* g) {
    if (!g || !is_float_type(g->type) || g->steps < 0 || g->envs < 0 || g->heads < 0 || g->key < 1 || g->key > B3_MAX_HEAD
            || g->value < 1 || g->value > B3_MAX_HEAD || !(g->scale == g->scale))
        return false;
    if (g->starts && g->starts_type != B3_F32 && g->starts_type != B3_U8) return false;
    if (g->envs == 0 || g->heads == 0) return true;
    if (g->envs > 0x7fffffff || g->heads > 0x7fffffff || g->steps > 0x7fffffff || g->envs * g->heads > B3_MAX_SEQUENCES) return false;
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
    m.forward = true;
    m.starts = (const char*)g.starts;
    m.starts_stride[0] = g.starts_stride[0] * size;
    m.starts_stride[1] = g.starts_stride[1] * size;
    m.enter = g.state;
    return m;
}

/* Before place p of the way back an episode starts where step steps - p's does. */
Mix backwards(const B3Attention& g, const float* d_last) {
    Mix m = forwards(g);
    m.reach = 1;
    m.update = (float)g.scale;
    m.forward = false;
    if (m.starts && g.steps) {
        m.leave_starts = m.starts;
        m.leave_starts_stride = m.starts_stride[1];
        m.starts += g.steps * m.starts_stride[0];
        m.starts_stride[0] = -m.starts_stride[0];
    }
    m.enter = d_last;
    return m;
}

int columns_of(int dims) { return dims <= 32 ? 32 : dims <= 64 ? 64 : 128; }
/* The state is at most 64 of a lane's registers, so that two waves fit a SIMD: two histories of 65,536 steps
 * and 8 heads of 128 are read in 491 us (and 1,230 back), 1,475 (4,310) with 128. */
int part_of(int key, int value) { return value <= 32 || key > 64 ? 32 : 64; }
int places_of(int type) { return type == B3_BF16 ? 32 : 16; }

/* How the work is cut: into parts of v's columns and, where that leaves
 * compute units idle, into pieces of the steps. */
struct Plan {
    int key, value, parts;                       // columns of tiles
    int64_t places, pieces;
};

/* Chunks' times that a launch's waves take for one each: 1.45 where two share a
 * SIMD, and of more waves something between what a last round takes by its
 * share and whole. */
double rounds(int64_t waves) {
    if (waves <= kAlone) return 1;
    if (waves <= kFull) return 1.45;
    return 1.45 * ((double)waves / kFull + (double)ceil_div(waves, kFull)) / 2;
}

/* What a pass takes in pieces, in us: a chunk 3.5 (1.8 of narrow heads), 0.6 of
 * it for a state alone; the two launches more 8, and 0.25 for a piece; the states, which are written,
 * added up and read, 4.5 MB a us.  Measured, us in 1, 2, 4, 8 and 16 pieces,
 * this took in brackets: bf16, heads of 64, 1,024 steps of 256 sequences 108,
 * 91, [62], 66, 91; 256 steps of them [29], 32, 33, 41, -; 4,096 of 64 sequences
 * 414, 320, 171, 97, [66], in 32 pieces 70; back, 12 pieces 139, 128 in 8, [119]
 * in 16; of 256 sequences of 1,024 steps [108], 119, 119, 141, 196.  It holds for
 * other types and heads as well: of 26 such rows of all types, with heads of
 * 32, 64 and 128, what it took was within 6 % of the best, but for bf16 heads of
 * 32 back (256 sequences of 1,024 steps [66], 69, 58, 64, 77).  fp32, heads of 64,
 * 1,024 steps of 256 sequences 243, 192, [120], 119, 143; fp16 249, 195, [119], 112,
 * 128; bf16, heads of 128, whose parts wait for each other, [113], 123, 164, 204,
 * 302, of 64 sequences of 4,096 413, 314, 182, [143], 164. */
double time_of(const B3Attention& g, const Plan& p, int64_t units, int64_t pieces, bool backward) {
    const double chunks = (double)ceil_div(ceil_div(g.steps, pieces), places_of(g.type)), chunk = p.key == 32 ? 1.8 : 3.5;
    const double walk = chunks * chunk * rounds(units * pieces);
    if (pieces == 1) return walk;
    const int ways = backward ? 2 : 1;
    const int64_t states = g.envs * g.heads * (pieces - 1) * ways;
    return walk + chunks * chunk * 0.6 * rounds(states * p.parts) + 8 + 0.25 * (double)pieces + (double)states * (double)(g.key * g.value) * 16 / 4.5e6;
}

Plan plan_of(const B3Attention& g, bool backward) {
    Plan p;
    const int most = g.key > g.value ? g.key : g.value;
    p.key = columns_of(backward ? most : g.key);
    p.value = part_of(backward ? most : g.key, backward ? most : g.value);
    p.parts = (int)ceil_div(backward ? most : g.value, p.value);
    const int64_t units = g.envs * g.heads * p.parts * (backward ? kRoles : 1);
    const int64_t chunk = places_of(g.type), chunks = ceil_div(g.steps, chunk);
    double least = 0;
    p.pieces = 1;
    auto look = [&](int64_t pieces) {
        const double time = time_of(g, p, units, pieces, backward);
        if (pieces > 1 && time >= least) return;
        p.pieces = pieces;
        least = time;
    };
    look(1);
    for (int64_t n = 2; n <= chunks && units * n <= 2 * kFull; n *= 2) look(n);
    for (int64_t waves : {kAlone, kFull})
        if (waves / units > 1 && waves / units <= chunks) look(waves / units);
    p.places = ceil_div(ceil_div(g.steps, p.pieces), chunk) * chunk;
    p.places = p.places > 0 ? p.places : chunk;
    p.pieces = g.steps > 0 ? ceil_div(g.steps, p.places) : 1;
    return p;
}

/* Floats of a way's pieces. */
int64_t pieces_size(const B3Attention& g, const Plan& p) {
    return (p.pieces - 1) * g.envs * g.heads * ((int64_t)g.key * g.value + 1);
}

size_t workspace_of(const B3Attention& g, const Plan& p, bool backward) {
    return (size_t)(pieces_size(g, p) * (backward ? 2 : 1)) * sizeof(float);
}

void place_pieces(Mix& m, const B3Attention& g, const Plan& p, void* workspace, int way) {
    m.pieces = (float*)workspace + way * pieces_size(g, p);
    m.carry = m.pieces + (p.pieces - 1) * g.envs * g.heads * g.key * g.value;
}

template <typename T, int KD, int VD, int W, bool STATE, bool PART>
hipError_t launch_walk(const Job& j, hipStream_t stream) {
    typedef Walk<T, KD, VD, W, STATE, PART> Walker;
    constexpr int kLds = 64 << 10, kMost = kLds / Walker::kBytes, kGroups = W > 1 ? 1 : kMost >= 4 ? 4 : 1;
    static_assert(kMost >= 1, "a workgroup's tiles");
    /* (workgroups of two would leave SIMDs empty: 32-bit heads of 128, two histories of 2,048 steps, take 88 us so, 72
     * one wave each; 1,000 environments of 512 steps 3,355 and 3,340) */
    const int64_t units = j.envs * j.heads * (STATE ? j.pieces - 1 : j.pieces) * j.roles * (W > 1 ? 1 : j.parts);
    la_walk<T, KD, VD, W, STATE, PART><<<(unsigned)ceil_div(units, kGroups), kGroups * W * kWave, kGroups * Walker::kBytes, stream>>>(j);
    return hipGetLastError();
}

template <typename T, int KD, int VD, int W, bool STATE>
hipError_t launch(const Job& j, hipStream_t stream) {
    for (int i = 0; i < j.roles; i++)
        if (j.mix[i].key < KD || j.mix[i].value % VD) return launch_walk<T, KD, VD, W, STATE, true>(j, stream);
    return launch_walk<T, KD, VD, W, STATE, false>(j, stream);
}

template <typename T, bool STATE>
hipError_t launch_columns(const Job& j, const Plan& p, hipStream_t stream) {
    if (p.key == 128) {
        /* In 16 bits parts share what they fetch: two histories of 65,536 steps and 8 heads of 128 take 491 us (1,230
         * back) so, 600 (1,550) each for itself.  In 32 the products take most of the time, and waves had better not
         * wait for each other: the backward pass of 333 steps of 57 x 3 with heads of 48 and 80 takes 98 us, 148 shared
         * (2,048 of two histories with 8 heads of 128, whose parts are all alike, 155 and 150). */
        if constexpr (__is_same(T, __bf16)) {
            if (p.parts > 2) return launch<T, 128, 32, 4, STATE>(j, stream);
            if (p.parts > 1) return launch<T, 128, 32, 2, STATE>(j, stream);
        }
        return launch<T, 128, 32, 1, STATE>(j, stream);
    }
    if (p.value == 32) return p.key == 32 ? launch<T, 32, 32, 1, STATE>(j, stream) : launch<T, 64, 32, 1, STATE>(j, stream);
    return p.key == 32 ? launch<T, 32, 64, 1, STATE>(j, stream) : launch<T, 64, 64, 1, STATE>(j, stream);
}

/* `ways`: what of the job's mixes learns the pieces' states, one for each. */
template <typename T>
hipError_t launch_typed(const Job& j, const Job& ways, const Plan& p, hipStream_t stream) {
    if (j.pieces > 1) {
        hipError_t err = launch_columns<T, true>(ways, p, stream);
        if (err != hipSuccess) return err;
        const int64_t all = j.envs * j.heads * j.mix[0].key * j.mix[0].value;
        if (j.pieces > 2) la_join<<<dim3((unsigned)ceil_div(all, kThreads), ways.roles), kThreads, 0, stream>>>(ways);
        if ((err = hipGetLastError()) != hipSuccess) return err;
    }
    return launch_columns<T, false>(j, p, stream);
}

hipError_t launch_job(Job& j, Job& ways, const Plan& p, int type, hipStream_t stream) {
    j.parts = ways.parts = p.parts;
    j.places = ways.places = p.places;
    j.pieces = ways.pieces = p.pieces;
    return type == B3_F32 ? launch_typed<float>(j, ways, p, stream)
        : type == B3_F16 ? launch_typed<_Float16>(j, ways, p, stream) : launch_typed<__bf16>(j, ways, p, stream);
}

template <typename T>
hipError_t launch_step(const StepJob& j, hipStream_t stream) {
    const unsigned blocks = (unsigned)ceil_div(j.g.envs * j.g.heads, kThreads / kWave);
    if (j.g.value <= 32) la_step<T, 8><<<blocks, kThreads, 0, stream>>>(j);
    else if (j.g.value <= 64) la_step<T, 16><<<blocks, kThreads, 0, stream>>>(j);
    else la_step<T, 32><<<blocks, kThreads, 0, stream>>>(j);
    return hipGetLastError();
}

}  // namespace
}  // namespace b3p

using namespace b3p;

extern "C" {

size_t b3_linear_attention_workspace(const B3Attention* g, int backward) {
    if (!valid(g) || g->envs == 0 || g->heads == 0) return 0;
    return workspace_of(*g, plan_of(*g, backward != 0), backward != 0);
}

hipError_t b3_linear_attention_gpu(const B3Attention* g, void* out, float* last_state, void* workspace,
        size_t workspace_bytes, hipStream_t stream) {
    if (!valid(g)) return hipErrorInvalidValue;
    if (g->envs == 0 || g->heads == 0 || (g->steps == 0 && !last_state)) return hipSuccess;
    const Plan p = plan_of(*g, false);
    if (!g->decay || (g->steps && !out) || !holds(workspace, workspace_bytes, workspace_of(*g, p, false))) return hipErrorInvalidValue;
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
    place_pieces(m, *g, p, workspace, 0);
    j.mix[0] = m;
    j.roles = 1;
    Job ways = j;
    return launch_job(j, ways, p, g->type, stream);
}

hipError_t b3_linear_attention_backward_gpu(const B3Attention* g, const void* d_out, const int64_t d_out_stride[3],
        const float* d_last_state, void* d_q, void* d_k, void* d_v, float* d_state, void* workspace,
        size_t workspace_bytes, hipStream_t stream) {
    if (!valid(g)) return hipErrorInvalidValue;
    if (g->envs == 0 || g->heads == 0 || (g->steps == 0 && !d_state)) return hipSuccess;
    const Plan p = plan_of(*g, true);
    if (!g->decay || (g->steps && (!d_out || !d_out_stride)) || !holds(workspace, workspace_bytes, workspace_of(*g, p, true)))
        return hipErrorInvalidValue;
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
    place_pieces(a, *g, p, workspace, 0);
    place_pieces(b, *g, p, workspace, 1);
    place_pieces(c, *g, p, workspace, 1);
    Job ways = j;
    if (d_q && g->steps) j.mix[j.roles++] = ways.mix[ways.roles++] = a;
    if (d_k && g->steps) j.mix[j.roles++] = b;
    if (d_v || d_state) j.mix[j.roles++] = c;
    if (!j.roles) return hipSuccess;
    if (!j.mix[j.roles - 1].forward) ways.mix[ways.roles++] = c;      // for d_k and d_v alike
    return launch_job(j, ways, p, g->type, stream);
}

hipError_t b3_linear_attention_step_gpu(const B3Attention* g, float* state, void* out, hipStream_t stream) {
    if (!valid(g) || g->steps != 1) return hipErrorInvalidValue;
    if (g->envs == 0 || g->heads == 0) return hipSuccess;
    if (!state || !out) return hipErrorInvalidValue;
    const StepJob j = {*g, (float)g->scale, state, out};
    return g->type == B3_F32 ? launch_step<float>(j, stream) : g->type == B3_F16 ? launch_step<_Float16>(j, stream)
                                                                                : launch_step<__bf16>(j, stream);
}

}  // extern "C"
