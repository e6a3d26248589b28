/*
 * b3_advantages.hip - generalised advantage estimates of a rollout
 * (include/b3_policy.h).
 *
 *   A_t = d_t + a_t A_{t+1},  d_t = r_t + gamma V_{t+1} - V_t,
 *   a_t = gamma lambda; a terminal at t drops the terms of t + 1.
 *
 * Each step maps the advantage after it to its own by x -> b + a x, and such
 * maps compose, so that time can be cut.  A thread holds the E steps of a
 * segment in registers and composes them; SEGS threads compose their
 * segments in LDS; then each goes over its steps again from the advantage
 * that enters its segment, and writes.  A workgroup's tile of SEGS E steps of
 * COLS environments moves from the end of the rollout to its start.  Where
 * environments alone would not give every compute unit a workgroup, the steps
 * are cut into pieces: a first launch composes each piece, and the second
 * folds the later pieces before it writes.  Everything is read once (twice
 * where cut: from the caches) and written once.
 */
#include "policy_common.h"

namespace b3p {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPieces = 512;
constexpr int64_t kFill = 256;                   // workgroups: one to a compute unit
constexpr int kWideCols = 64, kWideSteps = 16, kSteps = 8;

/* x -> b + a x.  a < 0 stands for a map that drops x altogether, as a
 * terminal does: 0 times a NaN would not.  A product of rates stays over 0,
 * since an infinity goes all the way back to the last terminal. */
struct Map {
    float a, b;
};

constexpr float kLeast = 1.17549435e-38f;

__device__ float apply(Map f, float x) { return f.a < 0 ? f.b : f.b + f.a * x; }

/* f after g: the earlier steps' f takes what the later ones' g gives. */
__device__ Map compose(Map f, Map g) {
    if (f.a < 0) return f;
    return Map{g.a < 0 ? -1.0f : fmaxf(f.a * g.a, kLeast), f.b + f.a * g.b};
}

struct Job {
    B3Rollout g;
    float gamma, decay;
    bool wide;                                   // steps are neighbours in every array
    bool once;                                   // past the caches, see stream_inputs
    int64_t tiles;                               // of a piece
    int64_t pieces;
    Map* piece;                                  // [pieces][envs]
};

/* Keeps the compiler from forming all steps' addresses ahead: they would take
 * more registers than the steps. */
template <typename T>
__device__ __forceinline__ void in_turn(T*& p) {
    asm("" : "+v"(p));
}

template <int SIZE, bool ONCE>
__device__ __forceinline__ uint32_t load_raw(const char* p) {
    if (SIZE == 4) return ONCE ? __builtin_nontemporal_load((const uint32_t*)p) : *(const uint32_t*)p;
    if (SIZE == 2) return ONCE ? __builtin_nontemporal_load((const uint16_t*)p) : *(const uint16_t*)p;
    return ONCE ? __builtin_nontemporal_load((const uint8_t*)p) : *(const uint8_t*)p;
}

/* E steps' elements of SIZE bytes as they lie: in words of their own, or,
 * where the steps are neighbours, packed.  Nothing is done with them here, so
 * that the loads of all arrays are in flight together.  Steps from `count`
 * (at least 1) on give the last one's. */
template <int E, int SIZE>
__device__ __forceinline__ void load_steps(const void* base, int64_t at, int64_t stride, int count, bool packed, bool once,
    uint32_t raw[E]) {
    const char* p = (const char*)base + at * SIZE;
    if (packed) {
        constexpr int kWords = E * SIZE / 4, kVec = kWords < 4 ? kWords : 4;
#pragma unroll
        for (int k = 0; k < kWords; k += kVec) {
            Bytes<uint32_t, kVec> b = *(const Bytes<uint32_t, kVec>*)(p + 4 * k);
#pragma unroll
            for (int w = 0; w < kVec; w++) raw[k + w] = b.v[w];
        }
        return;
    }
    const int64_t step = stride * SIZE;
    if (once) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            raw[e] = load_raw<SIZE, true>(p);
            p += e + 1 < count ? step : 0;
            in_turn(p);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) {
            raw[e] = load_raw<SIZE, false>(p);
            p += e + 1 < count ? step : 0;
            in_turn(p);
        }
    }
}

/* A value of TYPE as it lies. */
template <int TYPE>
__device__ __forceinline__ float float_of(uint32_t raw) {
    return TYPE == B3_F32 ? __uint_as_float(raw)
        : TYPE == B3_BF16 ? __uint_as_float(raw << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)raw);
}

template <int E, int TYPE>
__device__ __forceinline__ void floats_of(const uint32_t raw[E], bool packed, float x[E]) {
#pragma unroll
    for (int e = 0; e < E; e++)
        x[e] = float_of<TYPE>(TYPE != B3_F32 && packed ? raw[e / 2] >> (16 * (e % 2)) & 0xffffu : raw[e]);
}

/* Bit e: step e ends an episode. */
template <int E, int TYPE>
__device__ __forceinline__ uint32_t ends_of(const uint32_t raw[E], bool packed) {
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const uint32_t h = TYPE == B3_F32 ? raw[e] & 0x7fffffffu
            : packed ? raw[e / 4] >> (8 * (e % 4)) & 0xffu : raw[e];
        bits |= (h != 0) << e;
    }
    return bits;
}

template <int TYPE>
__device__ __forceinline__ float load_one(const void* p, int64_t at) {
    return float_of<TYPE>(TYPE == B3_F32 ? ((const uint32_t*)p)[at] : ((const uint16_t*)p)[at]);
}

/* BY_ENV: neighbouring threads have neighbouring environments, else
 * neighbouring segments.  SUM: compose the piece and write its map; else
 * write the advantages. */
template <int VALUES, int ENDS, bool BY_ENV, int COLS, int E, bool SUM>
__global__ __launch_bounds__(kThreads) void adv_tiles(Job job) {
    constexpr int SEGS = kThreads / COLS;
    __shared__ Map lds[2][kThreads];
    const B3Rollout& g = job.g;
    const int tid = threadIdx.x;
    const int col = BY_ENV ? tid % COLS : tid / SEGS, seg = BY_ENV ? tid / COLS : tid % SEGS;
    const int64_t blocks = (g.envs + COLS - 1) / COLS;
    /* workgroups go to the 8 dies in turn: each die's take neighbouring
     * blocks, whose rows share lines of its cache */
    const unsigned die = blockIdx.x % 8, share = gridDim.x / 8, rest = gridDim.x % 8;
    const unsigned block = die * share + (die < rest ? die : rest) + blockIdx.x / 8;
    const int64_t env = (int64_t)(block % blocks) * COLS + col, piece = block / blocks;
    const bool live = env < g.envs;
    const int64_t all_tiles = (g.steps + SEGS * E - 1) / (SEGS * E);
    const int64_t first = piece * job.tiles;
    int64_t tile = first + job.tiles < all_tiles ? first + job.tiles : all_tiles;

    /* lds[.][segment of a column]: the maps of its segments from `seg` on,
     * composed; the result is in lds[at] */
    auto compose_later = [&](Map mine, int& at) {
        lds[0][seg * COLS + col] = mine;
        at = 0;
        __syncthreads();
#pragma unroll
        for (int d = 1; d < SEGS; d *= 2) {
            if (seg + d < SEGS) mine = compose(mine, lds[at][(seg + d) * COLS + col]);
            at ^= 1;
            lds[at][seg * COLS + col] = mine;
            __syncthreads();
        }
    };

    /* the advantage after the piece, from the maps of the later ones */
    float carry = 0;
    if (!SUM && job.pieces > 1) {
        const int64_t later = job.pieces - piece - 1, each = (later + SEGS - 1) / SEGS;
        Map f = {1, 0};
        for (int64_t k = each - 1; k >= 0; k--) {
            const int64_t p = piece + 1 + seg * each + k;
            if (live && p < job.pieces) f = compose(job.piece[p * g.envs + env], f);
        }
        int at;
        compose_later(f, at);
        carry = apply(lds[at][col], 0);
        __syncthreads();
    }
    Map total = {1, 0};                          // of the piece's tiles so far

#pragma unroll 1
    while (--tile >= first) {
        const int64_t t = (tile * SEGS + seg) * E;
        const int64_t left = live ? g.steps - t : 0;
        const int count = left < 0 ? 0 : left < E ? (int)left : E;
        float r[E], v[E], after = 0;
        uint32_t ends = 0;
        if (count) {
            const bool packed = job.wide && count == E;
            uint32_t raw_r[E], raw_v[E], raw_end[E];
            load_steps<E, 4>(g.rewards, env * g.rewards_stride[1] + t * g.rewards_stride[0], g.rewards_stride[0], count,
                packed, BY_ENV && job.once, raw_r);
            load_steps<E, ENDS == B3_F32 ? 4 : 1>(g.terminals, env * g.terminals_stride[1] + t * g.terminals_stride[0],
                g.terminals_stride[0], count, packed, BY_ENV && job.once, raw_end);
            load_steps<E, VALUES == B3_F32 ? 4 : 2>(g.values, env * g.values_stride[1] + t * g.values_stride[0],
                g.values_stride[0], count, packed, BY_ENV && job.once, raw_v);
            after = t + count < g.steps
                ? load_one<VALUES>(g.values, env * g.values_stride[1] + (t + count) * g.values_stride[0])
                : load_one<VALUES>(g.last_values, env * g.last_values_stride);
            floats_of<E, B3_F32>(raw_r, packed, r);
            floats_of<E, VALUES>(raw_v, packed, v);
            ends = ends_of<E, ENDS>(raw_end, packed);
        }
        /* r becomes d; the map of the segment */
        Map f = {1, 0};
#pragma unroll
        for (int e = E - 1; e >= 0; e--) {
            if (e < count) {
                const bool end = ends >> e & 1;
                r[e] = end ? r[e] - v[e] : r[e] + job.gamma * after - v[e];
                after = v[e];
                f.b = end ? r[e] : r[e] + job.decay * f.b;
                f.a = end ? -1.0f : f.a < 0 ? f.a : fmaxf(f.a * job.decay, kLeast);
            }
        }
        int at;
        compose_later(f, at);
        const Map whole = lds[at][col];
        if (SUM) {
            total = compose(whole, total);
        } else {
            float x = seg + 1 < SEGS ? apply(lds[at][(seg + 1) * COLS + col], carry) : carry;
            carry = apply(whole, carry);
#pragma unroll
            for (int e = E - 1; e >= 0; e--) {
                if (e < count) {
                    x = ends >> e & 1 ? r[e] : r[e] + job.decay * x;
                    r[e] = x;
                    v[e] += x;
                }
            }
            const int64_t o = env * g.out_stride[1] + t * g.out_stride[0];
            if (job.wide && count >= E) {
#pragma unroll
                for (int k = 0; k < E / 4; k++) {
                    *(Pack<float, 4>*)(g.advantages + o + 4 * k) = Pack<float, 4>{r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]};
                    *(Pack<float, 4>*)(g.returns + o + 4 * k) = Pack<float, 4>{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]};
                }
            } else {
                float* adv = g.advantages + o;
                float* ret = g.returns + o;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    if (e < count) {
                        *adv = r[e];
                        *ret = v[e];
                    }
                    adv += g.out_stride[0];
                    ret += g.out_stride[0];
                    in_turn(adv);
                    in_turn(ret);
                }
            }
        }
        __syncthreads();
    }
    if (SUM && seg == 0 && live) job.piece[piece * g.envs + env] = total;
}

/* How a rollout is cut: lanes along environments or along steps, environments
 * to a workgroup, pieces of the steps. */
struct Plan {
    bool by_env;
    int cols, steps;                             // steps: E
    int64_t blocks, tiles, pieces;
};

Plan plan_of(int64_t steps, int64_t envs, bool by_env) {
    Plan p;
    p.by_env = by_env;
    if (by_env) {
        p.cols = envs >= kWideCols * kFill ? kWideCols : 16;
        p.steps = p.cols == 16 ? kSteps : kWideSteps;
    } else {
        p.cols = steps <= 64 ? 64 : steps <= 512 ? 16 : 1;
        /* where tiles of 4,096 steps are few, of 1,024 */
        p.steps = p.cols == 1 && envs * ceil_div(steps, kThreads * 16) < 2 * kFill ? 4 : 16;
    }
    const int64_t tile = (int64_t)(kThreads / p.cols) * p.steps, all = ceil_div(steps, tile);
    p.blocks = ceil_div(envs, p.cols);
    p.pieces = 1;
    if (p.blocks < kFill) {
        p.pieces = ceil_div(kFill * 2, p.blocks);
        p.pieces = p.pieces < all ? p.pieces : all;
        p.pieces = p.pieces < kMaxPieces ? p.pieces : kMaxPieces;
    }
    p.tiles = ceil_div(all, p.pieces);
    p.pieces = ceil_div(all, p.tiles);
    return p;
}

/* Lanes along the axis of neighbours; fewer environments than a workgroup
 * takes side by side leave its lanes to the steps. */
bool by_env(const B3Rollout& g) { return g.envs >= 16 && g.out_stride[1] <= g.out_stride[0]; }

template <int VALUES, int ENDS, bool BY_ENV, int COLS, int E>
hipError_t launch(const Job& job, const Plan& p, hipStream_t stream) {
    const unsigned grid = (unsigned)(p.blocks * p.pieces);
    if (p.pieces > 1) {
        adv_tiles<VALUES, ENDS, BY_ENV, COLS, E, true><<<grid, kThreads, 0, stream>>>(job);
        hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    adv_tiles<VALUES, ENDS, BY_ENV, COLS, E, false><<<grid, kThreads, 0, stream>>>(job);
    return hipGetLastError();
}

template <int VALUES, int ENDS>
hipError_t launch_plan(const Job& job, const Plan& p, hipStream_t stream) {
    if (p.by_env)
        return p.cols == kWideCols ? launch<VALUES, ENDS, true, kWideCols, kWideSteps>(job, p, stream)
                                   : launch<VALUES, ENDS, true, 16, kSteps>(job, p, stream);
    return p.cols == 64 ? launch<VALUES, ENDS, false, 64, 16>(job, p, stream)
        : p.cols == 16 ? launch<VALUES, ENDS, false, 16, 16>(job, p, stream)
        : p.steps == 16 ? launch<VALUES, ENDS, false, 1, 16>(job, p, stream) : launch<VALUES, ENDS, false, 1, 4>(job, p, stream);
}

template <int VALUES>
hipError_t launch_values(const Job& job, const Plan& p, hipStream_t stream) {
    return job.g.terminals_type == B3_F32 ? launch_plan<VALUES, B3_F32>(job, p, stream)
                                          : launch_plan<VALUES, B3_U8>(job, p, stream);
}

bool valid(const B3Rollout& g) {
    if (g.steps < 0 || g.envs < 0 || !is_float_type(g.values_type)) return false;
    if (g.terminals_type != B3_F32 && g.terminals_type != B3_U8) return false;
    if (g.steps == 0 || g.envs == 0) return true;
    return g.envs <= 0x7fffffff && g.steps <= 0x7fffffff && g.rewards && g.values && g.last_values && g.terminals
        && g.advantages && g.returns;
}

/* Whether every step's elements of a workgroup's environments are whole lines
 * of 128 bytes. */
bool whole_lines(const void* p, const int64_t stride[2], int64_t size, int cols) {
    return (uintptr_t)p % 128 == 0 && stride[1] == 1 && stride[0] * size % 128 == 0 && cols * size % 128 == 0;
}

/* Inputs that the caches would not keep go past them where no line is read by
 * two workgroups: 500 steps of 65,536 environments with bf16 values take 106 us
 * so, and 125 through the caches; 128 steps of 32,768 in fp32, which the caches
 * keep, 25 and 24.  Where lines are shared it goes either way: 500 of 65,537
 * take 131 us past them and 145 through, 128 of 300,007 178 and 162, 2,000 of
 * 16,387 210 and 179. */
bool stream_inputs(const B3Rollout& g, const Plan& p) {
    const int64_t value = g.values_type == B3_F32 ? 4 : 2, end = g.terminals_type == B3_F32 ? 4 : 1;
    return p.by_env && p.pieces == 1 && g.steps * g.envs > ((int64_t)1 << 27) / (4 + value + end)
        && whole_lines(g.rewards, g.rewards_stride, 4, p.cols) && whole_lines(g.values, g.values_stride, value, p.cols)
        && whole_lines(g.terminals, g.terminals_stride, end, p.cols);
}

size_t workspace_of(const Plan& p, int64_t envs) {
    return p.pieces > 1 ? (size_t)p.pieces * envs * sizeof(Map) : 0;
}

/* Environments from `first` on. */
B3Rollout some_envs(B3Rollout g, int64_t first, int64_t envs) {
    const int64_t value = g.values_type == B3_F32 ? 4 : 2, end = g.terminals_type == B3_F32 ? 4 : 1;
    g.envs = envs;
    g.rewards += first * g.rewards_stride[1];
    g.values = (const char*)g.values + first * g.values_stride[1] * value;
    g.last_values = (const char*)g.last_values + first * g.last_values_stride * value;
    g.terminals = (const char*)g.terminals + first * g.terminals_stride[1] * end;
    g.advantages += first * g.out_stride[1];
    g.returns += first * g.out_stride[1];
    return g;
}

}  // namespace
}  // namespace b3p

using namespace b3p;

extern "C" {

/* For either layout. */
size_t b3_advantages_workspace(int64_t steps, int64_t envs) {
    if (steps <= 0 || envs <= 0) return 0;
    const size_t a = workspace_of(plan_of(steps, envs, true), envs), b = workspace_of(plan_of(steps, envs, false), envs);
    return a > b ? a : b;
}

hipError_t b3_advantages_gpu(const B3Rollout* g, double gamma, double lambda, void* workspace, size_t workspace_bytes,
        hipStream_t stream) {
    if (!g || !valid(*g) || !(gamma >= 0 && gamma <= 1) || !(lambda >= 0 && lambda <= 1)) return hipErrorInvalidValue;
    if (g->steps == 0 || g->envs == 0) return hipSuccess;
    const Plan p = plan_of(g->steps, g->envs, by_env(*g));
    const size_t need = workspace_of(p, g->envs);
    if (!holds(workspace, workspace_bytes, need)) return hipErrorInvalidValue;
    const bool wide = g->rewards_stride[0] == 1 && g->values_stride[0] == 1 && g->terminals_stride[0] == 1
        && g->out_stride[0] == 1;
    Job job = {*g, (float)gamma, (float)(gamma * lambda), wide, stream_inputs(*g, p), p.tiles, p.pieces, (Map*)workspace};
    /* cut steps have few blocks: more than a launch's are of whole rollouts */
    const int64_t most = kMostBlocks * p.cols;
    hipError_t err = hipSuccess;
    for (int64_t e = 0; e < g->envs && err == hipSuccess; e += most) {
        Plan part = p;
        job.g = some_envs(*g, e, g->envs - e < most ? g->envs - e : most);
        part.blocks = ceil_div(job.g.envs, p.cols);
        err = g->values_type == B3_F32 ? launch_values<B3_F32>(job, part, stream)
            : g->values_type == B3_F16 ? launch_values<B3_F16>(job, part, stream) : launch_values<B3_BF16>(job, part, stream);
    }
    return err;
}

}  // extern "C"
