/*
 * b3_log_probs.hip - log probabilities, entropies and best alternatives of
 * rows of logits, and their gradient (include/b3_policy.h).
 *
 * With m = max x, z = x - m and S = sum exp(z):
 *   log p_j = z_j - log S          H = log S - (sum z exp(z)) / S
 *   dx_j = dlp ([j = taken] - p_j) - dH p_j (log p_j + H)
 *
 * Both directions are bound by memory: the forward reads the logits once,
 * the backward reads them once and writes as much.  A row, or a piece of one,
 * is held in the registers of the threads that share it, so that the maximum
 * comes before the sums with one read and no rescaling:
 *   up to 2,048 actions   G lanes of a wave to a row, by a rule on the
 *                         actions alone (with_small)
 *   more                  a workgroup to a row, or to a piece of one
 *                         (pieces_of); the pieces' (m, S, sum z exp(z)) and
 *                         best alternatives are joined by a wave per row
 * A lane loads W neighbouring logits at once; lanes take turns, so the order
 * of places is (load, lane, place in the load).
 */
#include "policy_common.h"

namespace b3p {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxActions = 1 << 21;
constexpr int kMaxPieces = 256;
constexpr float kLog2e = 1.44269504f;
constexpr float kLn2 = 0.693147181f;

/* A logit, -inf where its action is not allowed. */
template <typename T>
__device__ float logit(const T* row, const unsigned char* mask, int64_t j) {
    return mask && !mask[j] ? -INFINITY : to_float(row[j]);
}

template <typename T>
__device__ const T* row_of(const B3Logits& g, int64_t r) {
    return (const T*)g.data + r * g.row_stride;
}

__device__ const unsigned char* mask_of(const B3Logits& g, int64_t r) {
    return g.mask ? g.mask + r * g.mask_row_stride : NULL;
}

/* The logits of a thread: places from + (v G + lane) W + w below `n`; -inf in
 * the others.  All loads are issued before the first is used: whole vectors
 * first, then the elements of the one vector that passes n.  `once`: past the
 * caches (see stream_logits). */
template <typename T, int G, int PER, int W>
__device__ __forceinline__ void load_logits(const T* row, const unsigned char* mask, int from, int n, int lane, bool once,
    float x[PER]) {
    constexpr int NV = PER / W;
    Pack<T, W> p[NV];
    Pack<unsigned char, W> k[NV];
    if (n - from >= G * PER) {
        if (once) {
#pragma unroll
            for (int v = 0; v < NV; v++) p[v] = Stream<T, W>::load(row + from + (v * G + lane) * W);
        } else {
#pragma unroll
            for (int v = 0; v < NV; v++) p[v] = *(const Pack<T, W>*)(row + from + (v * G + lane) * W);
        }
        if (mask) {
#pragma unroll
            for (int v = 0; v < NV; v++) k[v] = *(const Pack<unsigned char, W>*)(mask + from + (v * G + lane) * W);
        }
#pragma unroll
        for (int i = 0; i < PER; i++) x[i] = to_float(p[i / W].v[i % W]);
        if (mask) {
#pragma unroll
            for (int i = 0; i < PER; i++) x[i] = k[i / W].v[i % W] ? x[i] : -INFINITY;
        }
        return;
    }
    const int last = (n - from) / (G * W);       // the load in which some lane passes n
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int j = from + (v * G + lane) * W;
        if (v < last || (v == last && j + W <= n)) {
            p[v] = *(const Pack<T, W>*)(row + j);
            if (mask) k[v] = *(const Pack<unsigned char, W>*)(mask + j);
        }
    }
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int j = from + (v * G + lane) * W;
        if (v < last) {
#pragma unroll
            for (int w = 0; w < W; w++) x[v * W + w] = to_float(p[v].v[w]);
            if (mask) {
#pragma unroll
                for (int w = 0; w < W; w++) x[v * W + w] = k[v].v[w] ? x[v * W + w] : -INFINITY;
            }
            continue;
        }
#pragma unroll
        for (int w = 0; w < W; w++) x[v * W + w] = -INFINITY;
        if (v > last) continue;
        if (j + W <= n) {
#pragma unroll
            for (int w = 0; w < W; w++) {
                x[v * W + w] = to_float(p[v].v[w]);
                if (mask) x[v * W + w] = k[v].v[w] ? x[v * W + w] : -INFINITY;
            }
        } else {
#pragma unroll
            for (int w = 0; w < W; w++)
                if (j + w < n) x[v * W + w] = logit(row, mask, j + w);
        }
    }
}

/* One instruction for two elements; of a NaN and a number the number. */
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

/* ---- reductions ---- */

template <int CONTROL, int ROWS>
__device__ __forceinline__ float from_lane(float x, float old) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(old), __float_as_uint(x), CONTROL, ROWS, 0xf, false));
}

__device__ __forceinline__ float last_lane(float x) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), kWave - 1));
}

/* Over a wave, the result in a scalar register: within rows of 16 lanes by
 * shifts of 1, 2, 4 and 8, then from each row's last lane to the rows after
 * it.  A lane that would read from outside takes the neutral value. */
__device__ __forceinline__ float wave_sum(float x) {
    x += from_lane<0x111, 0xf>(x, 0.0f);
    x += from_lane<0x112, 0xf>(x, 0.0f);
    x += from_lane<0x114, 0xf>(x, 0.0f);
    x += from_lane<0x118, 0xf>(x, 0.0f);
    x += from_lane<0x142, 0xa>(x, 0.0f);
    x += from_lane<0x143, 0xc>(x, 0.0f);
    return last_lane(x);
}

__device__ __forceinline__ float wave_max(float x) {
    x = max3(x, x, from_lane<0x111, 0xf>(x, x));
    x = max3(x, x, from_lane<0x112, 0xf>(x, x));
    x = max3(x, x, from_lane<0x114, 0xf>(x, x));
    x = max3(x, x, from_lane<0x118, 0xf>(x, x));
    x = max3(x, x, from_lane<0x142, 0xf>(x, x));
    x = max3(x, x, from_lane<0x143, 0xf>(x, x));
    return last_lane(x);
}

/* Over the G < 64 lanes that share a row. */
template <int G, typename F>
__device__ __forceinline__ float group_reduce(float x, F f) {
#pragma unroll
    for (int d = 1; d < G; d *= 2) x = f(x, __shfl_xor(x, d));
    return x;
}

/* m, S and D = sum z exp(z) of a row or a part of it.  m is 0 where nothing
 * is allowed, and where all that is allowed is NaN (S is then NaN). */
struct Sums {
    float m, s, d;
};

/* Loads of W in a thread's PER that have any place below n. */
template <int G, int PER, int W>
__device__ __forceinline__ int live_loads(int from, int n) {
    const int loads = (n - from + G * W - 1) / (G * W);
    return loads < PER / W ? loads : PER / W;
}

template <int PER, int W>
__device__ __forceinline__ float lane_max(const float x[PER], int live) {
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < PER / W; v++) {
        if (v < live) {
#pragma unroll
            for (int i = v * W; i < (v + 1) * W; i += 2) m = max3(m, x[i], x[i + 1]);
        }
    }
    return m;
}

/* The sums over G <= 64 lanes of a row, of its first `live` loads, from each
 * lane's maximum.  exp(z) is
 * 2^t with t = x log2 e - fl(m log2 e) in one rounding, which is z log2 e
 * but for `off`, what fl() left out; it is the same for every term and taken
 * back from the sums.  Beyond 2^16 it could be large, and t is formed from z.
 * A term is off by |t| 2^-24, relative to itself; those with |t| > 30 do not
 * count.  t is bounded in D alone, where 0 times -inf would be NaN. */
template <int G, int PER, int W>
__device__ __forceinline__ Sums sums_of(const float x[PER], int live, float lane_most) {
    float m = G == kWave ? wave_max(lane_most)
        : group_reduce<G>(lane_most, [](float a, float b) { return max3(a, b, b); });
    m = m == -INFINITY || m != m ? 0.0f : m;
    float s = 0, d = 0, off = 0;
    const bool small = fabsf(m) <= 65536.0f;
    const float ml = m * kLog2e;
    if (small) off = __builtin_fmaf(m, kLog2e, -ml);
#pragma unroll
    for (int v = 0; v < PER / W; v++) {
        if (v < live && small) {
#pragma unroll
            for (int i = v * W; i < (v + 1) * W; i++) {
                const float t = __builtin_fmaf(x[i], kLog2e, -ml), e = __builtin_amdgcn_exp2f(t);
                s += e;
                d = __builtin_fmaf(e, fmaxf(t, -1e4f), d);
            }
        } else if (v < live) {
#pragma unroll
            for (int i = v * W; i < (v + 1) * W; i++) {
                const float t = (x[i] - m) * kLog2e, e = __builtin_amdgcn_exp2f(t);
                s += e;
                d = __builtin_fmaf(e, fmaxf(t, -1e4f), d);
            }
        }
    }
    if (G == kWave) {
        s = wave_sum(s);
        d = wave_sum(d);
    } else {
        auto add = [](float a, float b) { return a + b; };
        s = group_reduce<G>(s, add);
        d = group_reduce<G>(d, add);
    }
    const float back = __builtin_amdgcn_exp2f(-off);
    return Sums{m, s * back, __builtin_fmaf(-off, s, d) * (back * kLn2)};
}

/* Two parts of a row as one.  A part that allows nothing has no say in m. */
__device__ __forceinline__ Sums join(Sums a, Sums b) {
    const float m = a.s == 0.0f ? b.m : b.s == 0.0f ? a.m : fmaxf(a.m, b.m);
    const float za = a.m - m, zb = b.m - m;
    const float ea = __builtin_amdgcn_exp2f(za * kLog2e), eb = __builtin_amdgcn_exp2f(zb * kLog2e);
    Sums r = {m, 0.0f, 0.0f};
    if (a.s != 0.0f) {
        r.s += ea * a.s;
        r.d += ea * (a.d + fmaxf(za, -1e4f) * a.s);
    }
    if (b.s != 0.0f) {
        r.s += eb * b.s;
        r.d += eb * (b.d + fmaxf(zb, -1e4f) * b.s);
    }
    return r;
}

struct Outputs {
    const int64_t* taken;
    float* log_prob;
    float* entropy;
    float* stats;
    int top;
    float* top_log_prob;
    int64_t* top_action;
};

/* The taken action's logit, fetched before the sums are formed. */
template <typename T>
__device__ __forceinline__ float taken_logit(const B3Logits& g, int64_t r, int64_t a) {
    return a >= 0 && a < g.actions ? logit(row_of<T>(g, r), mask_of(g, r), a) : 0.0f;
}

/* What one thread of a row writes; x is the logit of the taken action a. */
__device__ __forceinline__ void finish_row(const B3Logits& g, const Outputs& o, int64_t r, int64_t a, float x, Sums s,
    float log_sum) {
    const bool empty = s.s == 0.0f;
    float lp = 0.0f;
    if (a >= g.actions)
        lp = NAN;
    else if (a >= 0)
        lp = empty ? -INFINITY : x - s.m - log_sum;
    o.log_prob[r] = lp;
    o.entropy[r] = empty ? 0.0f : log_sum - s.d / s.s;
    if (o.stats) {
        o.stats[2 * r] = s.m;
        o.stats[2 * r + 1] = log_sum;
    }
}

/* ---- best alternatives ---- */

/* Whole numbers in the order of the logits: NaN above +inf, -0 as 0; never 0,
 * which stands for one that has been taken out. */
__device__ uint32_t order_of(float x) {
    if (x != x) return 0xfffffffeu;
    uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ float value_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}

__device__ void write_top(const Outputs& o, int64_t r, int k, uint32_t order, int64_t action, Sums s, float log_sum) {
    o.top_log_prob[r * o.top + k] = s.s == 0.0f ? -INFINITY : value_of(order) - s.m - log_sum;
    o.top_action[r * o.top + k] = action;
}

/* The wave's largest, in a scalar register: rows of 16 lanes by shifts, then
 * each row's last lane to the next row.  Lanes that would read from outside
 * keep what they have. */
__device__ __forceinline__ uint32_t wave_most(uint32_t x) {
    uint32_t y;
    y = __builtin_amdgcn_update_dpp(x, x, 0x111, 0xf, 0xf, false);
    x = x > y ? x : y;
    y = __builtin_amdgcn_update_dpp(x, x, 0x112, 0xf, 0xf, false);
    x = x > y ? x : y;
    y = __builtin_amdgcn_update_dpp(x, x, 0x114, 0xf, 0xf, false);
    x = x > y ? x : y;
    y = __builtin_amdgcn_update_dpp(x, x, 0x118, 0xf, 0xf, false);
    x = x > y ? x : y;
    y = __builtin_amdgcn_update_dpp(x, x, 0x142, 0xf, 0xf, false);
    x = x > y ? x : y;
    y = __builtin_amdgcn_update_dpp(x, x, 0x143, 0xf, 0xf, false);
    x = x > y ? x : y;
    return __builtin_amdgcn_readlane(x, kWave - 1);
}

/* Over the lanes up to and with this one. */
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}

/* The `top` largest of the wave's NV loads of W orders, one after the other:
 * lane k gets the k-th's order and place (load, lane, place in the load).
 * Among equals the lowest place is taken: the first load that any lane has it
 * in, the first such lane, its first place.  Every round takes one of at
 * least `top` orders that are not 0, or finds 0 and gives it. */
template <int NV, int W>
__device__ void wave_top(uint32_t order[NV * W], int top, uint32_t& my_order, int& my_load, int& my_lane, int& my_place) {
    const int lane = threadIdx.x % kWave;
    uint32_t best[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) {
        best[v] = order[v * W];
#pragma unroll
        for (int w = 1; w < W; w++) best[v] = best[v] > order[v * W + w] ? best[v] : order[v * W + w];
    }
    my_order = 0;
    my_load = my_lane = my_place = 0;
    for (int k = 0; k < top; k++) {
        uint32_t most = best[0];
#pragma unroll
        for (int v = 1; v < NV; v++) most = most > best[v] ? most : best[v];
        most = wave_most(most);
        bool found = false;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const uint64_t have = __ballot(best[v] == most);
            if (!found && have) {
                found = true;
                const int who = __builtin_ctzll(have);
                int place = W - 1;
#pragma unroll
                for (int w = W - 2; w >= 0; w--) place = order[v * W + w] == most ? w : place;
                place = __builtin_amdgcn_readlane(place, who);
                uint32_t b = 0;
#pragma unroll
                for (int w = 0; w < W; w++) {
                    if (w == place && lane == who) order[v * W + w] = 0;
                    b = b > order[v * W + w] ? b : order[v * W + w];
                }
                best[v] = b;
                if (lane == k) {
                    my_order = most;
                    my_load = v;
                    my_lane = who;
                    my_place = place;
                }
            }
        }
    }
}

/* The largest (or, of the complements, the smallest) over the G = 1, 4 or 16
 * lanes of a row, to all of them: lanes swapped in pairs, pairs swapped,
 * eights and sixteens mirrored. */
template <int G>
__device__ __forceinline__ uint32_t group_most(uint32_t x) {
    uint32_t y;
    if (G >= 4) {
        y = __builtin_amdgcn_update_dpp(x, x, 0xb1, 0xf, 0xf, false);
        x = x > y ? x : y;
        y = __builtin_amdgcn_update_dpp(x, x, 0x4e, 0xf, 0xf, false);
        x = x > y ? x : y;
    }
    if (G >= 16) {
        y = __builtin_amdgcn_update_dpp(x, x, 0x141, 0xf, 0xf, false);
        x = x > y ? x : y;
        y = __builtin_amdgcn_update_dpp(x, x, 0x140, 0xf, 0xf, false);
        x = x > y ? x : y;
    }
    return x;
}

/* The same for G < 64 lanes to a row: each round the largest order, its lowest
 * place, and that one taken out. */
template <int G, int PER, int W>
__device__ void group_top(const float x[PER], int n, const Outputs& o, int64_t r, Sums s, float log_sum) {
    static_assert(G == 1 || G == 4 || G == 16, "group_most");
    const int lane = threadIdx.x % G;
    uint32_t order[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) order[i] = ((i / W) * G + lane) * W + i % W < n ? order_of(x[i]) : 0;
    for (int k = 0; k < o.top; k++) {
        uint32_t most = order[0];
#pragma unroll
        for (int i = 1; i < PER; i++) most = most > order[i] ? most : order[i];
        most = group_most<G>(most);
        uint32_t not_place = 0;                  // the complement of the place: the lowest is the largest
#pragma unroll
        for (int i = PER - 1; i >= 0; i--) not_place = order[i] == most ? ~(uint32_t)(((i / W) * G + lane) * W + i % W) : not_place;
        not_place = group_most<G>(not_place);
#pragma unroll
        for (int i = 0; i < PER; i++) order[i] = ~(uint32_t)(((i / W) * G + lane) * W + i % W) == not_place ? 0 : order[i];
        if (lane == 0) write_top(o, r, k, most, ~not_place, s, log_sum);
    }
}

/* ---- forward ---- */

/* G lanes to a row: up to G PER actions. */
template <typename T, int G, int PER, int W>
__global__ __launch_bounds__(kThreads, 8) void lp_small(B3Logits g, Outputs o) {
    const int64_t r = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / G;
    if (r >= g.rows) return;                     // all G lanes of it
    const int lane = threadIdx.x % G, n = (int)g.actions;
    const int64_t a = o.taken[r];
    float x[PER];
    load_logits<T, G, PER, W>(row_of<T>(g, r), mask_of(g, r), 0, n, lane, false, x);
    const float xa = taken_logit<T>(g, r, a);
    const int live = live_loads<G, PER, W>(0, n);
    const Sums s = sums_of<G, PER, W>(x, live, lane_max<PER, W>(x, live));
    const float log_sum = logf(s.s);
    if (lane == 0) finish_row(g, o, r, a, xa, s, log_sum);
    if (!o.top) return;
    if constexpr (G == kWave) {
        uint32_t order[PER], my_order;
        int v, l, w;
#pragma unroll
        for (int i = 0; i < PER; i++) order[i] = ((i / W) * G + lane) * W + i % W < n ? order_of(x[i]) : 0;
        wave_top<PER / W, W>(order, o.top, my_order, v, l, w);
        if (lane < o.top) write_top(o, r, lane, my_order, (v * G + l) * W + w, s, log_sum);
    } else {
        group_top<G, PER, W>(x, n, o, r, s, log_sum);
    }
}

/* A piece's sums and alternatives, in the caller's workspace. */
struct Pieces {
    int count, size;                             // pieces of a row, actions of a piece
    bool once;
    Sums* sums;                                  // [rows][count]
    uint2* top;                                  // [rows][count][top]: order, action
};

/* The lane's first place of a value, or none. */
template <int THREADS, int PER, int W>
__device__ int first_place(const float x[PER], float value, int from, int n) {
    int place = INT32_MAX;
#pragma unroll
    for (int i = PER - 1; i >= 0; i--) {
        const int j = from + ((i / W) * THREADS + (int)threadIdx.x) * W + i % W;
        place = x[i] == value && j < n ? j : place;
    }
    return place;
}

/* A bound that at least `top` of the wave's logits reach: those over `order`,
 * and of equals those up to `place`.  It is taken from the lanes' maxima, bit
 * by bit the largest order that `top` lanes reach; a smaller one that few more
 * reach will do.  Where more reach the last, because they are equal, it is
 * the place up to which `top` do: so no more than `top` + kSlack lanes of the
 * wave hold any logit that reaches the bound. */
constexpr int kSlack = 8;
struct Bound {
    uint32_t order;
    int place;
};

template <int THREADS, int PER, int W>
__device__ __forceinline__ Bound wave_bound(const float x[PER], float lane_most, int top, int from, int n) {
    const uint32_t mine = order_of(lane_most), high = wave_most(mine), low = ~wave_most(~mine);
    /* the bits that all lanes share, and then one after the other */
    int bit = high == low ? -1 : 31 - __builtin_clz(high ^ low), reach = kWave;
    uint32_t order = bit < 0 ? high : high & ~((2u << bit) - 1);
    for (; bit >= 0 && reach > top + kSlack; bit--) {
        const uint32_t next = order | 1u << bit;
        const int count = __builtin_popcountll(__ballot(mine >= next));
        if (count >= top) {
            order = next;
            reach = count;
        }
    }
    if (reach <= top + kSlack) return Bound{order, INT32_MAX};
    const int need = top - __builtin_popcountll(__ballot(mine > order));
    const int place = mine == order ? first_place<THREADS, PER, W>(x, value_of(order), from, n) : INT32_MAX;
    int up_to = -1;                              // the largest that fewer than `need` do not pass
    for (int bit = 30; bit >= 0; bit--) {
        const int next = up_to + (1 << bit);
        if (__builtin_popcountll(__ballot(place <= next)) < need) up_to = next;
    }
    return Bound{order, up_to == INT32_MAX - 1 ? INT32_MAX : up_to + 1};
}

/* A workgroup to a row (one piece) or to a piece of it.  TOP: whether
 * alternatives are asked for.  Each wave finds a bound that `top` of its
 * logits reach; what reaches the highest of these is listed in LDS, a few
 * more than `top` as a rule, and a listed one's rank is the number of larger
 * ones in the list.  Rows with a NaN or +inf, whose sums say so, and lists
 * that would be too long (many large logits in one lane's places) go by
 * wave_top, all waves' in the end ranked alike. */
template <typename T, int THREADS, int PER, int W, bool TOP>
__global__ __launch_bounds__(THREADS, TOP ? 6 : 8) void lp_piece(B3Logits g, Outputs o, Pieces p) {
    constexpr int kWaves = THREADS / kWave, kList = 1024;
    static_assert(PER <= 32, "a bit for each");
    static_assert(kList >= kWaves * B3_MAX_TOP, "the waves' alternatives");
    __shared__ Sums part[kWaves];
    __shared__ Bound bounds[TOP ? kWaves : 1];
    __shared__ uint2 list[TOP ? kList : 1];
    __shared__ int places[TOP ? kList : 1];
    __shared__ int listed;
    const int64_t r = blockIdx.x / (unsigned)p.count;
    const int piece = blockIdx.x % (unsigned)p.count;
    const int from = piece * p.size, end = from + p.size, n = end < g.actions ? end : (int)g.actions;
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int64_t a = p.count == 1 ? o.taken[r] : -1;
    float x[PER];
    load_logits<T, THREADS, PER, W>(row_of<T>(g, r), mask_of(g, r), from, n, threadIdx.x, p.once, x);
    const float xa = taken_logit<T>(g, r, a);
    const int live = live_loads<THREADS, PER, W>(from, n);
    const float most = lane_max<PER, W>(x, live);
    const Sums mine = sums_of<kWave, PER, W>(x, live, most);
    if (lane == 0) part[wave] = mine;
    if (TOP) {
        const Bound b = wave_bound<THREADS, PER, W>(x, most, o.top, from, n);
        if (lane == 0) bounds[wave] = b;
        if (threadIdx.x == 0) listed = 0;
    }
    __syncthreads();
    if (!TOP && wave > 0) return;
    Sums s = part[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) s = join(s, part[w]);
    const float log_sum = logf(s.s);
    if (threadIdx.x == 0) {
        if (p.count == 1)
            finish_row(g, o, r, a, xa, s, log_sum);
        else
            p.sums[r * p.count + piece] = s;
    }
    if (!TOP) return;
    Bound bound = bounds[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) {
        const Bound b = bounds[w];
        if (b.order > bound.order || (b.order == bound.order && b.place < bound.place)) bound = b;
    }
    const float value = value_of(bound.order);
    int count = kList + 1;
    if (s.s == s.s) {
        uint32_t reaches = 0;                    // bit PER - 1 - i: x[i]
        if (most >= value) {
#pragma unroll
            for (int i = 0; i < PER; i++) reaches = reaches << 1 | (x[i] >= value);
        }
        if (__ballot(reaches != 0)) {
            /* the wave's part of the list, and the lane's of that */
            const int own = __builtin_popcount(reaches), upto = wave_scan(own);
            int at = 0;
            if (lane == kWave - 1) at = atomicAdd(&listed, upto);
            at = __builtin_amdgcn_readlane(at, kWave - 1) + upto - own;
            for (; reaches; at++) {
                const int i = PER - 1 - (31 - __builtin_clz(reaches));
                reaches &= ~(0x80000000u >> __builtin_clz(reaches));
                if (at < kList) places[at] = from + ((i / W) * THREADS + (int)threadIdx.x) * W + i % W;
            }
        }
        __syncthreads();
        count = listed;
        if (count <= kList) {
            /* their logits are fetched again: a thread cannot take those that
             * it has in registers by number */
            for (int i = threadIdx.x; i < count; i += THREADS) {
                const int j = places[i];
                const float xj = j < n ? logit(row_of<T>(g, r), mask_of(g, r), j) : -INFINITY;
                const bool in = j < n && (xj > value || (xj == value && j <= bound.place));
                list[i] = make_uint2(in ? order_of(xj) : 0, j);
            }
            __syncthreads();
        }
    }
    if (count > kList) {
        __syncthreads();
        uint32_t order[PER], my_order;
        int v, l, w;
#pragma unroll
        for (int i = 0; i < PER; i++)
            order[i] = from + ((i / W) * THREADS + (int)threadIdx.x) * W + i % W < n ? order_of(x[i]) : 0;
        wave_top<PER / W, W>(order, o.top, my_order, v, l, w);
        /* a wave of a short piece may have fewer than `top`: order 0 */
        if (lane < o.top)
            list[wave * o.top + lane] = make_uint2(my_order, from + (v * THREADS + wave * kWave + l) * W + w);
        __syncthreads();
        count = kWaves * o.top;
    }
    for (int i = threadIdx.x; i < count; i += THREADS) {
        const uint2 it = list[i];
        if (it.x == 0) continue;
        const uint64_t key = (uint64_t)it.x << 32 | ~it.y;
        int rank = 0;
#pragma unroll 8
        for (int k = 0; k < count; k++) {
            const uint2 other = list[k];
            rank += ((uint64_t)other.x << 32 | ~other.y) > key;
        }
        if (rank >= o.top) continue;
        if (p.count == 1)
            write_top(o, r, rank, it.x, it.y, s, log_sum);
        else
            p.top[(r * p.count + piece) * o.top + rank] = it;
    }
    /* a piece of fewer than `top` actions fills its list up */
    const int have = n - from;
    if (p.count > 1 && (int)threadIdx.x < o.top && (int)threadIdx.x >= have)
        p.top[(r * p.count + piece) * o.top + threadIdx.x] = make_uint2(0, 0);
}

/* A wave to a row, HEADS pieces to a lane.  With alternatives three more
 * waves fetch the lists.  Everything is fetched before anything is used. */
template <typename T, int HEADS>
__global__ __launch_bounds__(kThreads) void lp_join(B3Logits g, Outputs o, Pieces p) {
    extern __shared__ uint2 lists[];             // [count][top]
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x;
    const int64_t a = o.taken[r];
    Sums sums[HEADS];
#pragma unroll
    for (int q = 0; q < HEADS; q++) {
        const int c = q * kWave + lane;
        sums[q] = p.sums[r * p.count + (c < p.count ? c : 0)];
    }
    /* the pieces' lists are sorted, and of equal orders the one of the lower
     * piece has the lower action */
    const int entries = p.count * o.top;
    const uint2* from = p.top + r * entries;
    for (int i = threadIdx.x; i < entries; i += 4 * blockDim.x) {
        uint2 it[4];
#pragma unroll
        for (int k = 0; k < 4; k++) it[k] = from[min(i + k * (int)blockDim.x, entries - 1)];
#pragma unroll
        for (int k = 0; k < 4; k++) lists[min(i + k * (int)blockDim.x, entries - 1)] = it[k];
    }
    const float xa = taken_logit<T>(g, r, a);
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    Sums part = {0, 0, 0};
#pragma unroll
    for (int q = 0; q < HEADS; q++)
        if (q * kWave + lane < p.count) part = join(part, sums[q]);
#pragma unroll
    for (int d = 1; d < kWave; d *= 2)
        part = join(part, Sums{__shfl_xor(part.m, d), __shfl_xor(part.s, d), __shfl_xor(part.d, d)});
    const float log_sum = logf(part.s);
    if (lane == 0) finish_row(g, o, r, a, xa, part, log_sum);
    if (!o.top) return;
    /* the first of each list that is left, the largest of these, and so on;
     * lane k keeps the k-th */
    uint2 head[HEADS], mine = make_uint2(0, 0);
    int next[HEADS];
#pragma unroll
    for (int q = 0; q < HEADS; q++) {
        const int c = q * kWave + lane;
        head[q] = c < p.count ? lists[c * o.top] : make_uint2(0, 0);
        next[q] = c * o.top + 1;
    }
    for (int k = 0; k < o.top; k++) {
        uint32_t most = head[0].x;
#pragma unroll
        for (int q = 1; q < HEADS; q++) most = most > head[q].x ? most : head[q].x;
        most = wave_most(most);
        bool found = false;
#pragma unroll
        for (int q = 0; q < HEADS; q++) {
            const uint64_t have = __ballot(head[q].x == most);
            if (!found && have) {
                found = true;
                const int who = __builtin_ctzll(have);
                const uint32_t action = __builtin_amdgcn_readlane(head[q].y, who);
                mine = lane == k ? make_uint2(most, action) : mine;
                if (lane == who) {
                    head[q] = next[q] < (q * kWave + lane + 1) * o.top ? lists[next[q]] : make_uint2(0, 0);
                    next[q]++;
                }
            }
        }
    }
    if (lane < o.top) write_top(o, r, lane, mine.x, mine.y, part, log_sum);
}

/* ---- backward ---- */

/* What a row's gradient is made of. */
struct Upstream {
    const int64_t* taken;
    const float* stats;
    const float* entropy;
    const float* d_log_prob;
    int64_t d_log_prob_stride;
    const float* d_entropy;
    int64_t d_entropy_stride;
    void* out;
    int64_t row_stride;
    bool once;
};

struct RowGradient {
    int64_t a;
    float m, log_sum, h, dl, dh;
    bool empty;
};

__device__ RowGradient row_gradient(const Upstream& u, int64_t r, int64_t actions) {
    RowGradient q;
    q.a = u.taken[r];
    q.m = u.stats[2 * r];
    q.log_sum = u.stats[2 * r + 1];
    q.h = u.entropy[r];
    q.dl = u.d_log_prob && q.a >= 0 ? u.d_log_prob[r * u.d_log_prob_stride] : 0.0f;
    if (q.a >= actions) q.dl *= NAN;
    q.dh = u.d_entropy ? u.d_entropy[r * u.d_entropy_stride] : 0.0f;
    q.empty = q.log_sum == -INFINITY;
    return q;
}

/* p log p is 0 where p is, also where log p is -inf. */
__device__ float gradient_of(const RowGradient& q, float x, bool taken) {
    const float lp = x - q.m - q.log_sum, p = __builtin_amdgcn_exp2f(lp * kLog2e);
    const float d = (taken ? q.dl : 0.0f) - p * __builtin_fmaf(q.dh, fmaxf(lp, -1e4f) + q.h, q.dl);
    return q.empty || x == -INFINITY ? 0.0f : d;
}

template <typename T, int G, int PER, int W>
__device__ void backward_row(const B3Logits& g, const Upstream& u, int64_t r, int from, int lane) {
    const RowGradient q = row_gradient(u, r, g.actions);
    const int n = (int)g.actions;
    float x[PER];
    load_logits<T, G, PER, W>(row_of<T>(g, r), mask_of(g, r), from, n, lane, u.once, x);
    T* out = (T*)u.out + r * u.row_stride;
#pragma unroll
    for (int v = 0; v < PER / W; v++) {
        const int j = from + (v * G + lane) * W;
        Pack<T, W> p;
#pragma unroll
        for (int w = 0; w < W; w++) p.v[w] = (T)gradient_of(q, x[v * W + w], j + w == q.a);
        if (j + W <= n) {
            Stream<T, W>::store(out + j, p);
        } else {
#pragma unroll
            for (int w = 0; w < W; w++)
                if (j + w < n) out[j + w] = p.v[w];
        }
    }
}

template <typename T, int G, int PER, int W>
__global__ __launch_bounds__(kThreads) void lp_small_backward(B3Logits g, Upstream u) {
    const int64_t r = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / G;
    if (r < g.rows) backward_row<T, G, PER, W>(g, u, r, 0, threadIdx.x % G);
}

/* A workgroup to a piece of kThreads PER actions. */
template <typename T, int PER, int W>
__global__ __launch_bounds__(kThreads) void lp_piece_backward(B3Logits g, Upstream u, unsigned pieces) {
    backward_row<T, kThreads, PER, W>(g, u, blockIdx.x / pieces, (int)(blockIdx.x % pieces) * (kThreads * PER),
        threadIdx.x);
}

/* ---- launches ---- */

/* Calls f with the shape for rows of up to 2,048 actions: the fewest lanes
 * that hold them at 16 each, or 32, since what is done once a row is shared by
 * few elements already; four in a lane where that is all. */
template <typename T, typename F>
void with_small(int64_t actions, F f) {
    constexpr int W = 16 / sizeof(T);
    if (actions <= 4)
        f.template operator()<T, 1, 4, 4>();
    else if (actions <= 16)
        f.template operator()<T, 1, 16, W>();
    else if (actions <= 64)
        f.template operator()<T, 4, 16, W>();
    else if (actions <= 256)
        f.template operator()<T, 16, 16, W>();
    else if (actions <= 1024)
        f.template operator()<T, 64, 16, W>();
    else
        f.template operator()<T, 64, 32, W>();
}

constexpr int kSmall = 2048, kShortPiece = 4096, kPiece = 8192;
constexpr int64_t kFill = 512;                   // workgroups: two to a compute unit

template <typename F>
void with_type(int type, F f) {
    if (type == B3_F32)
        f(float());
    else if (type == B3_F16)
        f((_Float16)0);
    else
        f((__bf16)0);
}

/* Logits that the caches cannot hold from the forward pass to the backward go
 * past them (4,096 rows of 131,072 in bf16: 161 and 352 us forward and
 * backward, not 177 and 369); smaller ones do not (8,192 rows of 1,024: 17.0
 * us for both passes in a graph, 18.6 past the caches). */
bool stream_logits(const B3Logits& g) { return g.rows * g.actions * (g.type == B3_F32 ? 4 : 2) > (int64_t)1 << 28; }

/* Pieces of a row.  8,192 actions to a workgroup of 256 threads, also where
 * one of 512 could hold the row (16,384 rows of 16,384 in bf16: 88 us, not
 * 96; of 14,000: 88 us, not 117): with fewer to a barrier, loads and sums of
 * different workgroups overlap.  Where pieces of 8,192 would not give every
 * compute unit two, 4,096. */
Pieces pieces_of(int64_t rows, int64_t actions) {
    Pieces p = {};
    p.size = kPiece;
    if (rows * ceil_div(actions, kPiece) < kFill && ceil_div(actions, kShortPiece) <= kMaxPieces) p.size = kShortPiece;
    p.count = actions <= kSmall ? 1 : (int)ceil_div(actions, p.size);
    return p;
}

struct SmallForward {
    const B3Logits& g;
    const Outputs& o;
    hipStream_t stream;
    template <typename T, int G, int PER, int W>
    void operator()() const {
        lp_small<T, G, PER, W><<<(unsigned)ceil_div(g.rows, kThreads / G), kThreads, 0, stream>>>(g, o);
    }
};

struct SmallBackward {
    const B3Logits& g;
    const Upstream& u;
    hipStream_t stream;
    template <typename T, int G, int PER, int W>
    void operator()() const {
        lp_small_backward<T, G, PER, W><<<(unsigned)ceil_div(g.rows, kThreads / G), kThreads, 0, stream>>>(g, u);
    }
};

template <typename T, int THREADS, int PER, int W>
void launch_piece(const B3Logits& g, const Outputs& o, const Pieces& p, unsigned grid, hipStream_t stream) {
    if (o.top)
        lp_piece<T, THREADS, PER, W, true><<<grid, THREADS, 0, stream>>>(g, o, p);
    else
        lp_piece<T, THREADS, PER, W, false><<<grid, THREADS, 0, stream>>>(g, o, p);
}

template <typename T>
hipError_t forward(const B3Logits& g, const Outputs& o, Pieces p, hipStream_t stream) {
    constexpr int W = 16 / sizeof(T);
    if (g.actions <= kSmall) {
        with_small<T>(g.actions, SmallForward{g, o, stream});
        return hipGetLastError();
    }
    const unsigned grid = (unsigned)(g.rows * p.count);
    const int64_t most = p.count == 1 ? g.actions : p.size;
    if (most <= kShortPiece)
        launch_piece<T, 128, kShortPiece / 128, W>(g, o, p, grid, stream);
    else
        launch_piece<T, 256, kPiece / 256, W>(g, o, p, grid, stream);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess || p.count == 1) return err;
    const size_t lists = (size_t)p.count * o.top * sizeof(uint2);
    const int threads = o.top ? kThreads : kWave;
    if (p.count <= kWave)
        lp_join<T, 1><<<(unsigned)g.rows, threads, lists, stream>>>(g, o, p);
    else
        lp_join<T, kMaxPieces / kWave><<<(unsigned)g.rows, threads, lists, stream>>>(g, o, p);
    return hipGetLastError();
}

template <typename T>
hipError_t backward(const B3Logits& g, const Upstream& u, hipStream_t stream) {
    constexpr int W = 16 / sizeof(T), PER = 4 * W;
    if (g.actions <= kSmall) {
        with_small<T>(g.actions, SmallBackward{g, u, stream});
    } else {
        const int64_t pieces = ceil_div(g.actions, kThreads * PER);
        lp_piece_backward<T, PER, W><<<(unsigned)(g.rows * pieces), kThreads, 0, stream>>>(g, u, (unsigned)pieces);
    }
    return hipGetLastError();
}

/* Rows to a launch: no kernel has more workgroups to a row than a piece of
 * 4,096 (or less) takes. */
int64_t rows_of_launch(int64_t actions) { return kMostBlocks / ceil_div(actions, kShortPiece); }

/* Rows `first` to `first` + `rows`. */
B3Logits some_rows(B3Logits g, int64_t first, int64_t rows) {
    g.data = (const char*)g.data + first * g.row_stride * (g.type == B3_F32 ? 4 : 2);
    if (g.mask) g.mask += first * g.mask_row_stride;
    g.rows = rows;
    return g;
}

bool valid(const B3Logits& g, const int64_t* taken) {
    return is_float_type(g.type) && g.rows >= 0 && g.rows <= 0x7fffffff && g.actions >= 1 && g.actions <= kMaxActions
        && g.row_stride >= g.actions
        && (!g.mask || g.mask_row_stride == 0 || g.mask_row_stride >= g.actions) && (g.rows == 0 || (g.data && taken));
}

}  // namespace
}  // namespace b3p

using namespace b3p;

extern "C" {

size_t b3_log_probs_workspace(int64_t rows, int64_t actions, int top) {
    if (rows <= 0 || actions <= kSmall || actions > kMaxActions || top < 0) return 0;
    const Pieces p = pieces_of(rows, actions);
    return p.count == 1 ? 0 : (size_t)rows * p.count * (16 + (size_t)top * sizeof(uint2));
}

hipError_t b3_log_probs_gpu(B3Logits g, const int64_t* taken, float* log_prob, float* entropy, float* stats, int top,
        float* top_log_prob, int64_t* top_action, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!valid(g, taken) || top < 0 || top > B3_MAX_TOP || top > g.actions) return hipErrorInvalidValue;
    const size_t need = b3_log_probs_workspace(g.rows, g.actions, top);
    if (!holds(workspace, workspace_bytes, need)) return hipErrorInvalidValue;
    if (g.rows == 0) return hipSuccess;
    if (!log_prob || !entropy || (top && (!top_log_prob || !top_action))) return hipErrorInvalidValue;
    Outputs o = {taken, log_prob, entropy, stats, top, top_log_prob, top_action};
    Pieces p = pieces_of(g.rows, g.actions);
    p.once = stream_logits(g);
    p.top = (uint2*)workspace;
    p.sums = (Sums*)((char*)workspace + (size_t)g.rows * p.count * top * sizeof(uint2));
    const int64_t most = rows_of_launch(g.actions);
    hipError_t err = hipSuccess;
    for (int64_t r = 0; r < g.rows && err == hipSuccess; r += most) {
        const int64_t rows = g.rows - r < most ? g.rows - r : most;
        const B3Logits part = some_rows(g, r, rows);
        with_type(g.type, [&](auto t) { err = forward<decltype(t)>(part, o, p, stream); });
        o.taken += rows;
        o.log_prob += rows;
        o.entropy += rows;
        if (stats) o.stats += 2 * rows;
        if (top) {
            o.top_log_prob += rows * top;
            o.top_action += rows * top;
        }
        if (need) {
            p.sums += rows * p.count;
            p.top += rows * p.count * top;
        }
    }
    return err;
}

hipError_t b3_log_probs_backward_gpu(B3Logits g, const int64_t* taken, const float* stats, const float* entropy,
        const float* d_log_prob, int64_t dl_stride, const float* d_entropy, int64_t dh_stride, void* d_logits,
        int64_t d_row_stride, hipStream_t stream) {
    if (!valid(g, taken) || d_row_stride < g.actions || dl_stride < 0 || dh_stride < 0) return hipErrorInvalidValue;
    if (g.rows == 0) return hipSuccess;
    if (!stats || !entropy || !d_logits) return hipErrorInvalidValue;
    Upstream u = {taken, stats, entropy, d_log_prob, dl_stride, d_entropy, dh_stride, d_logits, d_row_stride,
        stream_logits(g)};
    const int64_t most = rows_of_launch(g.actions);
    hipError_t err = hipSuccess;
    for (int64_t r = 0; r < g.rows && err == hipSuccess; r += most) {
        const int64_t rows = g.rows - r < most ? g.rows - r : most;
        const B3Logits part = some_rows(g, r, rows);
        with_type(g.type, [&](auto t) { err = backward<decltype(t)>(part, u, stream); });
        u.taken += rows;
        u.stats += 2 * rows;
        u.entropy += rows;
        if (d_log_prob) u.d_log_prob += rows * dl_stride;
        if (d_entropy) u.d_entropy += rows * dh_stride;
        u.out = (char*)u.out + rows * d_row_stride * (g.type == B3_F32 ? 4 : 2);
    }
    return err;
}

}  // extern "C"
