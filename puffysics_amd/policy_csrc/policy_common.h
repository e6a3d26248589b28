/*
 * policy_common.h - what the kernels of include/b3_policy.h share: loads and
 * stores of vectors with the alignment of their elements, conversions, and the
 * bounds of launches and workspaces.
 */
#ifndef PUFFYSICS_AMD_POLICY_COMMON_H
#define PUFFYSICS_AMD_POLICY_COMMON_H

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "b3_policy.h"

namespace b3p {

constexpr int kWave = 64;

/* N elements that lie anywhere their type may: the hardware takes wide
 * global loads and stores at any such address. */
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[N];
};

/* Unsigned numbers that lie anywhere, as arrays of bytes do. */
template <typename T, int N>
struct __attribute__((packed, aligned(1))) Bytes {
    T v[N];
};

/* A Pack's data where it is used once: not kept in the caches.  N elements
 * are 4, 8 or 16 bytes. */
template <typename T, int N>
struct Stream {
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(T) * N / 4), aligned(sizeof(T))));
    static __device__ __forceinline__ Pack<T, N> load(const T* p) {
        return __builtin_bit_cast(Pack<T, N>, __builtin_nontemporal_load((const Words*)p));
    }
    static __device__ __forceinline__ void store(T* p, Pack<T, N> v) {
        __builtin_nontemporal_store(__builtin_bit_cast(Words, v), (Words*)p);
    }
};

inline __device__ float to_float(float x) { return x; }
inline __device__ float to_float(_Float16 x) { return (float)x; }
inline __device__ float to_float(__bf16 x) { return (float)x; }

inline bool is_float_type(int type) { return type == B3_F32 || type == B3_F16 || type == B3_BF16; }
/* Workgroups of up to 256 threads that a launch may have: it takes fewer than
 * 2^32 threads. */
constexpr int64_t kMostBlocks = (1 << 24) - 1;

/* Whether a workspace has `need` bytes, aligned for what kernels keep there. */
inline bool holds(const void* workspace, size_t bytes, size_t need) {
    return need == 0 || (bytes >= need && workspace && (uintptr_t)workspace % 8 == 0);
}

inline __host__ __device__ int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace b3p
#endif
