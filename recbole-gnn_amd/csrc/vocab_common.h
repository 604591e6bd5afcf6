// vocab_common.h — pieces shared by the operators over large item vocabularies (embed.hip, logits.hip, score_i8.hip): the three
// element types, 16-byte vectors of them, and reductions over a workgroup.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "internal.h"

namespace rbg {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

inline bool elem_ok(int dtype) { return dtype == RBG_F32 || dtype == RBG_BF16 || dtype == RBG_F16; }
inline int elem_size(int dtype) { return dtype == RBG_F32 ? 4 : 2; }
__device__ __forceinline__ bool on_16_dev(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool on_16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// N consecutive elements moved by one load or store (of 16 bytes at most; longer ones by several).
template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The same from and to any element boundary: global memory takes 16-byte accesses at every address of an element on this target.
template <class T, int N>
__device__ __forceinline__ Vec<T, N> load_any(const T *p) {
    Vec<T, N> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <class T, int N>
__device__ __forceinline__ void store_any(T *p, const Vec<T, N> &v) { __builtin_memcpy(p, &v, sizeof(v)); }

// All arithmetic is in 32 bits; a store rounds once, to nearest even (what the casts compile to on gfx950).
template <class T>
__device__ __forceinline__ float to_f32(T x) { return (float)x; }
template <class T>
__device__ __forceinline__ T from_f32(float x) { return (T)x; }

constexpr int kWave = 64;

// A grid holds fewer than 2^32 threads per dimension: operators with a workgroup of up to 1 024 threads per row launch for this many rows
// at a time.
constexpr int64_t kRowsPerLaunch = 1 << 21;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Runs f(type tag) for the element type named by an RBG_* code that elem_ok() has accepted.
template <class F>
inline int with_elem(int dtype, F f) {
    if (dtype == RBG_F32) return f(float{});
    if (dtype == RBG_BF16) return f(bf16_t{});
    return f(f16_t{});
}

}  // namespace rbg
