// Element types of the trunk operators (marl_gated.hip, marl_norm.hip, marl_dropout.hip, marl_sample.hip): float32,
// bfloat16 and float16 in memory, float32 in registers; 16-byte chunks that need no more than element alignment.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "marl_env.h"

namespace marl_types {

typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T> struct Chunk { static constexpr int n = 16 / (int)sizeof(T); };        // elements of 16 bytes

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(f16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }      // to nearest, ties to even

template <typename T> struct alignas(16) Vec { T e[Chunk<T>::n]; };

// 16 bytes from an address aligned to one element only: the hardware takes any alignment in global memory, so this is
// one load; the compiler must merely not assume more.
template <typename T> __device__ __forceinline__ Vec<T> load_chunk(const T* p) {
    Vec<T> v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, sizeof(T)), 16);
    return v;
}
template <typename T> __device__ __forceinline__ void store_chunk(T* p, const Vec<T>& v) {
    __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), &v, 16);
}
typedef unsigned int uint4v __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) Unaligned { uint4v v; };
// `left` elements remain from p on: whole chunks in one access, the last one element by element (the rest reads as zero)
template <typename T> __device__ __forceinline__ Vec<T> load_part(const T* p, int64_t left) {
    constexpr int n = Chunk<T>::n;
    if (left >= n) return load_chunk(p);
    Vec<T> v;
#pragma unroll
    for (int i = 0; i < n; ++i) v.e[i] = i < left ? p[i] : (T)0.0f;
    return v;
}
template <typename T> __device__ __forceinline__ void store_part(T* p, const Vec<T>& v, int64_t left) {
    constexpr int n = Chunk<T>::n;
    if (left >= n) { store_chunk(p, v); return; }
#pragma unroll
    for (int i = 0; i < n; ++i) if (i < left) p[i] = v.e[i];
}

// The chunk of a row of n elements that begins at element c, zeros from n on.  Rows of a chunk or more: the last whole chunk
// is loaded where c lies past it, and moved; no branch, whose loads would be waited for one by one.
template <typename T> __device__ __forceinline__ Vec<T> load_clipped(const T* row, int64_t c, int64_t n) {
    constexpr int CE = Chunk<T>::n;
    if (n < CE) return load_part(row + (c < n ? c : 0), n - c);
    const int64_t at = c < n - CE ? c : n - CE;
    Vec<T> v = load_chunk(row + at);
    const int by = c - at < CE ? (int)(c - at) : CE;
#pragma unroll
    for (int step = 1; step < CE; step *= 2)
#pragma unroll
        for (int e = 0; e < CE; ++e) v.e[e] = (by & step) && e + step < CE ? v.e[e + step] : v.e[e];
#pragma unroll
    for (int e = 0; e < CE; ++e) v.e[e] = e + by < CE ? v.e[e] : (T)0.0f;
    return v;
}
// N elements, 8 or 16 bytes.  stream_part: store_part for results that nothing reads soon, past the caches
template <typename T, int N> struct alignas(N * sizeof(T)) Part { T e[N]; };
typedef unsigned int uint2v __attribute__((ext_vector_type(2)));
struct __attribute__((packed, aligned(2))) Unaligned8 { uint2v v; };
template <typename T, int N> __device__ __forceinline__ void stream_part(T* p, const Part<T, N>& v, int64_t left) {
    static_assert(N * sizeof(T) == 16 || N * sizeof(T) == 8, "one store");
    if (left >= N) {
        if constexpr (N * sizeof(T) == 16) __builtin_nontemporal_store(__builtin_bit_cast(uint4v, v), &((Unaligned*)p)->v);
        else __builtin_nontemporal_store(__builtin_bit_cast(uint2v, v), &((Unaligned8*)p)->v);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) if (i < left) p[i] = v.e[i];
}

}  // namespace marl_types

// Calls FN<T>(...) for the element type of `dtype`
#define MARL_BY_TYPE(dtype, FN, ...)                                  \
    ((dtype) == MARL_F32 ? FN<float>(__VA_ARGS__)                     \
     : (dtype) == MARL_BF16 ? FN<marl_types::bf16>(__VA_ARGS__)       \
                            : FN<marl_types::f16>(__VA_ARGS__))
