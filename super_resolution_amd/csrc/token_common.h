// What the kernels on rows of channels ("tokens") share: element types, 16-byte units, fixed-order sums.
#pragma once
#include <type_traits>
#include <utility>

#include "sr355_internal.h"

namespace sr355 {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef unsigned tok_v4u __attribute__((ext_vector_type(4)));
typedef unsigned tok_v2u __attribute__((ext_vector_type(2)));

// f(0), f(1), ..., f(N - 1) with the index as a type, for what has to be an immediate of an instruction.
template <typename F, size_t... I>
__device__ __forceinline__ void tok_static_for_impl(F &&f, std::index_sequence<I...>) {
    (f(std::integral_constant<int, (int)I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void tok_static_for(F &&f) {
    tok_static_for_impl(f, std::make_index_sequence<N>{});
}

// One 16-byte unit of a row.
template <typename T>
struct TokUnit {
    static constexpr int E = 16 / sizeof(T);
    T v[E];
};

template <typename T>
__device__ __forceinline__ TokUnit<T> tok_load_unit(const T *p) {
    TokUnit<T> u;
    const tok_v4u raw = *reinterpret_cast<const tok_v4u *>(p);
    __builtin_memcpy(u.v, &raw, 16);
    return u;
}
template <typename T>
__device__ __forceinline__ void tok_store_unit(T *p, const TokUnit<T> &u) {
    tok_v4u raw;
    __builtin_memcpy(&raw, u.v, 16);
    *reinterpret_cast<tok_v4u *>(p) = raw;
}

// E consecutive elements as floats: one 16-byte access where E > 1 (the caller has checked the alignment).
template <typename T, int E>
__device__ __forceinline__ void tok_load(const T *p, float (&v)[E]) {
    if constexpr (E == 1) {
        v[0] = (float)p[0];
    } else {
        const TokUnit<T> u = tok_load_unit(p);
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = (float)u.v[j];
    }
}
template <typename T, int E>
__device__ __forceinline__ void tok_store(T *p, const float (&v)[E]) {
    if constexpr (E == 1) {
        p[0] = (T)v[0];
    } else {
        TokUnit<T> u;
#pragma unroll
        for (int j = 0; j < E; ++j) u.v[j] = (T)v[j];
        tok_store_unit(p, u);
    }
}

// E consecutive weights of a layer whose parameters are fp32 (`w32`) or of the activations' type T.
template <typename T, int E>
__device__ __forceinline__ void tok_load_param(const void *w, bool w32, size_t at, float (&v)[E]) {
    if (w32) {
        const float *p = (const float *)w + at;
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = p[j];
    } else {
        const T *p = (const T *)w + at;
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = (float)p[j];
    }
}

// Sum over aligned groups of L lanes (a power of two up to 64) in a fixed order, result in every lane of the group.
template <int L>
__device__ __forceinline__ float tok_lane_sum(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

int launch_tok_sum_parts(const float *parts, int n_parts, long long stride, const long long *first, const int *count, void *const *out,
                         int n_out, int out_dtype, hipStream_t stream);

inline size_t tok_type_bytes(int dtype) { return dtype == SR355_DTYPE_F32 ? 4 : 2; }
inline bool tok_dtype_ok(int dtype) {
    return dtype == SR355_DTYPE_BF16 || dtype == SR355_DTYPE_F32 || dtype == SR355_DTYPE_F16;
}
inline bool tok_aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline long long tok_cdiv(long long a, long long b) { return (a + b - 1) / b; }

}  // namespace sr355
