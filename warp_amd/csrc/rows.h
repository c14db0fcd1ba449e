// rows.h — device helpers of the operators on packed rows (conv.hip, scan.hip,
// dispatch.hip): elements of three types read and written a vector at a time,
// and where packed sequences begin and end.
#ifndef WARP_ROWS_H
#define WARP_ROWS_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "warp_hip.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// V elements, read and written at the alignment of one: rows of odd widths
// and strides go as wide as aligned ones (this target's global loads take any
// alignment).
template <typename T, int V>
struct vec_t {
    typedef T reg __attribute__((ext_vector_type(V)));
    typedef reg mem __attribute__((aligned(sizeof(T))));
    reg e;
};
template <typename T>
struct rows_of;
template <>
struct rows_of<float> {
    static constexpr int V = 4;                   // elements in 16 bytes
};
template <>
struct rows_of<uint32_t> {
    static constexpr int V = 4;
};
template <>
struct rows_of<uint16_t> {
    static constexpr int V = 8;
};
template <>
struct rows_of<bf16_t> {
    static constexpr int V = 8;
};
template <>
struct rows_of<f16_t> {
    static constexpr int V = 8;
};

// n of V elements (the last vector of a row may be short; the rest are 0)
template <typename T, int V>
__device__ __forceinline__ vec_t<T, V> load_vec(const T *p, int n) {
    vec_t<T, V> v;
    v.e = 0;
    if (n >= V) {
        v.e = *(const typename vec_t<T, V>::mem *)p;
    } else if (n > 0) {
        for (int i = 0; i < n; i++) v.e[i] = p[i];
    }
    return v;
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const vec_t<T, V> &v, int n) {
    if (n >= V) {
        *(typename vec_t<T, V>::mem *)p = v.e;
    } else if (n > 0) {
        for (int i = 0; i < n; i++) p[i] = v.e[i];
    }
}

// exp and the sigmoid on the exponential instruction (2^x within an ulp; the
// product with log2 e adds |x| 2^-24 of relative error, which only matters
// where the result is negligible beside 1)
__device__ __forceinline__ float rows_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float rows_silu(float x) { return x * __builtin_amdgcn_rcpf(1.0f + rows_exp(-x)); }

// Where sequence s of a packed batch begins and ends: starts[s] and
// starts[s + 1], kept within the rows there are.
struct seq_t {
    int b, e;
};
__device__ __forceinline__ seq_t seq_at(const int *__restrict__ starts, int s, int tokens) {
    const int b = min(max(starts[s], 0), tokens), e = min(max(starts[s + 1], 0), tokens);
    return {b, max(b, e)};
}
// the first sequence that does not end before row t (n_seq if all do)
__device__ __forceinline__ int seq_from(const int *__restrict__ starts, int n_seq, int t) {
    int lo = 0, hi = n_seq;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid + 1] >= t) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
// the slot of sequence s's state; -1: none, its rows are not computed
__device__ __forceinline__ int seq_slot(const int *__restrict__ slots, int s, int n_slots) {
    const int k = slots ? slots[s] : s;
    return (unsigned)k < (unsigned)n_slots ? k : -1;
}

#endif
