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

// A thread's vector of a row of C elements. Where C is no multiple of V the
// last thread's begins early, at C - V, so that it loads a whole vector too,
// and it stores only what no other thread has: its elements from `skip` on.
// ONE: rows shorter than a vector, element by element.
template <typename T, bool ONE, int V = rows_of<T>::V>
struct cols_t {
    typedef vec_t<T, V> vec;
    int c, skip, n;                               // its first column; see above; elements there are

    __device__ __forceinline__ cols_t(int c0, int C) : c(ONE ? c0 : min(c0, C - V)), skip(c0 - c), n(min(V, C - c)) {}
    __device__ __forceinline__ vec load(const T *p) const {
        vec v;
        if (!ONE) {
            v.e = *(const typename vec::mem *)p;
            return v;
        }
        v.e = 0;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) v.e[i] = p[i];
        return v;
    }
    // The same of rows that nothing reads again: they take no one's place in
    // the caches.
    __device__ __forceinline__ vec take(const T *p) const {
        if (ONE) return load(p);
        vec v;
        v.e = __builtin_nontemporal_load((const typename vec::mem *)p);
        return v;
    }
    __device__ __forceinline__ void part(T *p, const vec &v) const {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i >= skip && i < n) p[i] = v.e[i];
    }
    __device__ __forceinline__ void store(T *p, const vec &v) const {
        if (!ONE && skip == 0) *(typename vec::mem *)p = v.e;
        else part(p, v);
    }
    // The same past the caches, for outputs that are larger than those: what
    // they would push out of L2 is worth more.
    __device__ __forceinline__ void stream(T *p, const vec &v) const {
        if (!ONE && skip == 0) __builtin_nontemporal_store(v.e, (typename vec::mem *)p);
        else part(p, v);
    }
};
// n of V elements (0 where there are none)
template <typename T, int V>
__device__ __forceinline__ vec_t<T, V> load_vec(const T *p, int n) {
    vec_t<T, V> v;
    v.e = 0;
    if (n >= V) {
        v.e = *(const typename vec_t<T, V>::mem *)p;
    } else if (n > 0) {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) v.e[i] = p[i];
    }
    return v;
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const vec_t<T, V> &v, int n) {
    if (n >= V) {
        *(typename vec_t<T, V>::mem *)p = v.e;
    } else if (n > 0) {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) p[i] = v.e[i];
    }
}
// (past the caches, as above)
template <typename T, int V>
__device__ __forceinline__ void stream_vec(T *p, const vec_t<T, V> &v, int n) {
    if (n >= V) __builtin_nontemporal_store(v.e, (typename vec_t<T, V>::mem *)p);
    else store_vec<T, V>(p, v, n);
}

// exp and the sigmoid on the exponential instruction (2^x within an ulp; the
// product with log2 e adds |x| 2^-24 of relative error, which only matters
// where the result is negligible beside 1)
__device__ __forceinline__ float rows_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float rows_silu(float x) { return x * __builtin_amdgcn_rcpf(1.0f + rows_exp(-x)); }

// The sequences of a packed batch: sequence s holds the rows b .. e - 1,
// starts[s] and starts[s + 1] kept within the rows there are, and its state
// is in a slot (-1: in none, its rows are not computed). A wave loads up to 63
// sequences at once, a lane each, so that finding one and walking on from it
// costs one trip to memory; of more it searches 64 at a time.
struct seq_t {
    int b, e, slot;
};
struct seqs_t {
    const int *starts, *slots;
    int n, tokens, n_slots, lane, b, e, k;
    bool few;

    // (all 64 lanes take part here and in from())
    __device__ __forceinline__ seqs_t(const int *st, const int *sl, int n_seq, int rows, int ns)
        : starts(st), slots(sl), n(n_seq), tokens(rows), n_slots(ns), lane(threadIdx.x & 63), few(n_seq < 64) {
        const int i = min(lane, n - 1);
        b = few ? starts[i] : 0;
        e = few ? starts[i + 1] : 0;
        k = few && slots ? slots[i] : i;
    }
    // the first sequence that does not end before row t (n if all do)
    __device__ __forceinline__ int from(int t) const {
        if (few) {
            const uint64_t m = __ballot(lane < n && e >= t);
            return m ? __builtin_ctzll(m) : n;
        }
        int lo = 0, hi = n;                       // it is in lo .. hi
        while (hi > lo) {
            const int step = (hi - lo + 63) >> 6, i = lo + lane * step;
            const uint64_t m = __ballot(i < hi && starts[min(i, n - 1) + 1] < t);
            const int c = __popcll(m);            // that many of the samples are before it
            if (c == 0) return lo;
            lo += (c - 1) * step + 1;
            hi = min(hi, lo + step - 1);
        }
        return lo;
    }
    __device__ __forceinline__ seq_t at(int s) const {
        int vb, ve, vk;
        if (few) {
            vb = __builtin_amdgcn_readlane(b, s);
            ve = __builtin_amdgcn_readlane(e, s);
            vk = __builtin_amdgcn_readlane(k, s);
        } else {
            vb = starts[s];
            ve = starts[s + 1];
            vk = slots ? slots[s] : s;
        }
        vb = min(max(vb, 0), tokens);
        ve = min(max(ve, 0), tokens);
        return {vb, max(vb, ve), (unsigned)vk < (unsigned)n_slots ? vk : -1};
    }
};
// one token of each sequence: its slot
__device__ __forceinline__ int seq_slot(const int *__restrict__ slots, int s, int n_slots) {
    const int k = slots ? slots[s] : s;
    return (unsigned)k < (unsigned)n_slots ? k : -1;
}

#endif
