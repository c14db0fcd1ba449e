// dispatch.hip — tokens sorted by expert and brought back: the operators
// between a router's picks (warp_hip_route) and experts that the caller
// computes itself.
//   warp_hip_expert_dispatch: the pairs (token, k) in a stable order by
//     expert, and each pair's row of x there
//   warp_hip_expert_combine: out[t] = resid[t] + sum_k w[t][k] y[pos[t][k]]
//   warp_hip_expert_combine_backward: dy[pos[t][k]] = w[t][k] dout[t],
//     dw[t][k] = <dout[t], y[pos[t][k]]>
// All are bound by memory: rows are read once and written once, in 16-byte
// vectors. Nothing is summed by atomics, so every result is the same each time.

#include "rows.h"
#include "warp_internal.h"

constexpr int SORT_PAIRS = 2048;                  // pairs of a sorting block, 256 a wave's step
constexpr int SORT_WAVES = 8;

struct sort_p {
    int tokens, K, E, pairs, blocks, bits;
    const int *idx;
    int *offsets, *perm, *pos;
    int *rank, *count;                            // [pairs], [blocks][E]
    int hidden;
    const void *x;
    void *xs;
    size_t ldx, ldxs;
};

// How many of the wave's earlier lanes have this lane's key, and how many
// lanes have it: the lanes that agree in every bit of it.
__device__ __forceinline__ void same_key(int key, int bits, bool in, int lane, int &before, int &all) {
    uint64_t m = __ballot(in);
    for (int b = 0; b < bits; b++) {
        const uint64_t one = __ballot(key >> b & 1);
        m &= key >> b & 1 ? one : ~one;
    }
    before = __popcll(m & ((1ull << lane) - 1));
    all = __popcll(m);
}

// Each pair's rank among its block's pairs of the same expert, and the
// block's number of pairs of each expert. A wave takes a contiguous part of
// the block's pairs, 64 at a time, and counts them in its own row of LDS.
__global__ __launch_bounds__(64 * SORT_WAVES) void k_sort_rank(sort_p p) {
    extern __shared__ int cnt[];                  // [SORT_WAVES][E]
    constexpr int STEPS = SORT_PAIRS / SORT_WAVES / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < SORT_WAVES * p.E; i += 64 * SORT_WAVES) cnt[i] = 0;
    __syncthreads();
    int *mine = cnt + wave * p.E, key[STEPS], rank[STEPS];
    const int at = (int)blockIdx.x * SORT_PAIRS + wave * STEPS * 64 + lane;
#pragma unroll
    for (int i = 0; i < STEPS; i++) key[i] = at + 64 * i < p.pairs ? p.idx[at + 64 * i] : -1;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const bool in = (unsigned)key[i] < (unsigned)p.E;
        int before, all;
        same_key(key[i], p.bits, in, lane, before, all);
        const int had = in ? mine[key[i]] : 0;
        rank[i] = had + before;
        if (in && before == all - 1) mine[key[i]] = had + all;     // the last of them
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += 64 * SORT_WAVES) {
        int sum = 0;
        for (int w = 0; w < SORT_WAVES; w++) {
            const int c = cnt[w * p.E + e];
            cnt[w * p.E + e] = sum;
            sum += c;
        }
        p.count[(size_t)blockIdx.x * p.E + e] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < STEPS; i++)
        if ((unsigned)key[i] < (unsigned)p.E) p.rank[at + 64 * i] = rank[i] + mine[key[i]];
}

// Where each block's pairs of an expert begin: count becomes that.
__global__ __launch_bounds__(1024) void k_sort_scan(sort_p p) {
    __shared__ int wave_sum[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int base = 0;
    for (int e0 = 0; e0 < p.E; e0 += 1024) {
        const int e = e0 + (int)threadIdx.x;
        int n = 0;
        if (e < p.E) {
#pragma unroll 8
            for (int b = 0; b < p.blocks; b++) n += p.count[(size_t)b * p.E + e];
        }
        int s = n;                                // inclusive over the wave
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(s, d);
            if (lane >= d) s += o;
        }
        if (lane == 63) wave_sum[wave] = s;
        __syncthreads();
        int before = base, total = 0;
        for (int w = 0; w < 16; w++) {
            if (w < wave) before += wave_sum[w];
            total += wave_sum[w];
        }
        if (e < p.E) {
            const int first = before + s - n;
            p.offsets[e] = first;
            for (int b = 0, at = first; b < p.blocks; b += 8) {
                int c[8];
#pragma unroll
                for (int i = 0; i < 8; i++) c[i] = b + i < p.blocks ? p.count[(size_t)(b + i) * p.E + e] : 0;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (b + i < p.blocks) p.count[(size_t)(b + i) * p.E + e] = at;
                    at += c[i];
                }
            }
        }
        base += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) p.offsets[p.E] = base;
}

// The pairs' places, and the rows to them: a block takes 256 vectors of a
// token's row and writes it to the places of its pairs.
template <typename T>
__global__ __launch_bounds__(256) void k_sort_rows(sort_p p) {
    constexpr int V = rows_of<T>::V;
    const int c0 = ((int)blockIdx.x * 256 + (int)threadIdx.x) * V, n = min(V, p.hidden - c0);
    for (int t = blockIdx.y; t < p.tokens; t += gridDim.y) {
        vec_t<T, V> x;
        if (p.xs && n > 0) x = load_vec<T, V>((const T *)p.x + (size_t)t * p.ldx + c0, n);
        for (int k = 0; k < p.K; k++) {
            const int i = t * p.K + k, e = p.idx[i];
            const bool in = (unsigned)e < (unsigned)p.E;
            const int at = in ? p.count[(size_t)(i / SORT_PAIRS) * p.E + e] + p.rank[i] : -1;
            if (blockIdx.x == 0 && threadIdx.x == 0) {
                p.pos[i] = at;
                if (in) p.perm[at] = i;
            }
            if (in && p.xs && n > 0) store_vec<T, V>((T *)p.xs + (size_t)at * p.ldxs + c0, x, n);
        }
    }
}

extern "C" size_t wk_dispatch_work(int tokens, int K, int E) {
    const size_t n = (size_t)tokens * K;
    return (n + (n + SORT_PAIRS - 1) / SORT_PAIRS * E) * sizeof(int);
}

extern "C" int wk_expert_dispatch(const warp_hip_dispatch_args *a, void *stream) {
    const int pairs = a->tokens * a->top_k;
    sort_p p = {a->tokens, a->top_k, a->n_experts, pairs, (pairs + SORT_PAIRS - 1) / SORT_PAIRS, 1, a->idx, a->offsets,
                a->perm, a->pos, (int *)a->work, (int *)a->work + pairs, a->hidden, a->x, a->xs, a->ldx, a->ldxs};
    while ((p.E - 1) >> p.bits) p.bits++;
    hipStream_t st = (hipStream_t)stream;
    if (pairs)
        hipLaunchKernelGGL(k_sort_rank, dim3(p.blocks), dim3(64 * SORT_WAVES), SORT_WAVES * p.E * sizeof(int), st, p);
    hipLaunchKernelGGL(k_sort_scan, dim3(1), dim3(1024), 0, st, p);
    if (pairs) {
        const int V = a->type == WARP_HIP_F32 ? 4 : 8, cols = p.xs ? ((p.hidden + V - 1) / V + 255) / 256 : 1;
        const dim3 grid(cols, p.tokens < 32768 ? p.tokens : 32768);
        if (a->type == WARP_HIP_F32) hipLaunchKernelGGL((k_sort_rows<uint32_t>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((k_sort_rows<uint16_t>), grid, dim3(256), 0, st, p);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

struct comb_p {
    int tokens, K, hidden;
    const void *y;
    const int *pos;
    const float *w;
    const void *resid;
    void *out;
    const void *dout;
    void *dy;
    float *dw;
    size_t ldy, ldr, ldo, ldd, lddy;
};

// A thread adds one vector of a token's rows in the order of k, from the
// residual on, in f32.
template <typename T>
__global__ __launch_bounds__(256) void k_combine(comb_p p) {
    constexpr int V = rows_of<T>::V;
    const int c0 = ((int)blockIdx.x * (int)blockDim.x + (int)threadIdx.x) * V, n = min(V, p.hidden - c0);
    if (n <= 0) return;
    const int pairs = p.tokens * p.K;
    for (int t = blockIdx.y; t < p.tokens; t += gridDim.y) {
        float a[V];
        vec_t<T, V> r = load_vec<T, V>((const T *)p.resid + (size_t)t * p.ldr + c0, p.resid ? n : 0);
#pragma unroll
        for (int i = 0; i < V; i++) a[i] = (float)r.e[i];
        for (int k = 0; k < p.K; k++) {
            const int at = p.pos[t * p.K + k];
            if ((unsigned)at >= (unsigned)pairs) continue;
            const float w = p.w ? p.w[(size_t)t * p.K + k] : 1.0f;
            const vec_t<T, V> y = load_vec<T, V>((const T *)p.y + (size_t)at * p.ldy + c0, n);
#pragma unroll
            for (int i = 0; i < V; i++) a[i] = __builtin_fmaf(w, (float)y.e[i], a[i]);
        }
        vec_t<T, V> o;
#pragma unroll
        for (int i = 0; i < V; i++) o.e[i] = (T)a[i];
        store_vec<T, V>((T *)p.out + (size_t)t * p.ldo + c0, o, n);
    }
}

// A wave takes one pair: its row of dy, and the product of its row of y with
// the token's dout.
template <typename T>
__global__ __launch_bounds__(256) void k_combine_back(comb_p p) {
    constexpr int V = rows_of<T>::V;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int pairs = p.tokens * p.K;
    for (int i = (int)blockIdx.x * 4 + wave; i < pairs; i += (int)gridDim.x * 4) {
        const int at = p.pos[i];
        float sum = 0.0f;
        if ((unsigned)at < (unsigned)pairs) {
            const float w = p.w ? p.w[i] : 1.0f;
            const T *d = (const T *)p.dout + (size_t)(i / p.K) * p.ldd, *y = (const T *)p.y + (size_t)at * p.ldy;
            T *dy = (T *)p.dy + (size_t)at * p.lddy;
            for (int c = lane * V; c < p.hidden; c += 64 * V) {
                const int n = min(V, p.hidden - c);
                const vec_t<T, V> dv = load_vec<T, V>(d + c, n), yv = load_vec<T, V>(y + c, p.dw ? n : 0);
                vec_t<T, V> o;
#pragma unroll
                for (int e = 0; e < V; e++) {
                    sum = __builtin_fmaf((float)dv.e[e], (float)yv.e[e], sum);
                    o.e[e] = (T)(w * (float)dv.e[e]);
                }
                if (p.dy) store_vec<T, V>(dy + c, o, n);
            }
        }
        for (int m = 32; m; m >>= 1) sum += __shfl_xor(sum, m);
        if (p.dw && lane == 0) p.dw[i] = sum;
    }
}

extern "C" int wk_expert_combine(const warp_hip_combine_args *a, void *stream) {
    comb_p p = {a->tokens, a->top_k, a->hidden, a->y, a->pos, a->w, a->resid, a->out, nullptr, nullptr, nullptr,
                a->ldy, a->ldr, a->ldo, 0, 0};
    const int V = a->type == WARP_HIP_F32 ? 4 : 8, groups = (p.hidden + V - 1) / V;
    const dim3 grid((groups + 127) / 128, p.tokens < 32768 ? p.tokens : 32768), block(128);
    hipStream_t st = (hipStream_t)stream;
    if (a->type == WARP_HIP_F32) hipLaunchKernelGGL((k_combine<float>), grid, block, 0, st, p);
    else if (a->type == WARP_HIP_BF16) hipLaunchKernelGGL((k_combine<bf16_t>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((k_combine<f16_t>), grid, block, 0, st, p);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

extern "C" int wk_expert_combine_backward(const warp_hip_combine_back_args *a, void *stream) {
    comb_p p = {a->tokens, a->top_k, a->hidden, a->y, a->pos, a->w, nullptr, nullptr, a->dout, a->dy, a->dw,
                a->ldy, 0, 0, a->ldd, a->lddy};
    const int pairs = p.tokens * p.K, blocks = (pairs + 3) / 4;
    const dim3 grid(blocks < 65536 ? blocks : 65536);
    hipStream_t st = (hipStream_t)stream;
    if (a->type == WARP_HIP_F32) hipLaunchKernelGGL((k_combine_back<float>), grid, dim3(256), 0, st, p);
    else if (a->type == WARP_HIP_BF16) hipLaunchKernelGGL((k_combine_back<bf16_t>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_combine_back<f16_t>), grid, dim3(256), 0, st, p);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
