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

constexpr int SORT_WAVES = 8;

struct sort_p {
    int tokens, K, E, pairs, per, blocks, bits;   // per: pairs of a sorting block
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

// A block's pairs [at, at + STEPS 64 SORT_WAVES): each pair's rank among the
// block's earlier ones of its expert (without those of its wave's count row,
// cnt, which then holds where the wave's begin). A wave takes a contiguous
// part of them, 64 at a time, and counts them in its own row of LDS, so that
// the order is the pairs' own and no two waves meet at a counter.
template <int STEPS>
__device__ __forceinline__ void sort_rank(const sort_p &p, int first, uint16_t *cnt, int (&key)[STEPS], int (&rank)[STEPS]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < SORT_WAVES * p.E; i += 64 * SORT_WAVES) cnt[i] = 0;
    uint16_t *mine = cnt + wave * p.E;
    const int at = first + wave * STEPS * 64 + lane;
#pragma unroll
    for (int i = 0; i < STEPS; i++) key[i] = at + 64 * i < p.pairs ? p.idx[at + 64 * i] : -1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const bool in = (unsigned)key[i] < (unsigned)p.E;
        int before, all;
        same_key(key[i], p.bits, in, lane, before, all);
        const int had = in ? mine[key[i]] : 0;
        rank[i] = had + before;
        if (in && before == all - 1) mine[key[i]] = (uint16_t)(had + all);       // the last of them
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
}
// The waves' counts of expert e become where each wave's begin; their sum.
__device__ __forceinline__ int sort_waves(const sort_p &p, uint16_t *cnt, int e) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; w++) {
        const int c = cnt[w * p.E + e];
        cnt[w * p.E + e] = (uint16_t)sum;
        sum += c;
    }
    return sum;
}
// What lies before this thread's n, over the block's threads in order, and
// the sum of all (with room for a number per wave; all threads take part).
__device__ __forceinline__ int sort_before(int n, int *wave_sum, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int s = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(s, d);
        if (lane >= d) s += o;
    }
    __syncthreads();
    if (lane == 63) wave_sum[wave] = s;
    __syncthreads();
    int before = s - n;
    total = 0;
    for (int w = 0; w < waves; w++) {
        if (w < wave) before += wave_sum[w];
        total += wave_sum[w];
    }
    return before;
}

// Each pair's rank among its block's, and the block's pairs of each expert.
template <int STEPS>
__global__ __launch_bounds__(64 * SORT_WAVES) void k_sort_rank(sort_p p) {
    extern __shared__ uint16_t cnt[];             // [SORT_WAVES][E]
    int key[STEPS], rank[STEPS];
    const int first = (int)blockIdx.x * p.per;
    sort_rank<STEPS>(p, first, cnt, key, rank);
    for (int e = threadIdx.x; e < p.E; e += 64 * SORT_WAVES) p.count[(size_t)blockIdx.x * p.E + e] = sort_waves(p, cnt, e);
    __syncthreads();
    const int wave = threadIdx.x >> 6, at = first + wave * STEPS * 64 + (threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < STEPS; i++)
        if ((unsigned)key[i] < (unsigned)p.E) p.rank[at + 64 * i] = rank[i] + cnt[wave * p.E + key[i]];
}

// Where each block's pairs of an expert begin: count becomes that.
__global__ __launch_bounds__(1024) void k_sort_scan(sort_p p) {
    __shared__ int wave_sum[16];
    int base = 0;
    for (int e0 = 0; e0 < p.E; e0 += 1024) {
        const int e = e0 + (int)threadIdx.x;
        int n = 0, total;
        if (e < p.E) {
#pragma unroll 8
            for (int b = 0; b < p.blocks; b++) n += p.count[(size_t)b * p.E + e];
        }
        const int first = base + sort_before(n, wave_sum, total);
        if (e < p.E) {
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
    }
    if (threadIdx.x == 0) p.offsets[p.E] = base;
}

// 4,096 tokens of 2,304 bf16 to 8 of 256 experts: 31 us for the rows, 5.4 TB/s,
// behind 9 for ranks and scan (with four vectors a lane 32.4); with a block to
// 256 vectors of a row, the places read pair by pair and stores through L2 48.6.
// A part of a token's row, IT vectors a lane of a wave, and its copies to the
// places of the token's pairs: at(i) is the place of pair i, a lane's each.
template <typename T, bool ONE, int IT>
struct sort_part {
    static constexpr int V = rows_of<T>::V;
    vec_t<T, V> v[IT];

    __device__ __forceinline__ void load(const sort_p &p, int t, int part) {
        const T *x = (const T *)p.x + (size_t)t * p.ldx;
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int c0 = ((part * IT + i) * 64 + (threadIdx.x & 63)) * V;
            if (c0 < p.hidden) {
                const cols_t<T, ONE> k(c0, p.hidden);
                v[i] = k.load(x + k.c);
            }
        }
    }
    template <typename AT>
    __device__ __forceinline__ void copy(const sort_p &p, int t, int part, AT at) const {
        const int lane = threadIdx.x & 63;
        for (int k0 = 0; k0 < p.K; k0 += 64) {
            const int mine = k0 + lane < p.K ? at(t * p.K + k0 + lane) : -1;
            for (int k = 0; k < min(64, p.K - k0); k++) {
                const int to = __builtin_amdgcn_readlane(mine, k);
                if (to < 0) continue;
                T *row = (T *)p.xs + (size_t)to * p.ldxs;
#pragma unroll
                for (int i = 0; i < IT; i++) {
                    const int c0 = ((part * IT + i) * 64 + lane) * V;
                    if (c0 < p.hidden) {
                        const cols_t<T, ONE> c(c0, p.hidden);
                        c.stream(row + c.c, v[i]);
                    }
                }
            }
        }
    }
};

// The pairs' places, and the rows to them.
template <typename T, bool ONE, int IT>
__global__ __launch_bounds__(256) void k_sort_rows(sort_p p, int parts) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t items = (int64_t)p.tokens * parts;
    for (int64_t q = (int64_t)blockIdx.x * 4 + wave; q < items; q += (int64_t)gridDim.x * 4) {
        const int t = (int)(q / parts), part = (int)(q % parts);
        auto place = [&](int i) {
            const int e = p.idx[i];
            return (unsigned)e < (unsigned)p.E ? p.count[(size_t)(i / p.per) * p.E + e] + p.rank[i] : -1;
        };
        if (part == 0)
            for (int k = lane; k < p.K; k += 64) {
                const int i = t * p.K + k, at = place(i);
                p.pos[i] = at;
                if (at >= 0) p.perm[at] = i;
            }
        if (p.xs) {
            sort_part<T, ONE, IT> x;
            x.load(p, t, part);
            x.copy(p, t, part, place);
        }
    }
}

// All of it at once where a block can sort all pairs: every block does, into
// LDS, and copies its share of the rows (the first also writes the lists).
// Three launches take 15 us for 32 tokens of 7,168 bf16 to 16 of 384 experts,
// this one 6.9; 500 tokens of 1,012 to 8 of 239 11.2, 520 in three launches 14.4
// and the gaps between them.
constexpr int SMALL_PAIRS = 4096;
template <typename T, bool ONE, int STEPS>
__global__ __launch_bounds__(64 * SORT_WAVES) void k_sort_small(sort_p p, int parts) {
    extern __shared__ int lds[];                  // [pairs] places, [E] beginnings, [SORT_WAVES][E] counts
    __shared__ int wave_sum[SORT_WAVES];
    int *place = lds, *begin = lds + p.pairs;
    uint16_t *cnt = (uint16_t *)(begin + p.E);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int items = p.xs ? p.tokens * parts : 0, q0 = (int)blockIdx.x * SORT_WAVES + wave;
    sort_part<T, ONE, 1> x;
    if (q0 < items) x.load(p, q0 / parts, q0 % parts);
    int key[STEPS], rank[STEPS], base = 0;
    sort_rank<STEPS>(p, 0, cnt, key, rank);
    for (int e0 = 0; e0 < p.E; e0 += 64 * SORT_WAVES) {
        const int e = e0 + (int)threadIdx.x;
        int total;
        const int first = base + sort_before(e < p.E ? sort_waves(p, cnt, e) : 0, wave_sum, total);
        if (e < p.E) {
            begin[e] = first;
            if (blockIdx.x == 0) p.offsets[e] = first;
        }
        base += total;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.offsets[p.E] = base;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const int pair = (wave * STEPS + i) * 64 + lane;
        if (pair >= p.pairs) continue;
        const int at = (unsigned)key[i] < (unsigned)p.E ? begin[key[i]] + cnt[wave * p.E + key[i]] + rank[i] : -1;
        place[pair] = at;
        if (blockIdx.x == 0) {
            p.pos[pair] = at;
            if (at >= 0) p.perm[at] = pair;
        }
    }
    __syncthreads();
    for (int q = q0; q < items; q += (int)gridDim.x * SORT_WAVES) {
        if (q != q0) x.load(p, q / parts, q % parts);
        x.copy(p, q / parts, q % parts, [&](int i) { return place[i]; });
    }
}

// Sorting blocks of 1,024 pairs until there are 64 of them, then larger ones:
// the scan goes through every block's counts.
static int sort_per(int64_t pairs) {
    return pairs <= 64 * 1024 ? 1024 : 4096;
}
extern "C" size_t wk_dispatch_work(int tokens, int K, int E) {
    const int64_t n = (int64_t)tokens * K, per = sort_per(n);
    return n <= SMALL_PAIRS ? 0 : (size_t)(n + (n + per - 1) / per * E) * sizeof(int);
}

template <typename T, bool ONE>
static void dispatch_launch(sort_p p, hipStream_t st) {
    const int vecs = (p.hidden + rows_of<T>::V - 1) / rows_of<T>::V;
    if (p.pairs <= SMALL_PAIRS) {
        const int parts = (vecs + 63) / 64, blocks = p.xs ? (p.tokens * parts + SORT_WAVES - 1) / SORT_WAVES : 1;
        const dim3 grid(blocks < 1 ? 1 : blocks < 256 ? blocks : 256);
        const size_t lds = (p.pairs + p.E) * sizeof(int) + SORT_WAVES * p.E * sizeof(uint16_t);
        constexpr int step = 64 * SORT_WAVES;
        if (p.pairs <= step) hipLaunchKernelGGL((k_sort_small<T, ONE, 1>), grid, dim3(step), lds, st, p, parts);
        else if (p.pairs <= 4 * step) hipLaunchKernelGGL((k_sort_small<T, ONE, 4>), grid, dim3(step), lds, st, p, parts);
        else hipLaunchKernelGGL((k_sort_small<T, ONE, SMALL_PAIRS / step>), grid, dim3(step), lds, st, p, parts);
        return;
    }
    const size_t lds = SORT_WAVES * p.E * sizeof(uint16_t);
    if (p.per == 1024) hipLaunchKernelGGL((k_sort_rank<2>), dim3(p.blocks), dim3(64 * SORT_WAVES), lds, st, p);
    else hipLaunchKernelGGL((k_sort_rank<8>), dim3(p.blocks), dim3(64 * SORT_WAVES), lds, st, p);
    hipLaunchKernelGGL(k_sort_scan, dim3(1), dim3(1024), 0, st, p);
    const int parts = p.xs ? (vecs + 127) / 128 : 1;
    const int64_t blocks = ((int64_t)p.tokens * parts + 3) / 4;
    hipLaunchKernelGGL((k_sort_rows<T, ONE, 2>), dim3(blocks < 65536 ? blocks : 65536), dim3(256), 0, st, p, parts);
}

extern "C" int wk_expert_dispatch(const warp_hip_dispatch_args *a, void *stream) {
    const int pairs = a->tokens * a->top_k, per = sort_per(pairs);
    sort_p p = {a->tokens, a->top_k, a->n_experts, pairs, per, (int)(((int64_t)pairs + per - 1) / per), 1, a->idx, a->offsets,
                a->perm, a->pos, (int *)a->work, (int *)a->work + pairs, a->x ? a->hidden : 0, a->x, a->xs, a->ldx, a->ldxs};
    while ((p.E - 1) >> p.bits) p.bits++;
    hipStream_t st = (hipStream_t)stream;
    // (rows are copied as bits)
    if (a->type == WARP_HIP_F32) {
        if (p.hidden < 4) dispatch_launch<uint32_t, true>(p, st);
        else dispatch_launch<uint32_t, false>(p, st);
    } else {
        if (p.hidden < 8) dispatch_launch<uint16_t, true>(p, st);
        else dispatch_launch<uint16_t, false>(p, st);
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

// A wave adds 64 vectors of a token's rows in the order of k, from the
// residual on, in f32. The rows of eight pairs are loaded at once (row 0 in
// place of one that is not there, which is then not added). 4,096 tokens of
// 7,168 bf16, 16 rows each: 171 us, 5.8 TB/s; 190 us with loads that stay in
// the caches, 200 row by row.
template <typename T, bool ONE>
__global__ __launch_bounds__(256) void k_combine(comb_p p, int parts) {
    constexpr int V = rows_of<T>::V, KB = 8;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int pairs = p.tokens * p.K;
    const int64_t items = (int64_t)p.tokens * parts;
    for (int64_t q = (int64_t)blockIdx.x * 4 + wave; q < items; q += (int64_t)gridDim.x * 4) {
        const int t = (int)(q / parts), c0 = ((int)(q % parts) * 64 + lane) * V;
        const bool live = c0 < p.hidden;
        const cols_t<T, ONE> c(live ? c0 : p.hidden - 1, p.hidden);
        float a[V];
#pragma unroll
        for (int i = 0; i < V; i++) a[i] = 0.0f;
        if (p.resid && live) {
            const vec_t<T, V> r = c.load((const T *)p.resid + (size_t)t * p.ldr + c.c);
#pragma unroll
            for (int i = 0; i < V; i++) a[i] = (float)r.e[i];
        }
        for (int k0 = 0; k0 < p.K; k0 += 64) {
            const int i = t * p.K + k0 + lane, m = min(64, p.K - k0);
            const int at = lane < m ? p.pos[i] : -1;
            const float w = lane < m && p.w ? p.w[i] : 1.0f;
            for (int k = 0; k < m; k += KB) {
                vec_t<T, V> y[KB];
#pragma unroll
                for (int j = 0; j < KB; j++) {
                    const int r = __builtin_amdgcn_readlane(at, k + j);
                    if (live && k + j < m) y[j] = c.take((const T *)p.y + (size_t)((unsigned)r < (unsigned)pairs ? r : 0) * p.ldy + c.c);
                }
#pragma unroll
                for (int j = 0; j < KB; j++) {
                    if (k + j >= m || (unsigned)__builtin_amdgcn_readlane(at, k + j) >= (unsigned)pairs) continue;
                    const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), k + j));
#pragma unroll
                    for (int e = 0; e < V; e++) a[e] = __builtin_fmaf(f, (float)y[j].e[e], a[e]);
                }
            }
        }
        if (live) {
            vec_t<T, V> o;
#pragma unroll
            for (int i = 0; i < V; i++) o.e[i] = (T)a[i];
            c.store((T *)p.out + (size_t)t * p.ldo + c.c, o);
        }
    }
}

// W waves take a pair: its row of dy, and the product of its row of y with
// the token's dout (which the token's other pairs find in the caches). Many
// short waves beat fewer that hold more: with two or four pairs to a wave the
// 117 us below are 133 and 137. 8,192 tokens of 2,304 bf16, 8 rows each: 117
// us, 5.5 TB/s. Few pairs get four waves each: 10 tokens of 2,304 f32, 8 rows
// each, take 8.4 us with one and 4.1 with four; 8,192 as above 118 and 153.
template <typename T, bool ONE, int W>
__global__ __launch_bounds__(256) void k_combine_back(comb_p p) {
    constexpr int V = rows_of<T>::V, CU = 4;               // vectors a lane loads at once
    __shared__ float part[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int pairs = p.tokens * p.K, own = wave % W;
    for (int64_t i = (int64_t)blockIdx.x * (4 / W) + wave / W; i < pairs; i += (int64_t)gridDim.x * (4 / W)) {
        const int at = p.pos[i];
        float sum = 0.0f;
        if ((unsigned)at < (unsigned)pairs) {
            const float w = p.w ? p.w[i] : 1.0f;
            const T *d = (const T *)p.dout + (size_t)((int)i / p.K) * p.ldd, *y = (const T *)p.y + (size_t)at * p.ldy;
            T *dy = (T *)p.dy + (size_t)at * p.lddy;
            for (int c0 = (own * 64 + lane) * V; c0 < p.hidden; c0 += CU * W * 64 * V) {
                vec_t<T, V> dv[CU], yv[CU];
#pragma unroll
                for (int u = 0; u < CU; u++)
                    if (c0 + u * W * 64 * V < p.hidden) {
                        const cols_t<T, ONE> c(c0 + u * W * 64 * V, p.hidden);
                        dv[u] = c.load(d + c.c);
                        if (p.dw) yv[u] = c.take(y + c.c);
                    }
#pragma unroll
                for (int u = 0; u < CU; u++)
                    if (c0 + u * W * 64 * V < p.hidden) {
                        const cols_t<T, ONE> c(c0 + u * W * 64 * V, p.hidden);
                        vec_t<T, V> o;
#pragma unroll
                        for (int e = 0; e < V; e++) {
                            if (p.dw && e >= c.skip) sum = __builtin_fmaf((float)dv[u].e[e], (float)yv[u].e[e], sum);
                            o.e[e] = (T)(w * (float)dv[u].e[e]);
                        }
                        if (p.dy) c.stream(dy + c.c, o);
                    }
            }
        }
        if (!p.dw) continue;
#pragma unroll
        for (int m = 32; m; m >>= 1) sum += __shfl_xor(sum, m);
        if (W > 1) {
            if (lane == 0) part[wave] = sum;
            __syncthreads();
            sum = (part[0] + part[1]) + (part[2] + part[3]);
            __syncthreads();
        }
        if (lane == 0 && own == 0) p.dw[i] = sum;
    }
}

template <typename T>
static void combine_launch(const comb_p &p, hipStream_t st) {
    constexpr int V = rows_of<T>::V;
    const int parts = ((p.hidden + V - 1) / V + 63) / 64;
    const int64_t blocks = ((int64_t)p.tokens * parts + 3) / 4;
    const dim3 grid(blocks < 65536 ? blocks : 65536);
    if (p.hidden < V) hipLaunchKernelGGL((k_combine<T, true>), grid, dim3(256), 0, st, p, parts);
    else hipLaunchKernelGGL((k_combine<T, false>), grid, dim3(256), 0, st, p, parts);
}
template <typename T, bool ONE>
static void combine_back_launch(const comb_p &p, hipStream_t st) {
    // (four waves where one to each pair leaves SIMDs without any)
    const int64_t pairs = (int64_t)p.tokens * p.K;
    const int W = pairs < 4096 && p.hidden > 64 * rows_of<T>::V ? 4 : 1;
    const int64_t blocks = (pairs * W + 3) / 4;
    const dim3 grid(blocks < 65536 ? blocks : 65536);
    if (W == 4) hipLaunchKernelGGL((k_combine_back<T, ONE, 4>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_combine_back<T, ONE, 1>), grid, dim3(256), 0, st, p);
}
template <typename T>
static void combine_back_type(const comb_p &p, hipStream_t st) {
    if (p.hidden < rows_of<T>::V) combine_back_launch<T, true>(p, st);
    else combine_back_launch<T, false>(p, st);
}

extern "C" int wk_expert_combine(const warp_hip_combine_args *a, void *stream) {
    const comb_p p = {a->tokens, a->top_k, a->hidden, a->y, a->pos, a->w, a->resid, a->out, nullptr, nullptr, nullptr,
                      a->ldy, a->ldr, a->ldo, 0, 0};
    if (a->type == WARP_HIP_F32) combine_launch<float>(p, (hipStream_t)stream);
    else if (a->type == WARP_HIP_BF16) combine_launch<bf16_t>(p, (hipStream_t)stream);
    else combine_launch<f16_t>(p, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

extern "C" int wk_expert_combine_backward(const warp_hip_combine_back_args *a, void *stream) {
    const comb_p p = {a->tokens, a->top_k, a->hidden, a->y, a->pos, a->w, nullptr, nullptr, a->dout, a->dy, a->dw,
                      a->ldy, 0, 0, a->ldd, a->lddy};
    if (a->type == WARP_HIP_F32) combine_back_type<float>(p, (hipStream_t)stream);
    else if (a->type == WARP_HIP_BF16) combine_back_type<bf16_t>(p, (hipStream_t)stream);
    else combine_back_type<f16_t>(p, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
