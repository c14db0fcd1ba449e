// scan.hip — the selective state space scan (warp_hip_selective_scan). Per
// channel d with states n, row by row of a sequence:
//   dt' = softplus(dt + dt_bias)                        (or dt + dt_bias)
//   h[n] = exp(dt' A[d][n]) h[n] + dt' x B[n]
//   y    = (sum_n C[n] h[n] + D x) silu(z)
// with B and C shared by the channels of a group. The states are f32 from end
// to end, dt' and the sums too; only x, dt, B, C, z and y are of the rows' type.
//
// What bounds prompts is the vector units: per row, channel and state a
// product and an exponential for the decay (the exponential issues at a
// quarter of the rate), a product, and two fused multiply-adds, about eight
// issue slots, against 8 bytes of rows per channel. The decays differ by
// channel and state, so nothing of this is a matrix product. Single tokens
// are bound by their states, read and written once.

#include "rows.h"
#include "warp_internal.h"

struct scan_p {
    int tokens, n_seq, D, N, G, n_slots, softplus, chunk, chunks;
    const int *starts, *slots;
    const void *x, *dt, *B, *C, *z;
    size_t ldx, lddt, ldbc, ldz, ldy;
    const float *A, *skip, *bias, *sin;
    float *sout;
    void *y;
    float *end, *sum, *init;                      // per chunk: [D][N], [D], [D][N]
    int *reset;
};

constexpr float LOG2E = 1.44269504088896341f;

// log(1 + e^v) = max(v, 0) + log(1 + e), e = exp(-|v|) <= 1, and log(1 + e) =
// 2 atanh(s) with s = e / (2 + e) <= 1/3: the series to s^13 (the next term is
// below 2^-27 of the sum). Small results keep their digits, as the time steps
// of slow channels need them.
__device__ __forceinline__ float scan_softplus(float v) {
    const float e = rows_exp(-__builtin_fabsf(v)), s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
    float r = 1.0f / 13;
    r = __builtin_fmaf(r, q, 1.0f / 11);
    r = __builtin_fmaf(r, q, 1.0f / 9);
    r = __builtin_fmaf(r, q, 1.0f / 7);
    r = __builtin_fmaf(r, q, 1.0f / 5);
    r = __builtin_fmaf(r, q, 1.0f / 3);
    return __builtin_fmaf(2.0f * s, __builtin_fmaf(r, q, 1.0f), __builtin_fmaxf(v, 0.0f));
}

// The sum over the LPC lanes of a channel, in each of them.
template <int LPC>
__device__ __forceinline__ float scan_sum(float v) {
    if (LPC > 1) v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xb1, 0xf, 0xf, true));   // lane ^ 1
    if (LPC > 2) v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4e, 0xf, 0xf, true));   // lane ^ 2
    if (LPC > 4) v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xf, 0xf, true));  // 7 - lane
    if (LPC > 8) v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xf, 0xf, true));  // 15 - lane
    if (LPC > 16) v += __shfl_xor(v, 16);
    if (LPC > 32) v += __shfl_xor(v, 32);
    return v;
}

// One token of each of n_seq sequences. LPC lanes share a channel, W states
// each in a run (their state row is read and written 4 W bytes a lane), and
// keep that channel's decay rates for the rows of sequences they take in turn.
template <typename T, int W, int LPC>
__global__ __launch_bounds__(256) void k_scan_token(scan_p p) {
    constexpr int NI = W == 1 && LPC == 64 ? 4 : 1;        // (64 lanes of single states take them in up to four turns)
    const int lane = threadIdx.x % LPC, d = ((int)blockIdx.x * 256 + (int)threadIdx.x) / LPC;
    if (d >= p.D) return;
    const int n0 = lane * W, g = d / (p.D / p.G);
    float A[NI][W];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int n = n0 + i * LPC * W;
        const vec_t<float, W> a = load_vec<float, W>(p.A + (size_t)d * p.N + n, p.N - n);
#pragma unroll
        for (int j = 0; j < W; j++) A[i][j] = a.e[j] * LOG2E;
    }
    const float bias = p.bias ? p.bias[d] : 0.0f, skip = p.skip ? p.skip[d] : 0.0f;
    for (int s = blockIdx.y; s < p.n_seq; s += gridDim.y) {
        const int slot = seq_slot(p.slots, s, p.n_slots);
        if (slot < 0) continue;
        const float x = (float)((const T *)p.x)[(size_t)s * p.ldx + d];
        float dt = (float)((const T *)p.dt)[(size_t)s * p.lddt + d] + bias;
        if (p.softplus) dt = scan_softplus(dt);
        const size_t at = ((size_t)slot * p.D + d) * p.N, bc = (size_t)s * p.ldbc + (size_t)g * p.N;
        const float u = dt * x;
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int n = n0 + i * LPC * W, m = p.N - n;
            const vec_t<T, W> B = load_vec<T, W>((const T *)p.B + bc + n, m), C = load_vec<T, W>((const T *)p.C + bc + n, m);
            vec_t<float, W> h = load_vec<float, W>(p.sin + at + n, p.sin ? m : 0);
#pragma unroll
            for (int j = 0; j < W; j++) {
                h.e[j] = __builtin_fmaf(h.e[j], __builtin_amdgcn_exp2f(dt * A[i][j]), u * (float)B.e[j]);
                y = __builtin_fmaf(h.e[j], j < m ? (float)C.e[j] : 0.0f, y);
            }
            if (p.sout) store_vec<float, W>(p.sout + at + n, h, m);
        }
        y = scan_sum<LPC>(y);
        y = __builtin_fmaf(skip, x, y);
        if (p.z) y *= rows_silu((float)((const T *)p.z)[(size_t)s * p.ldz + d]);
        if (lane == 0) ((T *)p.y)[(size_t)s * p.ldy + d] = (T)y;
    }
}

// Prompts. LPC lanes of a wave share a channel, S states each in registers;
// a wave is a block and takes 64 / LPC channels of one group. A batch of U
// rows' B and C is laid out in LDS as f32, where all lanes read the same
// address; x, dt and z go to registers a batch ahead.
template <typename T, int S, int LPC, int U>
struct scan_t {
    static constexpr int RS = S * LPC;                     // states, filled up
    float A[S], h[S], bias, skip;
    int lane, part, d, g;
    bool live;

    __device__ __forceinline__ void open(const scan_p &p) {
        const int per = p.D / p.G, blocks = (per * LPC + 63) / 64, i = (int)blockIdx.x % blocks;
        lane = threadIdx.x;
        part = lane % LPC;
        g = (int)blockIdx.x / blocks;
        const int c = (i * 64 + lane) / LPC;
        live = c < per;
        d = g * per + min(c, per - 1);                     // (a wave's spare lanes repeat the last channel)
#pragma unroll
        for (int n = 0; n < S; n++) A[n] = part * S + n < p.N ? p.A[(size_t)d * p.N + part * S + n] * LOG2E : 0.0f;
        bias = p.bias ? p.bias[d] : 0.0f;
        skip = p.skip ? p.skip[d] : 0.0f;
    }
    __device__ __forceinline__ void state(const scan_p &p, const float *at) {
#pragma unroll
        for (int n = 0; n < S; n++)
            h[n] = at && part * S + n < p.N ? at[(size_t)d * p.N + part * S + n] : 0.0f;
    }
    __device__ __forceinline__ void store(const scan_p &p, float *at) const {
#pragma unroll
        for (int n = 0; n < S; n++)
            if (live && part * S + n < p.N) at[(size_t)d * p.N + part * S + n] = h[n];
    }

    // Rows lo .. hi of one sequence. OUT: with y; without, dt' is summed up.
    template <bool OUT>
    __device__ __forceinline__ float rows(const scan_p &p, int lo, int hi, float *bc) {
        constexpr int K = OUT ? 2 : 1;                     // B, or B and C
        constexpr int M = (U * K * RS + 63) / 64;
        if (lo >= hi) return 0.0f;
        float tx[U], td[U], tz[U], tb[M], sum = 0.0f;
        const T *x = (const T *)p.x + d, *dt = (const T *)p.dt + d, *z = (const T *)p.z + d;
        const T *B = (const T *)p.B + (size_t)g * p.N, *C = (const T *)p.C + (size_t)g * p.N;
        auto load = [&](int t) {
#pragma unroll
            for (int i = 0; i < U; i++) {
                const size_t r = min(t + i, hi - 1);
                tx[i] = (float)x[r * p.ldx];
                td[i] = (float)dt[r * p.lddt];
                if (OUT && p.z) tz[i] = (float)z[r * p.ldz];
            }
#pragma unroll
            for (int i = 0; i < M; i++) {
                const int e = lane + 64 * i, n = e % RS, k = e / RS % K;
                const size_t r = min(t + e / (RS * K), hi - 1);
                tb[i] = n < p.N ? (float)(k ? C : B)[r * p.ldbc + n] : 0.0f;
            }
        };
        load(lo);
        for (int t = lo; t < hi; t += U) {
            float cx[U], cd[U], cz[U];
#pragma unroll
            for (int i = 0; i < U; i++) cx[i] = tx[i], cd[i] = td[i], cz[i] = tz[i];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < M; i++)
                if (U * K * RS % 64 == 0 || lane + 64 * i < U * K * RS) bc[lane + 64 * i] = tb[i];
            __syncthreads();                               // (one wave: its LDS writes are done)
            if (t + U < hi) load(t + U);
#pragma unroll
            for (int i = 0; i < U; i++) {
                if (t + i >= hi) break;
                float v = cd[i] + bias;
                if (p.softplus) v = scan_softplus(v);
                const float u = v * cx[i];
                const float *b = bc + i * K * RS + part * S, *c = b + RS;
                float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int n = 0; n < S; n++) {
                    h[n] = __builtin_fmaf(h[n], __builtin_amdgcn_exp2f(v * A[n]), u * b[n]);
                    if (OUT) y[n & 3] = __builtin_fmaf(h[n], c[n], y[n & 3]);
                }
                if (OUT) {
                    float o = scan_sum<LPC>((y[0] + y[1]) + (y[2] + y[3]));
                    o = __builtin_fmaf(skip, cx[i], o);
                    if (p.z) o *= rows_silu(cz[i]);
                    if (live && part == 0) ((T *)p.y)[(size_t)(t + i) * p.ldy + d] = (T)o;
                } else {
                    sum += v;
                }
            }
            __syncthreads();                               // the batch's rows are read
        }
        return sum;
    }
};

// A whole sequence per wave (chunk = 0), or the rows [j chunk, (j + 1) chunk)
// of the packed batch, whatever sequences they hold, from the state that
// k_scan_join found at their beginning.
template <typename T, int S, int LPC, int U>
__global__ __launch_bounds__(64) void k_scan_rows(scan_p p) {
    __shared__ __attribute__((aligned(16))) float bc[U * 2 * S * LPC];
    scan_t<T, S, LPC, U> k;
    k.open(p);
    const size_t dn = (size_t)p.D * p.N;
    const int units = p.chunk ? p.chunks : p.n_seq;
    const seqs_t seqs(p.starts, p.slots, p.n_seq, p.tokens, p.n_slots);
    for (int j = blockIdx.y; j < units; j += gridDim.y) {
        const int r0 = j * p.chunk, r1 = p.chunk ? min(r0 + p.chunk, p.tokens) : p.tokens;
        for (int s = p.chunk ? seqs.from(r0) : j; s < p.n_seq; s++) {
            const seq_t q = seqs.at(s);
            if (p.chunk && q.b >= r1 && j + 1 < units) break;
            if (q.slot >= 0 && (q.b >= r0 || q.e > r0)) {
                // (a sequence that goes on past its chunk has its first state
                // in `init`: its last state may be in the same slot already)
                const bool past = p.chunk && q.e > r1;
                const float *from = q.b < r0 ? p.end + (size_t)(j - 1) * dn
                                    : !p.sin ? nullptr
                                    : past   ? p.init + (size_t)j * dn
                                             : p.sin + (size_t)q.slot * dn;
                k.state(p, from);
                k.template rows<true>(p, max(q.b, r0), min(q.e, r1), bc);
                if (!past && p.sout) k.store(p, p.sout + (size_t)q.slot * dn);
            }
            if (!p.chunk) break;
        }
    }
}

// What a chunk's last sequence has at the chunk's end, from a state of zero
// (or the sequence's first state, if it begins here: then `reset` says that
// nothing before counts), and the sum of its dt', of which the chunk's decay
// is the exponential. Only for a sequence that goes on in the next chunk.
template <typename T, int S, int LPC, int U>
__global__ __launch_bounds__(64) void k_scan_part(scan_p p) {
    __shared__ __attribute__((aligned(16))) float bc[U * S * LPC];
    scan_t<T, S, LPC, U> k;
    k.open(p);
    const size_t dn = (size_t)p.D * p.N;
    const seqs_t seqs(p.starts, p.slots, p.n_seq, p.tokens, p.n_slots);
    for (int j = blockIdx.y; j + 1 < p.chunks; j += gridDim.y) {
        const int r0 = j * p.chunk, r1 = r0 + p.chunk;
        // the sequence that row r1 belongs to, if it holds row r1 - 1 too
        const int s = seqs.from(r1 + 1);
        const seq_t q = s < p.n_seq ? seqs.at(s) : seq_t{r1, r1, -1};
        if (q.slot < 0 || q.b >= r1) continue;
        const bool begins = q.b >= r0;
        const float *from = begins && p.sin ? p.sin + (size_t)q.slot * dn : nullptr;
        k.state(p, from);
        if (from) k.store(p, p.init + (size_t)j * dn);
        const float sum = k.template rows<false>(p, max(q.b, r0), r1, bc);
        k.store(p, p.end + (size_t)j * dn);
        if (k.live && k.part == 0) p.sum[(size_t)j * p.D + k.d] = sum;
        if (blockIdx.x == 0 && k.lane == 0) p.reset[j] = begins;
    }
}

// The chunks in order: end[j] becomes the state at the end of chunk j.
__global__ __launch_bounds__(256) void k_scan_join(scan_p p) {
    const size_t dn = (size_t)p.D * p.N, i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= dn) return;
    const int d = (int)(i / p.N);
    const float A = p.A[i] * LOG2E;
    float h = 0.0f;
    for (int j = 0; j + 1 < p.chunks; j++) {
        const float e = p.end[(size_t)j * dn + i], s = p.sum[(size_t)j * p.D + d];
        h = p.reset[j] ? e : __builtin_fmaf(h, __builtin_amdgcn_exp2f(A * s), e);
        p.end[(size_t)j * dn + i] = h;
    }
}

// The split of a packed batch of prompts: chunk = 0, a wave (per 64 / LPC
// channels) for each sequence, or chunks of so many rows.
// A wave's rows come one after the other, so that a batch is fast when its
// longest sequence is short, or there are more waves than the 1,024 SIMDs hold
// anyway. Chunks make waves at the price of computing the states twice.
struct scan_plan {
    int lanes, chunk, chunks;
};
static scan_plan scan_split(int tokens, int D, int N, int n_seq, int longest) {
    scan_plan r = {1, 0, 0};
    while (r.lanes * 16 < N) r.lanes *= 2;
    const double simds = 1024, waves = ((double)D * r.lanes + 63) / 64, states = N < 16 ? N : 16;
    const double all = 8 * states + 45, part = 7 * states + 30;      // issue slots of a row
    if (longest <= 0 || longest > tokens) longest = tokens;
    double most = 2 * simds / waves;
    if (most > tokens / 32) most = tokens / 32;
    if (most < 2) return r;
    const int chunk = ((int)(tokens / most) + 7) / 8 * 8, chunks = (tokens + chunk - 1) / chunk;
    const double direct = all * (longest > tokens * waves / simds ? longest : tokens * waves / simds);
    const double split = (all + part) * (chunk > tokens * waves / simds ? chunk : tokens * waves / simds) + 4000;
    if (chunks >= 2 && split < direct) r.chunk = chunk, r.chunks = chunks;
    return r;
}
static size_t scan_floats(const scan_plan &s, int D, int N) {
    return s.chunk ? (size_t)s.chunks * (2 * (size_t)D * N + D + 1) : 0;
}

template <typename T, int S, int LPC, int U>
static void scan_rows_launch(const scan_p &p, hipStream_t st) {
    const int blocks = p.G * ((p.D / p.G * LPC + 63) / 64);
    auto rows = [](int n) { return (unsigned)(n < 32768 ? n : 32768); };
    if (p.chunk) {
        hipLaunchKernelGGL((k_scan_part<T, S, LPC, U>), dim3(blocks, rows(p.chunks - 1)), dim3(64), 0, st, p);
        hipLaunchKernelGGL(k_scan_join, dim3((unsigned)(((size_t)p.D * p.N + 255) / 256)), dim3(256), 0, st, p);
    }
    hipLaunchKernelGGL((k_scan_rows<T, S, LPC, U>), dim3(blocks, rows(p.chunk ? p.chunks : p.n_seq)), dim3(64), 0, st, p);
}
template <typename T, int W, int LPC>
static void scan_token_launch(const scan_p &p, hipStream_t st) {
    const int blocks = (int)(((size_t)p.D * LPC + 255) / 256), most = 4096 / blocks + 1;
    hipLaunchKernelGGL((k_scan_token<T, W, LPC>), dim3(blocks, p.n_seq < most ? p.n_seq : most), dim3(256), 0, st, p);
}

template <typename T>
static void scan_launch(const scan_p &p, hipStream_t st) {
    const int N = p.N;
    if (p.starts) {
        if (N <= 4) scan_rows_launch<T, 4, 1, 8>(p, st);
        else if (N <= 8) scan_rows_launch<T, 8, 1, 8>(p, st);
        else if (N <= 16) scan_rows_launch<T, 16, 1, 8>(p, st);
        else if (N <= 32) scan_rows_launch<T, 16, 2, 8>(p, st);
        else if (N <= 64) scan_rows_launch<T, 16, 4, 8>(p, st);
        else if (N <= 128) scan_rows_launch<T, 16, 8, 4>(p, st);
        else scan_rows_launch<T, 16, 16, 2>(p, st);
    } else if (N % 4 == 0) {
        if (N <= 4) scan_token_launch<T, 4, 1>(p, st);
        else if (N <= 8) scan_token_launch<T, 4, 2>(p, st);
        else if (N <= 16) scan_token_launch<T, 4, 4>(p, st);
        else if (N <= 32) scan_token_launch<T, 4, 8>(p, st);
        else if (N <= 64) scan_token_launch<T, 4, 16>(p, st);
        else if (N <= 128) scan_token_launch<T, 4, 32>(p, st);
        else scan_token_launch<T, 4, 64>(p, st);
    } else {
        if (N <= 8) scan_token_launch<T, 1, 8>(p, st);
        else if (N <= 32) scan_token_launch<T, 1, 32>(p, st);
        else scan_token_launch<T, 1, 64>(p, st);
    }
}

extern "C" size_t wk_scan_work(int tokens, int D, int N, int n_seq, int longest) {
    return scan_floats(scan_split(tokens, D, N, n_seq, longest), D, N) * 4;
}

extern "C" int wk_selective_scan(const warp_hip_scan_args *a, void *stream) {
    const size_t dn = (size_t)a->channels * a->states;
    scan_plan s = {0, 0, 0};
    if (a->starts) s = scan_split(a->tokens, a->channels, a->states, a->n_seq, a->longest);
    float *w = (float *)a->work;
    scan_p p = {a->tokens, a->n_seq, a->channels, a->states, a->groups, a->n_slots, a->softplus, s.chunk, s.chunks,
                a->starts, a->slots, a->x, a->dt, a->B, a->C, a->z, a->ldx, a->lddt, a->ldbc, a->ldz, a->ldy,
                a->A, a->D, a->dt_bias, a->state_in, a->state_out, a->y,
                w, w + 2 * s.chunks * dn, w + s.chunks * dn, (int *)(w + s.chunks * (2 * dn + a->channels))};
    if (a->type == WARP_HIP_F32) scan_launch<float>(p, (hipStream_t)stream);
    else if (a->type == WARP_HIP_BF16) scan_launch<bf16_t>(p, (hipStream_t)stream);
    else scan_launch<f16_t>(p, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
