// conv.hip — the short causal convolution in front of a recurrence
// (warp_hip_short_conv): y[t][c] = act(bias[c] + sum_j w[c][j] u[t - taps + 1 + j][c]),
// where u is a sequence's inputs with its last taps - 1 earlier ones before
// them. The reference's counterpart is one token's step on a ring
// (short_conv_step, src/waste_backend.h:73-74); here it is whole packed
// prompts too, and the carried rows lie in time order.
//
// What bounds it is memory: each input is read once, each output written
// once, 2 taps + 4 operations on the vector units between them.

#include "rows.h"
#include "warp_internal.h"

constexpr int CONV_MAX_TAPS = 8;

struct conv_p {
    int tokens, n_seq, C, taps, n_slots, run, silu;
    const int *starts, *slots;
    const void *x;
    size_t ldx;
    const float *w, *bias;
    const void *sin;
    void *sout, *y;
    size_t ldy;
};

// A thread's V channels: weights and bias in registers, taps aligned to the
// end of the window (KS = 0: any number of taps up to CONV_MAX_TAPS).
template <typename T, int V, int KS>
struct conv_t {
    static constexpr int NT = KS ? KS : CONV_MAX_TAPS;
    float w[NT][V], b[V];
    int first;                                    // of the window's NT places that hold a tap
    bool silu;

    __device__ __forceinline__ void weights(const conv_p &p, int c0, int n) {
        first = KS ? 0 : NT - p.taps;
        silu = p.silu;
#pragma unroll
        for (int i = 0; i < V; i++) {
            b[i] = i < n && p.bias ? p.bias[c0 + i] : 0.0f;
#pragma unroll
            for (int j = 0; j < NT; j++)
                w[j][i] = i < n && j >= first ? p.w[(size_t)(c0 + i) * (NT - first) + j - first] : 0.0f;
        }
    }
    // u[first .. NT - 1]: the inputs, the newest last
    __device__ __forceinline__ vec_t<T, V> out(const vec_t<T, V> *u) const {
        vec_t<T, V> y;
#pragma unroll
        for (int i = 0; i < V; i++) {
            float a = b[i];
#pragma unroll
            for (int j = 0; j < NT; j++)
                if (KS || j >= first) a = __builtin_fmaf(w[j][i], (float)u[j].e[i], a);
            y.e[i] = (T)(silu ? rows_silu(a) : a);
        }
        return y;
    }
};

// One token of each of n_seq sequences: a thread takes V channels of one.
template <typename T, int KS>
__global__ __launch_bounds__(256) void k_conv_token(conv_p p) {
    constexpr int V = rows_of<T>::V, NT = KS ? KS : CONV_MAX_TAPS;
    const int c0 = ((int)blockIdx.x * (int)blockDim.x + (int)threadIdx.x) * V, n = min(V, p.C - c0);
    if (n <= 0) return;
    conv_t<T, V, KS> k;
    k.weights(p, c0, n);
    const int hist = NT - 1 - k.first;
    for (int s = blockIdx.y; s < p.n_seq; s += gridDim.y) {
        const int slot = seq_slot(p.slots, s, p.n_slots);
        if (slot < 0) continue;
        vec_t<T, V> u[NT];
        const T *in = (const T *)p.sin + (size_t)slot * hist * p.C + c0;
#pragma unroll
        for (int j = 0; j < NT - 1; j++)
            if (KS || j >= k.first) u[j] = load_vec<T, V>(in + (size_t)(j - k.first) * p.C, p.sin ? n : 0);
        u[NT - 1] = load_vec<T, V>((const T *)p.x + (size_t)s * p.ldx + c0, n);
        store_vec<T, V>((T *)p.y + (size_t)s * p.ldy + c0, k.out(u), n);
        if (!p.sout) continue;
        T *out = (T *)p.sout + (size_t)slot * hist * p.C + c0;
#pragma unroll
        for (int j = 0; j < NT - 1; j++)
            if (KS || j >= k.first) store_vec<T, V>(out + (size_t)(j - k.first) * p.C, u[j + 1], n);
    }
}

// Packed sequences: a wave takes 64 V channels of a run of rows, whatever
// sequences the run holds, so that ragged batches split evenly. The window
// slides through registers, so a run reads its own rows once and taps - 1
// before it.
// A sequence's first taps - 1 rows (those that read the carried inputs) all
// belong to the run in which the sequence begins, past that run's end if
// need be; the same thread then writes the inputs to carry on. So state_out
// may be state_in: nobody else reads a slot's state.
template <typename T, int KS>
__global__ __launch_bounds__(256) void k_conv_rows(conv_p p) {
    constexpr int V = rows_of<T>::V, NT = KS ? KS : CONV_MAX_TAPS, U = 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c0 = ((int)blockIdx.x * 64 + lane) * V, n = min(V, p.C - c0);
    if (n <= 0) return;
    conv_t<T, V, KS> k;
    k.weights(p, c0, n);
    const int hist = NT - 1 - k.first, runs = max(1, (p.tokens + p.run - 1) / p.run);
    const T *x = (const T *)p.x + c0;
    T *y = (T *)p.y + c0;
    for (int q = (int)blockIdx.y * 4 + wave; q < runs; q += (int)gridDim.y * 4) {
        const int r0 = q * p.run, r1 = min(r0 + p.run, p.tokens);
        for (int s = seq_from(p.starts, p.n_seq, r0); s < p.n_seq; s++) {
            const seq_t seq = seq_at(p.starts, s, p.tokens);
            if (seq.b >= r1 && q + 1 < runs) break;
            const bool mine = seq.b >= r0;        // it begins here
            const int slot = seq_slot(p.slots, s, p.n_slots);
            if (slot < 0) continue;
            const T *in = p.sin ? (const T *)p.sin + (size_t)slot * hist * p.C + c0 : nullptr;
            const int lo = mine ? seq.b : max(r0, seq.b + hist), hi = min(seq.e, mine ? max(r1, seq.b + hist) : r1);
            if (lo < hi) {
                vec_t<T, V> u[NT - 1 + U], nx[U];
#pragma unroll
                for (int i = 0; i < U; i++) nx[i] = load_vec<T, V>(x + (size_t)(lo + i) * p.ldx, lo + i < hi ? n : 0);
#pragma unroll
                for (int j = 0; j < NT - 1; j++) {
                    const int at = lo - (NT - 1) + j;
                    if (!KS && j < k.first) continue;
                    if (at >= seq.b) u[j] = load_vec<T, V>(x + (size_t)at * p.ldx, n);
                    else u[j] = load_vec<T, V>(in + (ptrdiff_t)(hist + at - seq.b) * p.C, in ? n : 0);
                }
                for (int t = lo; t < hi; t += U) {
#pragma unroll
                    for (int i = 0; i < U; i++) u[NT - 1 + i] = nx[i];
#pragma unroll
                    for (int i = 0; i < U; i++)
                        nx[i] = load_vec<T, V>(x + (size_t)(t + U + i) * p.ldx, t + U + i < hi ? n : 0);
#pragma unroll
                    for (int i = 0; i < U; i++)
                        if (t + i < hi) store_vec<T, V>(y + (size_t)(t + i) * p.ldy, k.out(u + i), n);
#pragma unroll
                    for (int j = 0; j < NT - 1; j++) u[j] = u[j + U];
                }
            }
            if (!mine || !p.sout) continue;
            T *out = (T *)p.sout + (size_t)slot * hist * p.C + c0;
            // in ascending order, which state_out = state_in allows: a row
            // moves to its own place or one before it
            for (int j = 0; j < hist; j++) {
                const int at = seq.e - hist + j;
                const vec_t<T, V> v = at >= seq.b ? load_vec<T, V>(x + (size_t)at * p.ldx, n)
                                                  : load_vec<T, V>(in + (ptrdiff_t)(hist + at - seq.b) * p.C, in ? n : 0);
                store_vec<T, V>(out + (size_t)j * p.C, v, n);
            }
        }
    }
}

template <typename T>
static void conv_launch(const conv_p &p, bool token, hipStream_t st) {
    constexpr int V = rows_of<T>::V;
    const int groups = (p.C + V - 1) / V;
    if (token) {
        const dim3 grid((groups + 63) / 64, p.n_seq < 32768 ? p.n_seq : 32768), block(64);
        if (p.taps == 4) hipLaunchKernelGGL((k_conv_token<T, 4>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((k_conv_token<T, 0>), grid, block, 0, st, p);
        return;
    }
    const int runs = (p.tokens + p.run - 1) / p.run, blocks = runs < 4 ? 1 : (runs + 3) / 4;
    const dim3 grid((groups + 63) / 64, blocks < 32768 ? blocks : 32768), block(256);
    if (p.taps == 4) hipLaunchKernelGGL((k_conv_rows<T, 4>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((k_conv_rows<T, 0>), grid, block, 0, st, p);
}

extern "C" int wk_short_conv(const warp_hip_conv_args *a, void *stream) {
    conv_p p = {a->tokens, a->n_seq, a->channels, a->taps, a->n_slots, 16, a->silu, a->starts, a->slots, a->x, a->ldx,
                a->w, a->bias, a->state_in, a->state_out, a->y, a->ldy};
    if (a->type == WARP_HIP_F32) conv_launch<float>(p, !a->starts, (hipStream_t)stream);
    else if (a->type == WARP_HIP_BF16) conv_launch<bf16_t>(p, !a->starts, (hipStream_t)stream);
    else conv_launch<f16_t>(p, !a->starts, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
