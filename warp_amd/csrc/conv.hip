// conv.hip — the short causal convolution in front of a recurrence
// (warp_hip_short_conv): y[t][c] = act(bias[c] + sum_j w[c][j] u[t - taps + 1 + j][c]),
// where u is a sequence's inputs with its last taps - 1 earlier ones before
// them. The reference's counterpart is one token's step on a ring
// (short_conv_step, src/waste_backend.h:73-74); here it is whole packed
// prompts too, and the carried rows lie in time order.
//
// What bounds it is memory: each input is read once, each output written
// once, about 19 issue slots of the vector units between them (four taps, and
// SiLU's two instructions at half of the rate), half of the time memory takes.
// 8,191 bf16 rows of 4,640 channels in 11 sequences: 30.4 us, 5.0 TB/s (a copy
// that leaves the caches behind reaches 4.7); a quarter more with stores that
// go through L2.

#include "rows.h"
#include "warp_internal.h"

constexpr int CONV_MAX_TAPS = 8;

struct conv_p {
    int tokens, n_seq, C, taps, n_slots, run, silu;              // run: rows of a wave
    const int *starts, *slots;
    const void *x;
    size_t ldx;
    const float *w, *bias;
    const void *sin;
    void *sout, *y;
    size_t ldy;
};

// A thread's V channels: weights and bias in registers, taps aligned to the
// end of the window (KS = 0: any number of taps up to CONV_MAX_TAPS, for rows
// shorter than a vector). Up to three taps a vector is 16 bytes, above that 8:
// weights and window grow with the taps, and four of 16 bytes leave three
// waves to a SIMD (8,191 rows of 4,640 bf16 36.1 us, 31.5 with 8 bytes; with
// any number of taps in a loop, three take 54.8 us, so 31.6).
template <typename T, int KS, bool ONE>
struct conv_t {
    static constexpr int V = KS > 3 ? rows_of<T>::V / 2 : rows_of<T>::V, NT = KS ? KS : CONV_MAX_TAPS;
    typedef cols_t<T, ONE, V> cols;
    float w[NT][V], b[V];
    int first;                                    // of the window's NT places that hold a tap
    bool silu;

    __device__ __forceinline__ conv_t(const conv_p &p, const cols &k) {
        first = KS ? 0 : NT - p.taps;
        silu = p.silu;
#pragma unroll
        for (int i = 0; i < V; i++) {
            b[i] = (!ONE || i < k.n) && p.bias ? p.bias[k.c + i] : 0.0f;
#pragma unroll
            for (int j = 0; j < NT; j++)
                w[j][i] = (!ONE || i < k.n) && (KS || j >= first) ? p.w[(size_t)(k.c + i) * (NT - first) + j - first]
                                                                  : 0.0f;
        }
    }
    // A row's outputs, from the window u[first .. NT - 2] before it; the
    // window moves on by the row.
    __device__ __forceinline__ vec_t<T, V> step(float (&u)[NT][V], const vec_t<T, V> &x) const {
        vec_t<T, V> y;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const float c = (float)x.e[i];
            float a = b[i];
#pragma unroll
            for (int j = 0; j < NT - 1; j++)
                if (KS || j >= first) a = __builtin_fmaf(w[j][i], u[j][i], a);
            a = __builtin_fmaf(w[NT - 1][i], c, a);
#pragma unroll
            for (int j = 0; j + 1 < NT - 1; j++) u[j][i] = u[j + 1][i];
            if (NT > 1) u[NT - 2][i] = c;
            y.e[i] = (T)(silu ? rows_silu(a) : a);
        }
        return y;
    }
};

// One token of each of n_seq sequences: a thread takes V channels of one.
template <typename T, int KS, bool ONE>
__global__ __launch_bounds__(256) void k_conv_token(conv_p p) {
    constexpr int V = conv_t<T, KS, ONE>::V, NT = conv_t<T, KS, ONE>::NT;
    const int c0 = ((int)blockIdx.x * (int)blockDim.x + (int)threadIdx.x) * V;
    if (c0 >= p.C) return;
    const typename conv_t<T, KS, ONE>::cols k(c0, p.C);
    const conv_t<T, KS, ONE> conv(p, k);
    const int hist = NT - 1 - conv.first;
    for (int s = blockIdx.y; s < p.n_seq; s += gridDim.y) {
        const int slot = seq_slot(p.slots, s, p.n_slots);
        if (slot < 0) continue;
        vec_t<T, V> h[NT], x = k.load((const T *)p.x + (size_t)s * p.ldx + k.c);
        const T *in = (const T *)p.sin + (size_t)slot * hist * p.C + k.c;
        float u[NT][V];
#pragma unroll
        for (int j = 0; j < NT - 1; j++) {
            h[j].e = 0;
            if (p.sin && (KS || j >= conv.first)) h[j] = k.load(in + (size_t)(j - conv.first) * p.C);
        }
        h[NT - 1] = x;
#pragma unroll
        for (int j = 0; j < NT - 1; j++)
#pragma unroll
            for (int i = 0; i < V; i++) u[j][i] = (float)h[j].e[i];
        k.store((T *)p.y + (size_t)s * p.ldy + k.c, conv.step(u, x));
        if (!p.sout) continue;
        T *out = (T *)p.sout + (size_t)slot * hist * p.C + k.c;
#pragma unroll
        for (int j = 0; j < NT - 1; j++)
            if (KS || j >= conv.first) k.store(out + (size_t)(j - conv.first) * p.C, h[j + 1]);
    }
}

// Packed sequences: a wave takes 64 V channels of a run of rows, whatever
// sequences the run holds, so that ragged batches split evenly. The window
// slides through registers, so a run reads its own rows once and taps - 1
// before it; the next rows are loaded while these are computed.
// A sequence's first taps - 1 rows (those that read the carried inputs) all
// belong to the run in which the sequence begins, past that run's end if
// need be; the same thread then writes the inputs to carry on. So state_out
// may be state_in: what a thread uses of a slot's state nobody else writes.
template <typename T, int KS, bool ONE>
__global__ __launch_bounds__(256) void k_conv_rows(conv_p p) {
    constexpr int V = conv_t<T, KS, ONE>::V, NT = conv_t<T, KS, ONE>::NT, U = 4;
    typedef vec_t<T, V> vec;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c0 = ((int)blockIdx.x * 64 + lane) * V, runs = max(1, (p.tokens + p.run - 1) / p.run);
    const seqs_t seqs(p.starts, p.slots, p.n_seq, p.tokens, p.n_slots);
    const bool live = c0 < p.C;
    const typename conv_t<T, KS, ONE>::cols k(live ? c0 : p.C - 1, p.C);
    const conv_t<T, KS, ONE> conv(p, k);
    const int hist = NT - 1 - conv.first;
    const T *x = (const T *)p.x + k.c;
    T *y = (T *)p.y + k.c;
    for (int q = (int)blockIdx.y * 4 + wave; q < runs; q += (int)gridDim.y * 4) {
        const int r0 = q * p.run, r1 = min(r0 + p.run, p.tokens), s0 = seqs.from(r0);
        if (!live) continue;
        for (int s = s0; s < p.n_seq; s++) {
            const seq_t seq = seqs.at(s);
            if (seq.b >= r1 && q + 1 < runs) break;
            const bool mine = seq.b >= r0;        // it begins here
            if (seq.slot < 0) continue;
            const T *in = p.sin ? (const T *)p.sin + (size_t)seq.slot * hist * p.C + k.c : nullptr;
            // row t of the sequence, or of the inputs carried to it
            auto before = [&](int t) {
                vec v;
                v.e = 0;
                if (t >= seq.b) v = k.load(x + (size_t)t * p.ldx);
                else if (in) v = k.load(in + (size_t)(hist + t - seq.b) * p.C);
                return v;
            };
            const int lo = mine ? seq.b : max(r0, seq.b + hist), hi = min(seq.e, mine ? max(r1, seq.b + hist) : r1);
            if (lo < hi) {
                float u[NT][V];
                vec cu[U], nx[U];
#pragma unroll
                for (int i = 0; i < U; i++) nx[i] = k.load(x + (size_t)min(lo + i, hi - 1) * p.ldx);
#pragma unroll
                for (int j = 0; j < NT - 1; j++) {
                    if (!KS && j < conv.first) continue;
                    const vec v = before(lo - (NT - 1) + j);
#pragma unroll
                    for (int i = 0; i < V; i++) u[j][i] = (float)v.e[i];
                }
                for (int t = lo; t < hi; t += U) {
#pragma unroll
                    for (int i = 0; i < U; i++) cu[i] = nx[i];
                    if (t + U < hi) {
#pragma unroll
                        for (int i = 0; i < U; i++) nx[i] = k.load(x + (size_t)min(t + U + i, hi - 1) * p.ldx);
                    }
#pragma unroll
                    for (int i = 0; i < U; i++)
                        if (t + i < hi) k.stream(y + (size_t)(t + i) * p.ldy, conv.step(u, cu[i]));
                }
            }
            if (!mine || !p.sout) continue;
            T *out = (T *)p.sout + (size_t)seq.slot * hist * p.C + k.c;
            // in ascending order, which state_out = state_in allows: a row
            // moves to its own place or one before it
            for (int j = 0; j < hist; j++) k.store(out + (size_t)j * p.C, before(seq.e - hist + j));
        }
    }
}

template <typename T, int KS, bool ONE>
static void conv_launch(conv_p p, hipStream_t st) {
    constexpr int V = conv_t<T, KS, ONE>::V;
    const int cols = ((p.C + V - 1) / V + 63) / 64;
    if (!p.starts) {
        // (waves that take sequences in turn load their weights once: 400
        // sequences of 8,000 bf16 channels 13.7 us, 18.6 with a wave each)
        const int most = 2048 / cols + 1;
        hipLaunchKernelGGL((k_conv_token<T, KS, ONE>), dim3(cols, p.n_seq < most ? p.n_seq : most), dim3(64), 0, st, p);
        return;
    }
    // Runs of 12 rows read 3 of 15 twice and load their weights once, but a
    // batch has to make enough waves of them: in runs of 4, 8, 12 and 24,
    // 8,191 bf16 rows of 4,640 channels take 38.6, 30.6, 30.4 and 33.1 us, 1,537
    // f32 rows of 4,096 10.0, 10.0, 9.8 and 11.0, 300 f16 rows of 4,640 8.0, 8.5,
    // 9.2 and 11.7, 1,000 f32 rows of 1,000 6.5, 6.7, 7.2 and 9.5.
    p.run = (int64_t)p.tokens * cols >= 24576 ? 12 : 4;
    const int blocks = (p.tokens + 4 * p.run - 1) / (4 * p.run);
    hipLaunchKernelGGL((k_conv_rows<T, KS, ONE>), dim3(cols, blocks < 1 ? 1 : blocks < 32768 ? blocks : 32768), dim3(256), 0,
                       st, p);
}
template <typename T>
static void conv_type(const conv_p &p, hipStream_t st) {
    if (p.C < rows_of<T>::V) return conv_launch<T, 0, true>(p, st);
    switch (p.taps) {
    case 1: return conv_launch<T, 1, false>(p, st);
    case 2: return conv_launch<T, 2, false>(p, st);
    case 3: return conv_launch<T, 3, false>(p, st);
    case 4: return conv_launch<T, 4, false>(p, st);
    case 5: return conv_launch<T, 5, false>(p, st);
    case 6: return conv_launch<T, 6, false>(p, st);
    case 7: return conv_launch<T, 7, false>(p, st);
    default: return conv_launch<T, 8, false>(p, st);
    }
}

extern "C" int wk_short_conv(const warp_hip_conv_args *a, void *stream) {
    conv_p p = {a->tokens, a->n_seq, a->channels, a->taps, a->n_slots, 16, a->silu, a->starts, a->slots, a->x, a->ldx,
                a->w, a->bias, a->state_in, a->state_out, a->y, a->ldy};
    if (a->type == WARP_HIP_F32) conv_type<float>(p, (hipStream_t)stream);
    else if (a->type == WARP_HIP_BF16) conv_type<bf16_t>(p, (hipStream_t)stream);
    else conv_type<f16_t>(p, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
