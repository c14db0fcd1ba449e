// scan.hip — the selective state space scan (warp_hip_selective_scan). Per
// channel d with states n, row by row of a sequence:
//   dt' = softplus(dt + dt_bias)                        (or dt + dt_bias)
//   h[n] = exp(dt' A[d][n]) h[n] + dt' x B[n]
//   y    = (sum_n C[n] h[n] + D x) silu(z)
// with B and C shared by the channels of a group. The states are f32 from end
// to end, dt' and the sums too; only x, dt, B, C, z and y are of the rows' type.
//
// What bounds prompts is the vector units: per row, channel and state a
// product and an exponential for the decay (the exponential issues at half
// the rate), a product, and two fused multiply-adds, six issue slots, against
// 8 bytes of rows per channel. The decays differ by channel and state, so
// nothing of this is a matrix product but dt' x B, an outer one over channels
// and states: as four 4 x 4 x 1 matrix instructions a row it takes the place of
// a fifth of the vector instructions and the same time (70 + 97 us of
// a prompt that took 70 + 94), as each holds those up for some 15 cycles. Single
// tokens are bound by their states, read and written once.

#include <math.h>
#include <type_traits>

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
};

constexpr float LOG2E = 1.44269504088896341f;

// log(1 + e^v) = max(v, 0) + log(1 + e), e = exp(-|v|) <= 1, and log(1 + e) =
// 2 atanh(s) with s = e / (2 + e) <= 1/3, whose series in s^2 over s is here
// the polynomial of degree 4 with the least relative error on [0, 1/9], 4e-9.
// Small results keep their digits, as the time steps of slow channels need them.
__device__ __forceinline__ float scan_softplus(float v) {
    const float e = rows_exp(-__builtin_fabsf(v)), s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
    float r = 0.14089166f;
    r = __builtin_fmaf(r, q, 0.13980304f);
    r = __builtin_fmaf(r, q, 0.20012455f);
    r = __builtin_fmaf(r, q, 0.33333158f);
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
// each in a run (of rows that are no whole number of runs the last is short),
// and keep that channel's decay rates for the sequences they take in turn.
// 256 sequences of 4,608 channels by 16 states, bf16: 31.1 us, 5.2 TB/s (a
// copy that leaves the caches behind reaches 4.7); 44 us with stores through
// L2. Single states (W = 1) for rows that are no multiple of 4 take 69 us for
// 200 sequences of 3,000 by 23, these 57.
template <typename T, int W, int LPC>
__global__ __launch_bounds__(256) void k_scan_token(scan_p p) {
    const int lane = threadIdx.x % LPC, d = ((int)blockIdx.x * 256 + (int)threadIdx.x) / LPC;
    if (d >= p.D) return;
    const int n = lane * W, m = p.N - n, g = d / (p.D / p.G);
    vec_t<float, W> A = load_vec<float, W>(p.A + (size_t)d * p.N + n, m);
    A.e *= LOG2E;
    const float bias = p.bias ? p.bias[d] : 0.0f, skip = p.skip ? p.skip[d] : 0.0f;
    for (int s = blockIdx.y; s < p.n_seq; s += gridDim.y) {
        const int slot = seq_slot(p.slots, s, p.n_slots);
        if (slot < 0) continue;
        const size_t at = ((size_t)slot * p.D + d) * p.N + n, bc = (size_t)s * p.ldbc + (size_t)g * p.N + n;
        vec_t<float, W> h = load_vec<float, W>(p.sin + at, p.sin ? m : 0);
        const vec_t<T, W> B = load_vec<T, W>((const T *)p.B + bc, m), C = load_vec<T, W>((const T *)p.C + bc, m);
        const float x = (float)((const T *)p.x)[(size_t)s * p.ldx + d];
        float v = (float)((const T *)p.dt)[(size_t)s * p.lddt + d] + bias;
        if (p.softplus) v = scan_softplus(v);
        const float u = v * x;
        float y = 0.0f;
#pragma unroll
        for (int j = 0; j < W; j++) {
            h.e[j] = __builtin_fmaf(h.e[j], __builtin_amdgcn_exp2f(v * A.e[j]), u * (float)B.e[j]);
            y = __builtin_fmaf(h.e[j], (float)C.e[j], y);
        }
        // (past L2: by the next token the other layers' states have been through it)
        if (p.sout) stream_vec<float, W>(p.sout + at, h, m);
        y = scan_sum<LPC>(y);
        y = __builtin_fmaf(skip, x, y);
        if (p.z) y *= rows_silu((float)((const T *)p.z)[(size_t)s * p.ldz + d]);
        if (lane == 0) ((T *)p.y)[(size_t)s * p.ldy + d] = (T)y;
    }
}

// What lane p of each group of LPC lanes has, in all of the group's lanes.
template <int LPC>
__device__ __forceinline__ float scan_from(float v, int p) {
    const int x = __float_as_int(v);
#define DPP(old, ctl, banks) __builtin_amdgcn_update_dpp(old, x, ctl, 0xf, banks, false)
#define FROM(ctl) __int_as_float(__builtin_amdgcn_mov_dpp(x, ctl, 0xf, 0xf, true))
    if (LPC == 1) return v;
    if (LPC == 2) return p == 0 ? FROM(0xa0) : FROM(0xf5);                       // quad_perm
    if (LPC == 4) return p == 0 ? FROM(0x00) : p == 1 ? FROM(0x55) : p == 2 ? FROM(0xaa) : FROM(0xff);
    // a row's lane to the row; with two groups in a row, lane p to the banks of one and 8 + p to the other's
#define ROW(n) (LPC == 16 ? FROM(0x150 + n) : __int_as_float(DPP(DPP(x, 0x150 + n, 0x3), 0x150 + ((n + 8) & 15), 0xc)))
    switch (p) {
    case 0: return ROW(0);
    case 1: return ROW(1);
    case 2: return ROW(2);
    case 3: return ROW(3);
    case 4: return ROW(4);
    case 5: return ROW(5);
    case 6: return ROW(6);
    default: return ROW(7);
    }
#undef ROW
#undef FROM
#undef DPP
}

// A lane's element `at` bytes into a row. ONE: the row is the wave's, its
// address stays in scalar registers and the lane's offset is the load's own
// (left to itself, the compiler adds the two in each lane).
template <bool ONE, typename T>
__device__ __forceinline__ __attribute__((address_space(1))) T *scan_at(const char *row, unsigned at) {
    typedef __attribute__((address_space(1))) char *bytes;
    bytes b = (bytes)(char *)row;
    if (ONE) asm volatile("" : "+s"(b));
    return (__attribute__((address_space(1))) T *)(b + at);
}

// Prompts. LPC lanes of a wave share a channel, S states each in registers;
// a wave is a block and takes 64 / LPC channels of one group. The rows go in
// batches of U: their B and C are laid out in LDS as f32, where a row's lie at
// one address for all channels. Of x, dt and z a lane takes the rows that are
// its own among the group's (all of them, if it has the channel to itself):
// loads them a batch ahead, makes dt' of them, hands that to the other lanes
// row by row, and gates and stores their outputs. A full batch is one straight
// run of instructions (the states' chain of multiply-adds is the only thing
// that waits, S of them in turn).
template <typename T, int S, int LPC, int U>
struct scan_t {
    static constexpr int RS = S * LPC;                     // states, filled up
    static constexpr int P = LPC < U ? LPC : U, R = U / P; // lanes of a group with rows of their own, rows each
    static_assert(P <= 8 || LPC == 1, "scan_from hands on the first eight lanes' values");
    float A[S], h[S], bias, skip;
    int lane, part, d, g;

    // (a wave's spare lanes repeat its last channel, and store what that does)
    __device__ __forceinline__ void open(const scan_p &p) {
        const int per = p.D / p.G, blocks = (per * LPC + 63) / 64, i = (int)blockIdx.x % blocks;
        lane = threadIdx.x;
        part = lane % LPC;
        g = (int)blockIdx.x / blocks;
        d = g * per + min((i * 64 + lane) / LPC, per - 1);
        bias = p.bias ? p.bias[d] : 0.0f;
        skip = p.skip ? p.skip[d] : 0.0f;
        get(p, A, p.A);
#pragma unroll
        for (int n = 0; n < S; n++) A[n] *= LOG2E;
    }
    // This lane's states' values of an array [D][N] (0 where it has none), four
    // at a time if the rows are whole fours: the lanes' are a row apart, and
    // each instruction costs a look into a cache line per lane.
    __device__ __forceinline__ void get(const scan_p &p, float (&v)[S], const float *from) const {
        const float *at = from + (size_t)d * p.N + part * S;
        const int m = p.N - part * S;
        if (p.N % 4 == 0) {
#pragma unroll
            for (int n = 0; n < S; n += 4) {
                const vec_t<float, 4> q = load_vec<float, 4>(at + n, n < m ? 4 : 0);
#pragma unroll
                for (int i = 0; i < 4; i++) v[n + i] = q.e[i];
            }
        } else {
#pragma unroll
            for (int n = 0; n < S; n++) v[n] = n < m ? at[n] : 0.0f;
        }
    }
    __device__ __forceinline__ void state(const scan_p &p, const float *from) {
        if (from) {
            get(p, h, from);
        } else {
#pragma unroll
            for (int n = 0; n < S; n++) h[n] = 0.0f;
        }
    }
    __device__ __forceinline__ void store(const scan_p &p, float *to) const {
        float *at = to + (size_t)d * p.N + part * S;
        const int m = p.N - part * S;
        if (p.N % 4 == 0) {
#pragma unroll
            for (int n = 0; n < S; n += 4) {
                vec_t<float, 4> q;
#pragma unroll
                for (int i = 0; i < 4; i++) q.e[i] = h[n + i];
                if (n < m) store_vec<float, 4>(at + n, q, 4);
            }
        } else {
#pragma unroll
            for (int n = 0; n < S; n++)
                if (n < m) at[n] = h[n];
        }
    }

    // Rows lo .. hi - 1 of one sequence. OUT: with y; without, dt' is summed up.
    template <bool OUT>
    __device__ __forceinline__ float rows(const scan_p &p, int lo, int hi, float *bc) {
        // B, or B and C, by fours of states a lane where a row has more than 4, else one by one
        constexpr int K = OUT ? 2 : 1, W = LPC > 1 ? 4 : 1, Q = U * K * RS / W, M = (Q + 63) / 64;
        if (lo >= hi) return 0.0f;
        T tx[R], td[R], tz[R];
        vec_t<T, W> tb[M];
        float sum = 0.0f;
        // this lane's offset in a row (anew each time, or the additions to it would leave their loads)
        auto mine = [&] {
            unsigned at = d * sizeof(T);
            if (P == 1) asm volatile("" : "+v"(at));
            return at;
        };
        const int own = part % P;                          // this lane's rows: own, own + P, ...
        const void *gate = p.z ? p.z : p.x;                // (without one x again, which saves the loads a branch each)
        const size_t sx = p.ldx * sizeof(T), sd = p.lddt * sizeof(T), sz = p.z ? p.ldz * sizeof(T) : sx, sy = p.ldy * sizeof(T);
        // With one row a batch to a lane, where it and the lane's parts of B and C lie behind the batch's first
        // row is multiplied out once, for full batches: a product of 64 bits costs as much as three states
        // (1,999 f32 rows of 2,304 channels and 64 states 130 -> 125 us; lanes with two rows gain nothing).
        constexpr bool ONCE = P > 1 && R == 1;
        size_t wx, wd, wz, wb[M];
        auto reach = [&](int rows) {
            const size_t r = min(own, rows - 1);
            wx = r * sx, wd = r * sd, wz = r * sz;
#pragma unroll
            for (int i = 0; i < M; i++) {
                const int e = (lane + 64 * i) * W;
                wb[i] = (size_t)min(e / (RS * K), rows - 1) * p.ldbc + (size_t)g * p.N + min(e % RS, p.N - W);
            }
        };
        auto load = [&](int t) {
            if constexpr (ONCE) {
                if (t + U > hi) reach(hi - t);             // (which is the last)
                tx[0] = *(const T *)((const char *)p.x + t * sx + wx + d * sizeof(T));
                td[0] = *(const T *)((const char *)p.dt + t * sd + wd + d * sizeof(T));
                if (OUT) tz[0] = *(const T *)((const char *)gate + t * sz + wz + d * sizeof(T));
#pragma unroll
                for (int i = 0; i < M; i++) {
                    const T *row = (const T *)(OUT && (lane + 64 * i) * W / RS % K ? p.C : p.B) + t * p.ldbc;
                    tb[i].e = *(const typename vec_t<T, W>::mem *)(row + wb[i]);
                }
                return;
            }
            const unsigned at = mine();
            size_t r = min(t + (P > 1 ? own : 0), hi - 1);
            const char *xr = (const char *)p.x + r * sx, *dr = (const char *)p.dt + r * sd, *zr = (const char *)gate + r * sz;
#pragma unroll
            for (int i = 0; i < R; i++) {
                tx[i] = *scan_at<P == 1, const T>(xr, at);
                td[i] = *scan_at<P == 1, const T>(dr, at);
                if (OUT) tz[i] = *scan_at<P == 1, const T>(zr, at);
                const bool on = t + (i + 1) * P + (P > 1 ? own : 0) < hi;      // (behind the last the last again)
                if (P == 1) {
                    xr += on ? sx : 0;
                    dr += on ? sd : 0;
                    zr += on ? sz : 0;
                } else {
                    r = min(t + (i + 1) * P + own, hi - 1);
                    xr = (const char *)p.x + r * sx, dr = (const char *)p.dt + r * sd, zr = (const char *)gate + r * sz;
                }
            }
#pragma unroll
            for (int i = 0; i < M; i++) {
                const int e = (lane + 64 * i) * W, n = e % RS, r = min(e / (RS * K), hi - 1 - t);
                const T *row = (const T *)(OUT && e / RS % K ? p.C : p.B) + (size_t)t * p.ldbc + (size_t)g * p.N;
                // (the last of a row's begins early, as not to pass its end)
                tb[i].e = *(const typename vec_t<T, W>::mem *)(row + (size_t)r * p.ldbc + min(n, p.N - W));
            }
        };
        int t = lo;
        auto batch = [&](auto all) {
            constexpr bool FULL = decltype(all)::value;
            float x[R], v[R], u[R], z[R], y[R];
#pragma unroll
            for (int i = 0; i < R; i++) {
                x[i] = (float)tx[i];
                v[i] = (float)td[i] + bias;
                if (OUT) z[i] = (float)tz[i];
            }
#pragma unroll
            for (int i = 0; i < M; i++) {
                const int e = (lane + 64 * i) * W, n = e % RS, skip = n + W - p.N;
                vec_t<float, W> w;
#pragma unroll
                for (int j = 0; j < W; j++) w.e[j] = n < p.N ? (float)tb[i].e[j] : 0.0f;
                if (W > 1 && p.N % W && skip > 0) {
                    const auto all = w.e;
#pragma unroll
                    for (int j = 0; j < W; j++)
                        w.e[j] = skip == 1 && j < 3 ? all[(j + 1) & 3] : skip == 2 && j < 2 ? all[(j + 2) & 3]
                                 : skip == 3 && j < 1 ? all[3] : 0.0f;
                }
                if (Q % 64 == 0 || lane + 64 * i < Q) *(typename vec_t<float, W>::reg *)(bc + e) = w.e;
            }
            // (one wave: what it writes to LDS is there for its next reads)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (FULL) load(min(t + U, hi - 1));
            if (p.softplus) {
#pragma unroll
                for (int i = 0; i < R; i++) v[i] = scan_softplus(v[i]);
            }
#pragma unroll
            for (int i = 0; i < R; i++) u[i] = v[i] * x[i];
            auto row = [&](int i) {
                const float vi = scan_from<LPC>(v[i / P], i % P), ui = scan_from<LPC>(u[i / P], i % P);
                // (in fours of their own accord: as single loads some went out in twos)
                typedef vec_t<float, 4>::reg four;
                const four *b = (const four *)(bc + i * K * RS + part * S), *c = b + RS / 4;
                four o = 0;
#pragma unroll
                for (int m = 0; m < S / 4; m++) {
                    const four bm = b[m], cm = OUT ? c[m] : bm;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int n = 4 * m + j;
                        h[n] = __builtin_fmaf(h[n], __builtin_amdgcn_exp2f(vi * A[n]), ui * bm[j]);
                        if (OUT) o[j] = m == 0 ? h[n] * cm[j] : __builtin_fmaf(h[n], cm[j], o[j]);
                    }
                }
                if (OUT) {
                    const float all = scan_sum<LPC>((o[0] + o[1]) + (o[2] + o[3]));
                    y[i / P] = i % P == 0 || own == i % P ? all : y[i / P];
                }
            };
            auto out = [&](int n) {
#pragma unroll
                for (int i = 0; i < R; i++) y[i] = __builtin_fmaf(skip, x[i], y[i]);
                if (p.z) {
#pragma unroll
                    for (int i = 0; i < R; i++) y[i] *= rows_silu(z[i]);
                }
                const unsigned at = mine();
                char *to = (char *)p.y + (size_t)(t + (P > 1 ? own : 0)) * sy;
#pragma unroll
                for (int i = 0; i < R; i++, to += P * sy)
                    if ((FULL || i * P + (P > 1 ? own : 0) < n) && (P == LPC || part < P)) *scan_at<P == 1, T>(to, at) = (T)y[i];
            };
            if (!OUT) {
#pragma unroll
                for (int i = 0; i < R; i++)
                    if ((FULL || t + i * P + own < hi) && part < P) sum += v[i];
            }
#pragma unroll
            for (int i = 0; !FULL && i < R; i++) y[i] = 0.0f;
#pragma unroll
            for (int i = 0; i < U; i++)
                if (FULL || t + i < hi) row(i);
            if (OUT) out(hi - t);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };
        // (the last, short batch by itself: on a common way out of a loop
        // each batch would move every state from one register to another)
        if constexpr (ONCE) reach(U);
        load(lo);
        for (; t + U <= hi; t += U) batch(std::true_type());
        if (t < hi) batch(std::false_type());
        return scan_sum<LPC>(sum);
    }
};

// Waves to a SIMD that a batch's chunks are cut for. Of 16 states to a lane 3
// hold the vector units 90% busy, 4 95%, and no more may share a SIMD, or some
// get more than others. Fewer states leave room for more than their chunks are
// cut for (5 cost more in chunks), which whole sequences use: 100 of 30 rows of
// 4,608 channels by 16, four states a lane, 103 us, with three waves 120.
constexpr int scan_waves(int S, int lanes) { return S == 8 || (S == 16 && lanes >= 8) ? 3 : 4; }
#define SCAN_WAVES \
    __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(scan_waves(S, LPC), S == 16 ? scan_waves(S, LPC) : 8)))

// A whole sequence per wave (chunk = 0), or the rows [j chunk, (j + 1) chunk)
// of the packed batch, whatever sequences they hold, from the state that
// k_scan_join found at their beginning.
template <typename T, int S, int LPC, int U>
__global__ SCAN_WAVES void k_scan_rows(scan_p p) {
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
// (or the sequence's first state, if it begins here), and the sum of its dt',
// of which the chunk's decay is the exponential (NaN if it begins here: nothing
// before counts). Only for a sequence that goes on in the next chunk.
template <typename T, int S, int LPC, int U>
__global__ SCAN_WAVES void k_scan_part(scan_p p) {
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
        if (k.part == 0) p.sum[(size_t)j * p.D + k.d] = begins ? __builtin_nanf("") : sum;
    }
}

// What a chunk makes of the state h before it: exp2(l) h + e, e what it makes
// of zero, l its decay's exponent (NaN: nothing of what was before counts, or
// e is none either). A zero stays zero and an infinity one, as row by row, and
// the factor goes in halves, so that a state may grow or shrink by more than
// f32 can say at once.
__device__ __forceinline__ float scan_over(float h, float l, float e) {
    const float half = __builtin_fmaxf(__builtin_amdgcn_exp2f(0.5f * l), 1.17549435e-38f);
    return l != l || h == 0.0f ? e : __builtin_fmaf(h * half, half, e);
}

// The chunks in order: end[j] becomes the state at the end of chunk j. A lane
// takes one state, each of the block's waves a part of the chunks: first what
// the part makes of a state of zero and how much it leaves of one, then, from
// the state that the parts before it leave, the states themselves. Up to
// JOIN_Q chunks of a part stay in registers between the two.
constexpr int JOIN_Q = 10, JOIN_W = 16;
__global__ __launch_bounds__(64 * JOIN_W, 8) void k_scan_join(scan_p p) {
    __shared__ float sum[JOIN_W][64], left[JOIN_W][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = blockDim.x >> 6;
    const size_t dn = (size_t)p.D * p.N;                   // (at most 2^32: any state's index fits)
    const unsigned i = blockIdx.x * 64 + lane, at = min(i, (unsigned)(dn - 1));
    const int d = (int)(at / (unsigned)p.N), most = p.chunks - 1, q = (most + waves - 1) / waves;
    const int j0 = min(wave * q, most), j1 = min(j0 + q, most);
    const float A = p.A[at] * LOG2E;
    float h = 0.0f, w = 0.0f, e[JOIN_Q], l[JOIN_Q];
    // (behind the part's last chunk: ones that leave a state as it is)
    auto load = [&](int j) {
#pragma unroll
        for (int b = 0; b < JOIN_Q; b++) {
            const int c = min(j + b, most - 1);
            e[b] = p.end[(size_t)c * dn + at];
            l[b] = p.sum[(size_t)c * p.D + d];
        }
#pragma unroll
        for (int b = 0; b < JOIN_Q; b++) {
            e[b] = j + b < j1 ? e[b] : 0.0f;
            l[b] = j + b < j1 ? A * l[b] : 0.0f;
        }
    };
    auto walk = [&](int j, bool keep) {
#pragma unroll
        for (int b = 0; b < JOIN_Q; b++) {
            h = scan_over(h, l[b], e[b]);
            w += l[b];
            if (keep && j + b < j1 && i < dn) p.end[(size_t)(j + b) * dn + at] = h;
        }
    };
    for (int j = j0; j < j1; j += JOIN_Q) {
        load(j);
        if (waves > 1 || q > JOIN_Q) walk(j, waves == 1);
    }
    if (waves > 1) {
        sum[wave][lane] = h;
        left[wave][lane] = w;
        __syncthreads();
        h = 0.0f;
        for (int v = 0; v < wave; v++) h = scan_over(h, left[v][lane], sum[v][lane]);
    }
    if (q <= JOIN_Q) {
        walk(j0, true);
    } else if (waves > 1) {
        for (int j = j0; j < j1; j += JOIN_Q) {
            load(j);
            walk(j, true);
        }
    }
}

// How a packed batch of prompts is split: S states of a channel to a lane,
// and chunk = 0, a wave (per 64 / lanes channels) for each sequence, or chunks
// of so many rows, whose states are computed twice.
// A wave's rows come one after the other, so few long sequences want many
// waves of few rows each, and a short batch wants few states to a lane; but
// chunks cost their second computation and two more launches, and lanes of 4
// states more in all than lanes of 16. The choice is the least of a model, in
// ns, of what was measured: a row of a wave by itself (`alone`), a row among
// as many waves as keep the SIMDs busy (`rows`, and `part` for the chunks'
// first pass), and what the launches take. One bf16 prompt of 4,608 channels
// and 16 states: 4,096 rows take 1,840 us in one piece, 609 with 4 states a
// lane, 164 in 54 chunks (66 + 11 + 87), 400 rows 176, 63 and 38. 1,999 f32 rows
// of 2,304 channels and 64 states in 13 sequences: 137 in chunks (53 + 10 + 74)
// or, as their lengths are more or less even, 120 to 187 a wave to a sequence.
struct scan_plan {
    int S, lanes, chunk, chunks;
    double ns;
};
static scan_plan scan_try(int S, int lanes, int tokens, int D, int n_seq, int longest) {
    const double simds = 1024, waves = ((double)D * lanes + 63) / 64, load = tokens * waves / simds;
    const double alone = 70 + 21 * S + 60.0 / lanes, rows = 40 + 15 * S + 65.0 / lanes, part = 20 + 11 * S + 60.0 / lanes;
    // (a sequence longer than the others runs on by itself)
    const double over = longest - (double)tokens / n_seq;
    scan_plan r = {S, lanes, 0, 0, fmax(5000 + alone * longest, rows * load + alone * fmax(over, 0))};
    // as many chunks as there are waves for, or as k_scan_join joins in one go
    const int once = JOIN_Q * JOIN_W + 1, fit = (int)fmin(scan_waves(S, lanes) * simds / waves, tokens / 16);
    for (int most : {fit, once}) {
        if (most < 2 || most > fit) continue;
        // (one more than fits would run by itself at the end)
        const int chunk = ((tokens + most - 1) / most + 3) / 4 * 4, chunks = (tokens + chunk - 1) / chunk;
        const double join = 4000 + 0.0016 * chunks * D * S * lanes + (chunks > once ? 8000 : 0);
        const double ns = 4000 + join + fmax(8000 + alone * chunk, rows * load) + fmax(8000 + 0.75 * alone * chunk, part * load);
        if (chunks >= 2 && ns < r.ns) r = {S, lanes, chunk, chunks, ns};
    }
    return r;
}
static scan_plan scan_split(int tokens, int D, int N, int n_seq, int longest) {
    if (longest <= 0 || longest > tokens) longest = tokens;
    auto best = [&](int S, int lanes) { return scan_try(S, lanes, tokens, D, n_seq, longest); };
    if (N <= 4) return best(4, 1);
    if (N > 128) return best(16, 16);
    int lanes = 2;
    while (lanes * 4 < N) lanes *= 2;             // of 4 states each
    const scan_plan few = N > 64 ? best(8, 16) : best(4, lanes), many = N <= 8 ? best(8, 1) : best(16, lanes / 4);
    return few.ns < many.ns ? few : many;
}
static size_t scan_floats(const scan_plan &s, int D, int N) {
    return s.chunk ? (size_t)s.chunks * (2 * (size_t)D * N + D) : 0;
}

template <typename T, int S, int LPC, int U>
static void scan_rows_launch(const scan_p &p, hipStream_t st) {
    const int blocks = p.G * ((p.D / p.G * LPC + 63) / 64);
    auto rows = [](int n) { return (unsigned)(n < 32768 ? n : 32768); };
    if (p.chunk) {
        hipLaunchKernelGGL((k_scan_part<T, S, LPC, U>), dim3(blocks, rows(p.chunks - 1)), dim3(64), 0, st, p);
        const int parts = (p.chunks + JOIN_Q - 2) / JOIN_Q;
        hipLaunchKernelGGL(k_scan_join, dim3((unsigned)(((size_t)p.D * p.N + 63) / 64)),
                           dim3(64 * (parts < JOIN_W ? parts : JOIN_W)), 0, st, p);
    }
    hipLaunchKernelGGL((k_scan_rows<T, S, LPC, U>), dim3(blocks, rows(p.chunk ? p.chunks : p.n_seq)), dim3(64), 0, st, p);
}
template <typename T, int W, int LPC>
static void scan_token_launch(const scan_p &p, hipStream_t st) {
    const int blocks = (int)(((size_t)p.D * LPC + 255) / 256), most = 9216 / blocks + 1;     // (36 blocks a CU: 32.6 us; 16: 33.2, a block a row: 34.9)
    hipLaunchKernelGGL((k_scan_token<T, W, LPC>), dim3(blocks, p.n_seq < most ? p.n_seq : most), dim3(256), 0, st, p);
}

template <typename T>
static void scan_launch(const scan_p &p, const scan_plan &s, hipStream_t st) {
    const int N = p.N;
    if (p.starts) {
#define SCAN(S_, L_, U_) \
    if (s.S == S_ && s.lanes == L_) return scan_rows_launch<T, S_, L_, U_>(p, st)
        SCAN(4, 1, 8);
        SCAN(4, 2, 8);
        SCAN(4, 4, 8);
        SCAN(4, 8, 8);
        SCAN(4, 16, 8);
        SCAN(8, 1, 8);
        SCAN(8, 16, 8);
        SCAN(16, 1, 4);
        SCAN(16, 2, 4);
        SCAN(16, 4, 4);
        SCAN(16, 8, 8);
        SCAN(16, 16, 4);
#undef SCAN
    } else {
        if (N < 4) scan_token_launch<T, 1, 4>(p, st);
        else if (N == 4) scan_token_launch<T, 4, 1>(p, st);
        else if (N <= 8) scan_token_launch<T, 4, 2>(p, st);
        else if (N <= 16) scan_token_launch<T, 4, 4>(p, st);
        else if (N <= 32) scan_token_launch<T, 4, 8>(p, st);
        else if (N <= 64) scan_token_launch<T, 4, 16>(p, st);
        else if (N <= 128) scan_token_launch<T, 4, 32>(p, st);
        else scan_token_launch<T, 4, 64>(p, st);
    }
}

extern "C" size_t wk_scan_work(int tokens, int D, int N, int n_seq, int longest) {
    return scan_floats(scan_split(tokens, D, N, n_seq, longest), D, N) * 4;
}

extern "C" int wk_selective_scan(const warp_hip_scan_args *a, void *stream) {
    const size_t dn = (size_t)a->channels * a->states;
    scan_plan s = {0, 0, 0, 0, 0};
    if (a->starts) s = scan_split(a->tokens, a->channels, a->states, a->n_seq, a->longest);
    float *w = (float *)a->work;
    scan_p p = {a->tokens, a->n_seq, a->channels, a->states, a->groups, a->n_slots, a->softplus, s.chunk, s.chunks,
                a->starts, a->slots, a->x, a->dt, a->B, a->C, a->z, a->ldx, a->lddt, a->ldbc, a->ldz, a->ldy,
                a->A, a->D, a->dt_bias, a->state_in, a->state_out, a->y,
                w, w + 2 * s.chunks * dn, w + s.chunks * dn};
    if (a->type == WARP_HIP_F32) scan_launch<float>(p, s, (hipStream_t)stream);
    else if (a->type == WARP_HIP_BF16) scan_launch<bf16_t>(p, s, (hipStream_t)stream);
    else scan_launch<f16_t>(p, s, (hipStream_t)stream);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
