/* The operators around a layer's recurrence and experts: what include/warp_hip.h
 * section 3 promises of their arguments, checked before anything is queued.
 * The kernels are in conv.hip, scan.hip and dispatch.hip. */
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#include "warp_hip.h"
#include "warp_internal.h"

#define CONV_MAX_TAPS 8
#define SCAN_MAX_STATES 256
#define MAX_CHANNELS (1 << 24)
#define MAX_ROWS (1 << 30)       /* what the kernels count in ints, with room to step over the end */
#define DISPATCH_MAX_EXPERTS 2048

static int type_size(int type)
{
    return type == WARP_HIP_F32 ? 4 : type == WARP_HIP_BF16 || type == WARP_HIP_F16 ? 2 : 0;
}

static int off(const void *p, size_t to)
{
    return ((uintptr_t)p & (to - 1)) != 0;
}

/* The work goes to the stream's device, whichever is current: *back is the
 * device to return to, or -1. */
static int enter(void *stream, int *back)
{
    int now, want;
    *back = -1;
    if (!stream) return 0;
    if (hipGetDevice(&now) != hipSuccess || hipStreamGetDevice((hipStream_t)stream, &want) != hipSuccess) return -1;
    if (want == now) return 0;
    if (hipSetDevice(want) != hipSuccess) return -1;
    *back = now;
    return 0;
}

static int leave(int rc, int back)
{
    if (back >= 0 && hipSetDevice(back) != hipSuccess) rc = -1;
    return rc ? WARP_HIP_E_DEVICE : 0;
}

#define QUEUE(call)                                        \
    do {                                                   \
        int back_;                                         \
        if (enter(stream, &back_)) return WARP_HIP_E_DEVICE; \
        return leave(call, back_);                         \
    } while (0)

/* A row stride: the width if none is given; 0 if it is shorter than that */
static size_t stride(size_t ld, size_t width)
{
    return ld == 0 ? width : ld < width ? 0 : ld;
}

/* The sequences' part of the convolution's and the scan's arguments. */
static int sequences_ok(int tokens, int n_seq, int channels, const int *starts, const int *slots, int n_slots)
{
    if (tokens < 0 || n_seq < 0 || channels < 1 || n_slots < 0 || off(starts, 4) || off(slots, 4)) return 0;
    if (tokens > MAX_ROWS || n_seq > MAX_ROWS || channels > MAX_CHANNELS) return 0;
    if (!starts && n_seq != tokens) return 0;
    return slots || n_slots >= n_seq;
}

int warp_hip_short_conv(const warp_hip_conv_args *args, void *stream)
{
    if (!args) return WARP_HIP_E_ARG;
    warp_hip_conv_args a = *args;
    const int es = type_size(a.type);
    if (!es || a.taps < 1 || a.taps > CONV_MAX_TAPS) return WARP_HIP_E_ARG;
    if (!sequences_ok(a.tokens, a.n_seq, a.channels, a.starts, a.slots, a.n_slots)) return WARP_HIP_E_ARG;
    a.ldx = stride(a.ldx, (size_t)a.channels);
    a.ldy = stride(a.ldy, (size_t)a.channels);
    if (!a.ldx || !a.ldy || !a.w || off(a.w, 4) || off(a.bias, 4)) return WARP_HIP_E_ARG;
    if (off(a.x, es) || off(a.y, es) || off(a.state_in, es) || off(a.state_out, es)) return WARP_HIP_E_ARG;
    if (a.tokens && (!a.x || !a.y || a.x == a.y)) return WARP_HIP_E_ARG;
    if (a.n_seq == 0) return 0;
    QUEUE(wk_short_conv(&a, stream));
}

size_t warp_hip_selective_scan_work(int tokens, int channels, int states, int n_seq, int longest)
{
    if (tokens < 1 || channels < 1 || states < 1 || states > SCAN_MAX_STATES || n_seq < 1) return 0;
    if (tokens > MAX_ROWS || channels > MAX_CHANNELS) return 0;
    return wk_scan_work(tokens, channels, states, n_seq, longest);
}

int warp_hip_selective_scan(const warp_hip_scan_args *args, void *stream)
{
    if (!args) return WARP_HIP_E_ARG;
    warp_hip_scan_args a = *args;
    const int es = type_size(a.type);
    if (!es || a.states < 1 || a.states > SCAN_MAX_STATES || a.groups < 1) return WARP_HIP_E_ARG;
    if (!sequences_ok(a.tokens, a.n_seq, a.channels, a.starts, a.slots, a.n_slots)) return WARP_HIP_E_ARG;
    if (a.channels % a.groups || a.longest < 0) return WARP_HIP_E_ARG;
    a.ldx = stride(a.ldx, (size_t)a.channels);
    a.lddt = stride(a.lddt, (size_t)a.channels);
    a.ldz = stride(a.ldz, (size_t)a.channels);
    a.ldy = stride(a.ldy, (size_t)a.channels);
    a.ldbc = stride(a.ldbc, (size_t)a.groups * a.states);
    if (!a.ldx || !a.lddt || !a.ldz || !a.ldy || !a.ldbc) return WARP_HIP_E_ARG;
    if (!a.A || off(a.A, 4) || off(a.D, 4) || off(a.dt_bias, 4) || off(a.state_in, 4) || off(a.state_out, 4))
        return WARP_HIP_E_ARG;
    if (off(a.x, es) || off(a.dt, es) || off(a.B, es) || off(a.C, es) || off(a.z, es) || off(a.y, es))
        return WARP_HIP_E_ARG;
    if (a.tokens && (!a.x || !a.dt || !a.B || !a.C || !a.y)) return WARP_HIP_E_ARG;
    if (a.n_seq == 0) return 0;
    if (a.starts && a.tokens) {
        const size_t need = wk_scan_work(a.tokens, a.channels, a.states, a.n_seq, a.longest);
        if (need && (!a.work || a.work_bytes < need || off(a.work, 16))) return WARP_HIP_E_ARG;
    }
    QUEUE(wk_selective_scan(&a, stream));
}

/* tokens * top_k pairs, as the kernels count them */
static int pairs_ok(int tokens, int top_k)
{
    return tokens >= 0 && top_k >= 1 && (int64_t)tokens * top_k <= MAX_ROWS;
}

size_t warp_hip_expert_dispatch_work(int tokens, int top_k, int n_experts)
{
    if (!pairs_ok(tokens, top_k) || n_experts < 1 || n_experts > DISPATCH_MAX_EXPERTS) return 0;
    return wk_dispatch_work(tokens, top_k, n_experts);
}

int warp_hip_expert_dispatch(const warp_hip_dispatch_args *args, void *stream)
{
    if (!args) return WARP_HIP_E_ARG;
    warp_hip_dispatch_args a = *args;
    if (!pairs_ok(a.tokens, a.top_k) || a.n_experts < 1 || a.n_experts > DISPATCH_MAX_EXPERTS) return WARP_HIP_E_ARG;
    if (!a.offsets || off(a.offsets, 4) || off(a.idx, 4) || off(a.perm, 4) || off(a.pos, 4)) return WARP_HIP_E_ARG;
    if (a.tokens && (!a.idx || !a.perm || !a.pos)) return WARP_HIP_E_ARG;
    if (!a.x != !a.xs) return WARP_HIP_E_ARG;
    if (a.x) {
        const int es = type_size(a.type);
        if (!es || a.hidden < 1 || a.hidden > MAX_CHANNELS || off(a.x, es) || off(a.xs, es)) return WARP_HIP_E_ARG;
        a.ldx = stride(a.ldx, (size_t)a.hidden);
        a.ldxs = stride(a.ldxs, (size_t)a.hidden);
        if (!a.ldx || !a.ldxs) return WARP_HIP_E_ARG;
    }
    const size_t need = wk_dispatch_work(a.tokens, a.top_k, a.n_experts);
    if (need && (!a.work || a.work_bytes < need || off(a.work, 4))) return WARP_HIP_E_ARG;
    QUEUE(wk_expert_dispatch(&a, stream));
}

int warp_hip_expert_combine(const warp_hip_combine_args *args, void *stream)
{
    if (!args) return WARP_HIP_E_ARG;
    warp_hip_combine_args a = *args;
    const int es = type_size(a.type);
    if (!es || !pairs_ok(a.tokens, a.top_k) || a.hidden < 1 || a.hidden > MAX_CHANNELS) return WARP_HIP_E_ARG;
    a.ldy = stride(a.ldy, (size_t)a.hidden);
    a.ldr = stride(a.ldr, (size_t)a.hidden);
    a.ldo = stride(a.ldo, (size_t)a.hidden);
    if (!a.ldy || !a.ldr || !a.ldo) return WARP_HIP_E_ARG;
    if (off(a.y, es) || off(a.resid, es) || off(a.out, es) || off(a.pos, 4) || off(a.w, 4)) return WARP_HIP_E_ARG;
    if (a.tokens == 0) return 0;
    if (!a.y || !a.pos || !a.out || a.out == a.y || (a.out == a.resid && a.ldo != a.ldr)) return WARP_HIP_E_ARG;
    QUEUE(wk_expert_combine(&a, stream));
}

int warp_hip_expert_combine_backward(const warp_hip_combine_back_args *args, void *stream)
{
    if (!args) return WARP_HIP_E_ARG;
    warp_hip_combine_back_args a = *args;
    const int es = type_size(a.type);
    if (!es || !pairs_ok(a.tokens, a.top_k) || a.hidden < 1 || a.hidden > MAX_CHANNELS) return WARP_HIP_E_ARG;
    a.ldd = stride(a.ldd, (size_t)a.hidden);
    a.ldy = stride(a.ldy, (size_t)a.hidden);
    a.lddy = stride(a.lddy, (size_t)a.hidden);
    if (!a.ldd || !a.ldy || !a.lddy) return WARP_HIP_E_ARG;
    if (off(a.dout, es) || off(a.y, es) || off(a.dy, es) || off(a.pos, 4) || off(a.w, 4) || off(a.dw, 4))
        return WARP_HIP_E_ARG;
    if (!a.dy && !a.dw) return WARP_HIP_E_ARG;
    if (a.tokens == 0) return 0;
    if (!a.dout || !a.pos || (a.dw && !a.y) || a.dy == a.dout || (a.dy && a.dy == a.y && a.lddy != a.ldy))
        return WARP_HIP_E_ARG;
    QUEUE(wk_expert_combine_backward(&a, stream));
}
