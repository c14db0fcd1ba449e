"""Plain 64-bit statements of the operators around a layer's recurrence and
experts (include/warp_hip.h, section 3), with a bound on how far f32
arithmetic may be from them, worked out along with the value.

Rows are numpy f32 arrays whose values the row type holds exactly. EPS is half
an f32 step, 2^-24; the hardware's exponential and reciprocal are within two
of those."""
import numpy as np

EPS = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}      # half a step, relative
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}   # and where steps no longer shrink (or flush)
TYPE = {"f32": 0, "bf16": 1, "f16": 2}


def pack(a, t):
    """f32 values as the row type's bits, rounded to nearest even."""
    a = np.ascontiguousarray(a, np.float32)
    if t == "f32":
        return a
    if t == "f16":
        return a.astype(np.float16)
    u = a.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r).astype(np.uint16)


def unpack(b, t):
    if t == "bf16":
        return (b.astype(np.uint32) << 16).view(np.float32)
    return b.astype(np.float32)


def rounded(a, t):
    return unpack(pack(a, t), t)


def spans(starts, n_seq, tokens):
    if starts is None:
        return [(s, s + 1) for s in range(n_seq)]
    return [(int(starts[s]), int(starts[s + 1])) for s in range(n_seq)]


def sigmoid(v):
    return np.where(v >= 0, 1 / (1 + np.exp(-np.abs(v))), np.exp(-np.abs(v)) / (1 + np.exp(-np.abs(v))))


def silu(v, err):
    """(v sigmoid(v), its bound): |silu'| <= 1.1; the sigmoid's exponential is off by
    its argument's rounding, |v| 2 EPS, and an ulp, the sum and the reciprocal by as much again."""
    y = v * sigmoid(v)
    return y, 1.1 * err + np.abs(y) * (2 * np.abs(v) + 8) * EPS


def conv(x, w, bias, sil, spans_, slots, state):
    """y, its bound (before rounding to the type), new states; rows and slots not computed are NaN."""
    T, C = x.shape
    K = w.shape[1]
    y, e = np.full((T, C), np.nan), np.zeros((T, C))
    new = np.full(state.shape, np.nan) if state is not None else None
    for s, (b, end) in enumerate(spans_):
        k = slots[s]
        if k < 0:
            continue
        h = np.zeros((K - 1, C)) if state is None else state[k].astype(np.float64)
        u = np.concatenate([h, x[b:end].astype(np.float64)])
        a = np.zeros((end - b, C)) + (0 if bias is None else bias.astype(np.float64))
        mag = np.abs(a)
        for j in range(K):
            p = w[:, j].astype(np.float64) * u[j:j + end - b]
            a, mag = a + p, mag + np.abs(p)
        err = K * EPS * mag                       # one rounding a tap, each at most EPS of the sum so far
        y[b:end], e[b:end] = silu(a, err) if sil else (a, err)
        if new is not None:
            new[k] = u[end - b:]
    return y, e, new


def scan(x, dt, A, B, C, D, z, bias, softplus, spans_, slots, h0, n_slots):
    """y, its bound, new states, their bound."""
    T, Ch = x.shape
    N = A.shape[1]
    G = B.shape[1]
    f = lambda a: a.astype(np.float64)
    x, dt, A, B, C = f(x), f(dt), f(A), f(B), f(C)
    v = dt + (0 if bias is None else f(bias))
    verr = np.abs(v) * EPS                        # the sum's rounding
    if softplus:
        d = np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))
        # the exponential's argument and ulp, the reciprocal, six steps of the series, the last sum
        derr = verr * sigmoid(v) + d * (2 * np.abs(v) + 16) * EPS
    else:
        d, derr = v, verr
    group = np.arange(Ch) // (Ch // G)
    y, ye = np.full((T, Ch), np.nan), np.zeros((T, Ch))
    new, ne = np.full((n_slots, Ch, N), np.nan), np.zeros((n_slots, Ch, N))
    for s, (b, end) in enumerate(spans_):
        k = slots[s]
        if k < 0:
            continue
        h = np.zeros((Ch, N)) if h0 is None else f(h0[k])
        e = np.zeros((Ch, N))
        for t in range(b, end):
            arg = d[t][:, None] * A
            a = np.exp(arg)
            # rate: A log2 e, the product with dt' and dt's own error; a decay may also be one exponential of
            # the sum of up to (end - b) dt', whose roundings are (end - b) EPS of it
            da = np.abs(A) * derr[t][:, None] + np.abs(arg) * (4 + end - b) * EPS + 4 * EPS
            u = (d[t] * x[t])[:, None] * B[t][group]
            du = np.abs(u) * (3 * EPS) + np.abs(x[t] * derr[t])[:, None] * np.abs(B[t][group])
            e = a * (e * (1 + da) + da * np.abs(h)) + du
            h = a * h + u
            e = e + 2 * EPS * np.abs(h) + TINY["f32"]
            c = C[t][group]
            o, oe = (c * h).sum(1), (np.abs(c) * e).sum(1) + (N + 4) * EPS * (np.abs(c * h)).sum(1)
            if D is not None:
                o, oe = o + f(D) * x[t], oe + 2 * EPS * (np.abs(f(D) * x[t]) + np.abs(o))
            if z is not None:
                g, ge = silu(f(z[t]), 0)
                o, oe = o * g, np.abs(g) * oe + np.abs(o) * ge + np.abs(o * g) * EPS
            y[t], ye[t] = o, oe
        new[k], ne[k] = h, e
    return y, ye, new, ne


def dispatch(idx, E):
    """offsets, perm (kept places only), pos"""
    flat = idx.reshape(-1)
    perm = np.concatenate([np.flatnonzero(flat == e) for e in range(E)] or [np.zeros(0, int)]).astype(np.int32)
    counts = [np.count_nonzero(flat == e) for e in range(E)]
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    pos = np.full(len(flat), -1, np.int32)
    pos[perm] = np.arange(len(perm))
    return offsets, perm, pos.reshape(idx.shape)


def combine(y, pos, w, resid):
    """out and its bound: a rounding for each row added, of at most EPS of the sum so far"""
    T, K = pos.shape
    out = np.zeros((T, y.shape[1])) if resid is None else resid.astype(np.float64)
    mag = np.abs(out)
    for k in range(K):
        live = pos[:, k] >= 0
        p = y[pos[live, k]].astype(np.float64) * (1 if w is None else w[live, k].astype(np.float64)[:, None])
        out[live] += p
        mag[live] += np.abs(p)
    return out, K * EPS * mag


def combine_backward(dout, y, pos, w):
    """dy (NaN where no pair is), dw and its bound: H products, each in a chain of sums"""
    T, K = pos.shape
    dy, dw, e = np.full(y.shape, np.nan), np.zeros((T, K)), np.zeros((T, K))
    for k in range(K):
        live = np.flatnonzero(pos[:, k] >= 0)
        at = pos[live, k]
        d = dout[live].astype(np.float64)
        dy[at] = d * (1 if w is None else w[live, k].astype(np.float64)[:, None])
        p = d * y[at].astype(np.float64)
        dw[live, k], e[live, k] = p.sum(1), y.shape[1] * EPS * np.abs(p).sum(1)
    return dy, dw, e


def check(got, ref, err, t, untouched=None):
    """got (row type's bits) against ref within err plus the type's rounding, where ref is a number; where
    it is NaN, got's bits are `untouched`."""
    live = ~np.isnan(ref)
    if untouched is not None:
        assert got[~live].tobytes() == untouched[~live].tobytes()
    g = unpack(got, t).astype(np.float64)[live]
    r, e = ref[live], np.broadcast_to(err, ref.shape)[live]
    lim = e + (np.abs(r) + e) * HALF[t] + TINY[t]
    bad = ~(np.abs(g - r) <= lim)
    assert not bad.any(), (int(bad.sum()), float(np.abs(g - r)[bad].max()), float((np.abs(g - r) / lim)[bad].max()))
