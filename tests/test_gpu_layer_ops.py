"""The short convolution, the selective scan, expert dispatch, combine and its
gradient through the C ABI against their 64-bit statements (layer_ref.py), at
the shapes and masks where they can go wrong: empty and one-row sequences,
sequences that cross the splits of the work, odd widths, strides, padding
slots, states in place, rows outside every sequence, dropped pairs, NaN where
nothing may read."""
import ctypes as C

import numpy as np
import pytest

import layer_ref as lr
from gpu_util import dev, empty, host

pytestmark = pytest.mark.gpu
NAN = float("nan")


def hip():
    import warp_amd.hip as wh
    return wh


def normal(rng, shape, t, std=1.0):
    return lr.rounded(rng.normal(size=shape) * std, t)


def strided(a, t, ld, at):
    """A device buffer of rows `ld` apart whose columns at.. are a, NaN elsewhere; and the address of a's first."""
    wide = lr.pack(np.full((a.shape[0], ld), NAN), t)
    wide[:, at:at + a.shape[1]] = lr.pack(a, t)
    b = dev(wide)
    return b, b.ptr + at * wide.itemsize


def layout(lengths, lead=0, behind=0):
    starts = np.concatenate([[lead], lead + np.cumsum(lengths)]).astype(np.int32)
    return starts, int(starts[-1]) + behind


RAGGED = [0, 5, 1, 0, 37, 2, 16, 3, 0]
LONG = [130, 1, 0, 700, 64, 3, 333]


def run_conv(rng, t, C, taps, lengths, *, single=False, silu=True, bias=True, state="in", pad=0, lead=0, behind=0, ld=0,
             poison=False):
    n = len(lengths)
    starts, T = (None, n) if single else layout(lengths, lead, behind)
    n_slots = n + 2
    slots = rng.permutation(n_slots)[:n].astype(np.int32)
    if pad:
        slots[rng.permutation(n)[:pad]] = rng.choice([-1, n_slots, -2 ** 31, 2 ** 31 - 1], size=pad)
    x, w = normal(rng, (T, C), t), (rng.normal(size=(C, taps)) * taps ** -0.5).astype(np.float32)
    b = rng.normal(size=C).astype(np.float32) if bias else None
    h = normal(rng, (n_slots, taps - 1, C), t)
    live = np.where((slots >= 0) & (slots < n_slots), slots, -1)
    y, e, new = lr.conv(x, w, b, silu, lr.spans(starts, n, T), live, h if state != "none" else h * 0)
    before_y, before_h = lr.pack(normal(rng, (T, C), t), t), lr.pack(normal(rng, h.shape, t), t)
    if poison:                                    # what is not computed is not read
        x[np.isnan(y)], h[np.setdiff1d(np.arange(n_slots), live)] = NAN, NAN
    xb, xp = strided(x, t, ld or C, (ld - C) // 2 if ld else 0)
    yb, hin = dev(before_y), dev(lr.pack(h, t))
    hout = hin if state == "inplace" else dev(before_h)
    hip().short_conv(xp, dev(w), yb, dtype=lr.TYPE[t], tokens=T, channels=C, taps=taps, n_seq=n, n_slots=n_slots,
                     starts=dev(starts) if starts is not None else None, slots=dev(slots), bias=dev(b) if bias else None,
                     state_in=None if state == "none" else hin, state_out=hout, silu=silu, ldx=ld)
    lr.check(host(yb), y, e, t, before_y)
    lr.check(host(hout), new, 0.0 * np.nan_to_num(new), t, lr.pack(h, t) if state == "inplace" else before_h)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("taps,C", [(4, 1), (4, 7), (4, 8), (4, 515), (4, 4640), (1, 33), (2, 130), (3, 64), (5, 9), (8, 257)])
def test_conv_ragged(t, taps, C):
    rng = np.random.default_rng(taps * 1000 + C)
    run_conv(rng, t, C, taps, RAGGED, state="in", pad=2, lead=3, behind=2)
    run_conv(rng, t, C, taps, LONG if C < 1000 else RAGGED, state="inplace", silu=False, ld=C + 6)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("taps,C,n", [(4, 1, 1), (4, 4640, 9), (4, 13, 70), (1, 8, 3), (3, 100, 5), (8, 30, 4)])
def test_conv_tokens(t, taps, C, n):
    rng = np.random.default_rng(taps * 77 + C + n)
    run_conv(rng, t, C, taps, [1] * n, single=True, state="inplace", pad=n // 3)
    run_conv(rng, t, C, taps, [1] * n, single=True, state="none", bias=False, ld=C + 3)


def test_conv_short_runs_at_every_offset():
    """Sequences of 1 to 9 rows one after the other meet the work's 16-row runs at every offset, in place."""
    for taps in (4, 8):
        for n in range(1, 10):
            run_conv(np.random.default_rng(n), "f32", 70, taps, [n] * 20, state="inplace")


def test_conv_no_tokens_carries_states():
    run_conv(np.random.default_rng(1), "f32", 40, 4, [0, 0, 0], state="in", pad=1)


def run_scan(rng, t, Ch, N, lengths, *, G=1, single=False, gate=True, skip=True, softplus=True, bias=True, state="in", pad=0,
             lead=0, behind=0, wide=0, longest=None, rates=None, poison=False):
    n = len(lengths)
    starts, T = (None, n) if single else layout(lengths, lead, behind)
    n_slots = n + 2
    slots = rng.permutation(n_slots)[:n].astype(np.int32)
    if pad:
        slots[rng.permutation(n)[:pad]] = rng.choice([-1, n_slots, -2 ** 31, 2 ** 31 - 1], size=pad)
    x, z = normal(rng, (T, Ch), t), normal(rng, (T, Ch), t, 2.0) if gate else None
    B, Cc = normal(rng, (T, G, N), t), normal(rng, (T, G, N), t)
    A = -(np.arange(1, N + 1) * rng.uniform(0.1, 1.2, size=(Ch, 1))).astype(np.float32) if rates is None else rates(rng, Ch, N)
    step = np.exp(rng.uniform(np.log(1e-3), np.log(0.3), size=Ch))
    if softplus:
        dt, db = normal(rng, (T, Ch), t, 0.5), np.log(np.expm1(step)).astype(np.float32)
    else:
        dt, db = lr.rounded(step * np.exp(rng.normal(size=(T, Ch)) * 0.5), t), np.zeros(Ch, np.float32) + 0.01
    db = db if bias else None
    D = rng.normal(size=Ch).astype(np.float32) if skip else None
    h = (rng.normal(size=(n_slots, Ch, N)) * 0.3).astype(np.float32)
    live = np.where((slots >= 0) & (slots < n_slots), slots, -1)
    y, ye, new, ne = lr.scan(x, dt, A, B, Cc, D, z, db, softplus, lr.spans(starts, n, T), live,
                             None if state == "none" else h, n_slots)
    before_y, before_h = lr.pack(normal(rng, (T, Ch), t), t), (rng.normal(size=h.shape)).astype(np.float32)
    if poison:
        rows = np.isnan(y).any(1)
        x[rows], dt[rows], B[rows], Cc[rows], h[np.setdiff1d(np.arange(n_slots), live)] = NAN, NAN, NAN, NAN, NAN
        if gate:
            z[rows] = NAN
    ldx, ldbc = Ch + wide, G * N + wide
    xb, xp = strided(x, t, ldx, wide // 2)
    Bb, Bp = strided(B.reshape(T, -1), t, ldbc, wide // 2)
    Cb, Cp = strided(Cc.reshape(T, -1), t, ldbc, wide // 2)
    db_, D_ = (dev(v) if v is not None else None for v in (db, D))
    zb, zp = strided(z, t, ldx, wide // 2) if gate else (None, None)
    tb, tp = strided(dt, t, ldx, wide // 2)
    yb, hin = dev(before_y), dev(h)
    hout = hin if state == "inplace" else dev(before_h)
    longest = max(lengths, default=0) if longest is None else longest
    wh = hip()
    need = 0 if single else wh.selective_scan_work(T, Ch, N, n, longest)
    work = dev(np.full(need // 4, NAN, np.float32)) if need else None
    wh.selective_scan(xp, tp, dev(A), Bp, Cp, yb, dtype=lr.TYPE[t], tokens=T, channels=Ch, n_state=N, groups=G, n_seq=n,
                      n_slots=n_slots, starts=dev(starts) if starts is not None else None, slots=dev(slots),
                      state_in=None if state == "none" else hin, state_out=hout, D=D_, z=zp, dt_bias=db_, softplus=softplus,
                      ldx=ldx, lddt=ldx, ldz=ldx, ldbc=ldbc, longest=longest, work=work, work_bytes=need)
    lr.check(host(yb), y, ye, t, before_y)
    lr.check(host(hout), new, ne, "f32", h if state == "inplace" else before_h)
    return need


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Ch,N,G", [(1, 1, 1), (64, 16, 1), (130, 16, 2), (96, 5, 3), (40, 4, 1), (33, 8, 1), (30, 17, 2),
                                    (20, 32, 1), (72, 50, 4), (9, 64, 3), (16, 100, 1), (10, 128, 2), (6, 200, 1), (5, 256, 1)])
def test_scan_ragged(t, Ch, N, G):
    rng = np.random.default_rng(Ch * 1000 + N)
    run_scan(rng, t, Ch, N, RAGGED, G=G, pad=2, lead=3, behind=2, wide=6)
    run_scan(rng, t, Ch, N, RAGGED, G=G, state="inplace", gate=False, skip=False, softplus=False)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("Ch,N,G", [(64, 16, 1), (70, 3, 2), (130, 24, 1), (20, 64, 2), (12, 130, 1)])
def test_scan_across_chunks(t, Ch, N, G):
    """Batches whose sequences are split over chunks of rows, several in a chunk and one over many; states in
    place, where a sequence's first state is overwritten while others still run."""
    rng = np.random.default_rng(Ch + N)
    assert run_scan(rng, t, Ch, N, LONG, G=G, state="inplace", pad=1, longest=0) > 0
    assert run_scan(rng, t, Ch, N, [640], G=G, state="in", lead=7, behind=9) > 0
    assert run_scan(rng, t, Ch, N, [500, 200, 0], G=G, state="none", longest=0, bias=False) > 0


def test_scan_rates_and_steps_at_their_ends():
    """Rates of zero and of -1e4 (a decay of 1, and of exactly 0), over chunks."""
    def rates(rng, Ch, N):
        A = -rng.uniform(0.1, 2, size=(Ch, N)).astype(np.float32)
        A[:, 0], A[:, 1] = 0.0, -1e4
        return A
    rng = np.random.default_rng(5)
    run_scan(rng, "f32", 64, 16, [400, 3, 0, 90], rates=rates, state="inplace")
    run_scan(rng, "f32", 64, 16, [1] * 9, single=True, rates=rates, state="inplace")


@pytest.mark.parametrize("T", [160, 640])
def test_scan_states_that_grow(T):
    """Without a softplus a state may grow: by up to e^96 in the rows 16 .. 31, more than f32 can say, and back in the next
    16. A state of zero stays zero meanwhile, and a small one is what it is row by row, however the rows are split."""
    Ch, N, wh = 64, 16, hip()
    rng = np.random.default_rng(T)
    x, B, Cc = normal(rng, (T, Ch), "f32"), normal(rng, (T, 1, N), "f32"), normal(rng, (T, 1, N), "f32")
    x[:64] = 0
    dt = lr.rounded(rng.uniform(0.001, 0.01, size=(T, Ch)), "f32")
    dt[16:32], dt[32:48] = 6, -6
    A = rng.uniform(0.9, 1, size=(Ch, N)).astype(np.float32)
    A[:, 0] = 1
    h = np.zeros((1, Ch, N), np.float32)
    h[0, Ch // 2:] = 1e-30
    ref = lambda b, h: lr.scan(x[b:], dt[b:], A, B[b:], Cc[b:], None, None, None, False, [(0, T - b)], [0], h, 1)
    y, ye, new, ne = ref(0, h)
    # (of a zero state nothing is lost below f32's least number: the same from row 64 on)
    zero = ref(64, None)
    y[64:, :Ch // 2], ye[64:, :Ch // 2] = zero[0][:, :Ch // 2], zero[1][:, :Ch // 2]
    new[:, :Ch // 2], ne[:, :Ch // 2] = zero[2][:, :Ch // 2], zero[3][:, :Ch // 2]
    ye[:64, :Ch // 2] = 0
    need = wh.selective_scan_work(T, Ch, N, 1, T)
    assert need > 0 and np.isfinite(y).all()
    yb, hb = dev(np.full((T, Ch), NAN, np.float32)), dev(h)
    wh.selective_scan(dev(x), dev(dt), dev(A), dev(B), dev(Cc), yb, dtype=lr.TYPE["f32"], tokens=T, channels=Ch, n_state=N,
                      n_seq=1, n_slots=1, starts=dev(np.array([0, T], np.int32)), state_in=hb, state_out=hb, softplus=False,
                      longest=T, work=dev(np.full(need // 4, NAN, np.float32)), work_bytes=need)
    lr.check(host(yb), y, ye, "f32")
    lr.check(host(hb), new, ne, "f32")


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Ch,N,G,n", [(1, 1, 1, 1), (4608, 16, 1, 3), (130, 16, 2, 70), (33, 4, 1, 5), (20, 8, 2, 3), (30, 24, 1, 4),
                                      (12, 64, 3, 2), (9, 128, 1, 3), (5, 256, 1, 2), (21, 5, 7, 9), (14, 23, 2, 3), (6, 33, 1, 2),
                                      (5, 201, 1, 3)])
def test_scan_tokens(t, Ch, N, G, n):
    rng = np.random.default_rng(Ch * 10 + N + n)
    run_scan(rng, t, Ch, N, [1] * n, G=G, single=True, state="inplace", pad=n // 3)
    run_scan(rng, t, Ch, N, [1] * n, G=G, single=True, state="none", gate=False, softplus=False, wide=5)


def run_dispatch(idx, E, H, t, ldx=0, ldxs=0, rows=True):
    rng = np.random.default_rng(E + H)
    T, K = idx.shape
    offsets, perm, pos = lr.dispatch(idx, E)
    x = normal(rng, (T, H), t)
    x[::3] = NAN                                  # copied as they are
    xb, xp = strided(x, t, ldx or H, 0)
    before = np.arange(T * K, dtype=np.int32) + 1000
    old = lr.pack(np.zeros((T * K, ldxs or H)), t)
    ob, pb, qb, sb = dev(np.full(E + 1, -7, np.int32)), dev(before), dev(before), dev(old)
    wh = hip()
    n = wh.expert_dispatch_work(T, K, E)
    kw = dict(x=xp, xs=sb, dtype=lr.TYPE[t], hidden=H, ldx=ldx, ldxs=ldxs) if rows else {}
    wh.expert_dispatch(dev(idx) if T else None, ob, pb, qb, tokens=T, top_k=K, n_experts=E, work=empty(max(n, 4), np.uint8),
                       work_bytes=n, **kw)
    assert np.array_equal(host(ob), offsets)
    assert np.array_equal(host(qb).reshape(T, K), pos)
    got = host(pb)
    assert np.array_equal(got[:len(perm)], perm) and np.array_equal(got[len(perm):], before[len(perm):])
    want = old.copy()
    if rows:
        want[:len(perm), :H] = lr.pack(x, t)[perm // K]
    assert np.array_equal(host(sb).view(np.uint8), want.view(np.uint8))


@pytest.mark.parametrize("T,K,E,H", [(1, 1, 1, 1), (1, 8, 256, 2304), (32, 16, 384, 513), (7, 3, 5, 64), (300, 8, 896, 9),
                                     (255, 8, 17, 8), (256, 8, 256, 7), (257, 8, 256, 40), (2049, 2, 2048, 12), (5000, 16, 300, 3),
                                     (1500, 64, 100, 2), (4096, 1, 3, 5)])
def test_dispatch(T, K, E, H):
    rng = np.random.default_rng(T + K)
    idx = rng.integers(0, E, size=(T, K)).astype(np.int32)
    run_dispatch(idx, E, H, "bf16")
    idx[rng.random((T, K)) < 0.3] = -1
    idx[rng.random((T, K)) < 0.1] = E
    idx[rng.random((T, K)) < 0.05] = -2 ** 31
    run_dispatch(idx, E, H, "f32", ldx=H + 3, ldxs=H + 5)
    run_dispatch(np.minimum(idx, 0), E, H, "f16")        # one expert, and dropped ones
    run_dispatch(np.full((T, K), E, np.int32), E, H, "f16", rows=False)


def test_dispatch_of_nothing():
    run_dispatch(np.zeros((0, 4), np.int32), 9, 8, "f32", rows=False)


def places(rng, T, K, drop):
    """Distinct places of T K rows, some pairs without one."""
    pos = rng.permutation(T * K).astype(np.int32).reshape(T, K)
    pos[rng.random((T, K)) < drop] = -1
    return pos


SHAPES = [(1, 1, 1), (7, 8, 2304), (3, 16, 7168), (50, 2, 513), (33, 64, 8), (129, 4, 1000), (5, 3, 4097)]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,K,H", SHAPES)
def test_combine(t, T, K, H):
    rng = np.random.default_rng(T * 100 + H)
    for drop, weights, residual, wide in ((0.0, True, True, 0), (0.3, True, False, 5), (0.2, False, True, 0), (1.0, False, False, 3)):
        pos = places(rng, T, K, drop)
        y, w = normal(rng, (T * K, H), t), rng.normal(size=(T, K)).astype(np.float32)
        w[pos < 0] = NAN
        y[np.setdiff1d(np.arange(T * K), pos)] = NAN     # rows that no pair names
        r = normal(rng, (T, H), t) if residual else None
        w = w if weights else None
        ref, err = lr.combine(y, pos, w, r)
        bad = np.where(pos < 0, rng.choice([-1, T * K, -2 ** 31, 2 ** 31 - 1], size=pos.shape), pos).astype(np.int32)
        yb, yp = strided(y, t, H + wide, wide // 2)
        out = dev(lr.pack(r, t)) if residual else dev(lr.pack(np.full((T, H), NAN), t))
        hip().expert_combine(yp, dev(bad), out, dtype=lr.TYPE[t], tokens=T, top_k=K, hidden=H, ldy=H + wide,
                             w=dev(w) if weights else None, resid=out if residual else None)
        lr.check(host(out), ref, err, t)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,K,H", SHAPES)
def test_combine_backward(t, T, K, H):
    rng = np.random.default_rng(T * 100 + H + 1)
    for drop, weights, wide, inplace in ((0.0, True, 0, False), (0.3, True, 5, True), (0.2, False, 0, False), (1.0, True, 3, False)):
        pos = places(rng, T, K, drop)
        y, w = normal(rng, (T * K, H), t), rng.normal(size=(T, K)).astype(np.float32)
        y[np.setdiff1d(np.arange(T * K), pos)] = NAN
        d = normal(rng, (T, H), t)
        dy, dw, err = lr.combine_backward(d, y, pos, w if weights else None)
        yb, yp = strided(y, t, H + wide, 0)
        db, dp = strided(d, t, H + wide, wide // 2)
        before = lr.pack(y if inplace else np.ones(y.shape), t)
        gb, gw = yb if inplace else dev(before), dev(np.full((T, K), NAN, np.float32))
        kw = dict(dtype=lr.TYPE[t], tokens=T, top_k=K, hidden=H, w=dev(w) if weights else None, ldd=H + wide)
        hip().expert_combine_backward(dp, yp, dev(pos), gb, gw, ldy=H + wide, lddy=H + wide if inplace else 0, **kw)
        got = host(gb).reshape(T * K, -1)[:, :H]
        lr.check(got, dy, np.abs(np.nan_to_num(dy)) * lr.EPS, t, before)
        lr.check(host(gw), dw, err, "f32")
        if not inplace:                           # either alone
            g2, w2 = dev(before), dev(np.full((T, K), NAN, np.float32))
            hip().expert_combine_backward(dp, None, dev(pos), g2, None, **kw)
            hip().expert_combine_backward(dp, yp, dev(pos), None, w2, ldy=H + wide, **kw)
            assert np.array_equal(host(g2).view(np.uint8), host(gb).view(np.uint8)) and np.array_equal(host(w2), host(gw))


def test_combine_gradient_against_differences():
    """The gradients of L = <out, c> are what out's change gives: L is linear in y and in w, so a step of 1
    in one element changes it by that element's gradient."""
    rng = np.random.default_rng(9)
    T, K, H = 4, 3, 37
    pos = places(rng, T, K, 0.2)
    y, w, c = (rng.normal(size=s).astype(np.float32) for s in ((T * K, H), (T, K), (T, H)))
    kw = dict(dtype=0, tokens=T, top_k=K, hidden=H)

    def loss(y, w):
        out = empty((T, H))
        hip().expert_combine(dev(y), dev(pos), out, w=dev(w), **kw)
        return float((host(out).astype(np.float64) * c).sum())
    dy, dw = dev(np.zeros((T * K, H), np.float32)), empty((T, K))
    hip().expert_combine_backward(dev(c), dev(y), dev(pos), dy, dw, w=dev(w), **kw)
    dy, dw, base = host(dy), host(dw), loss(y, w)
    # an element of out is a sum of K products of this size, each rounded to EPS of it; two losses and a step
    lim = 8 * K * lr.EPS * (np.abs(y).max() + 1) * (np.abs(w).max() + 1) * np.abs(c).sum()
    for p, h in ((0, 0), (5, 36), (11, 7)):
        y2 = y.copy()
        y2[p, h] += 1
        assert abs(loss(y2, w) - base - dy[p, h]) <= lim
    for t, k in ((0, 0), (3, 2), (1, 1)):
        w2 = w.copy()
        w2[t, k] += 1
        assert abs(loss(y, w2) - base - dw[t, k]) <= lim


def test_more_rows_than_a_grid_takes_at_once():
    """Blocks that take further rows, sequences, tokens and pairs in turn."""
    rng = np.random.default_rng(8)
    run_conv(rng, "f32", 5, 2, [1_000_000, 0, 3, 700_000], state="inplace", silu=False)
    run_conv(rng, "f32", 5, 4, [1] * 9000, single=True, state="inplace", pad=3000)
    run_scan(rng, "f32", 2, 4, [1] * 20000, single=True, state="inplace", pad=3000)
    run_scan(rng, "f32", 2, 4, [1] * 33000 + [0] * 3000 + [2] * 500, state="inplace", pad=3000)


@pytest.mark.parametrize("T,K,E,H", [(300000, 2, 7, 4), (20, 70, 90, 33), (40, 130, 900, 9), (1000, 8, 256, 2070)])
def test_dispatch_and_combine_of_many_pairs(T, K, E, H):
    rng = np.random.default_rng(T + K)
    idx = rng.integers(-1, E, size=(T, K)).astype(np.int32)
    run_dispatch(idx, E, H, "bf16")
    pos, y, w, r, d = places(rng, T, K, 0.1), normal(rng, (T * K, H), "f16"), rng.normal(size=(T, K)).astype(np.float32), normal(
        rng, (T, H), "f16"), normal(rng, (T, H), "f16")
    ref, err = lr.combine(y, pos, w, r)
    out, pb, wb, yb = empty((T, H), np.float16), dev(pos), dev(w), dev(lr.pack(y, "f16"))
    kw = dict(dtype=lr.TYPE["f16"], tokens=T, top_k=K, hidden=H, w=wb)
    hip().expert_combine(yb, pb, out, resid=dev(lr.pack(r, "f16")), **kw)
    lr.check(host(out), ref, err, "f16")
    dy, dw, err = lr.combine_backward(d, y, pos, w)
    before = np.ones((T * K, H), np.float16)
    gb, gw = dev(before), empty((T, K))
    hip().expert_combine_backward(dev(lr.pack(d, "f16")), yb, pb, gb, gw, **kw)
    lr.check(host(gb), dy, np.abs(np.nan_to_num(dy)) * lr.EPS, "f16", before)
    lr.check(host(gw), dw, err, "f32")


def test_rows_that_are_not_computed_may_hold_anything():
    """NaN in padding rows, in rows outside every sequence and in states of no sequence."""
    rng = np.random.default_rng(12)
    for lengths in (RAGGED, LONG):
        run_conv(rng, "bf16", 70, 4, lengths, state="inplace", pad=3, lead=5, behind=4, poison=True)
        run_scan(rng, "bf16", 70, 16, lengths, state="inplace", pad=3, lead=5, behind=4, poison=True, longest=0)
        run_scan(rng, "f32", 33, 5, lengths, state="in", pad=3, lead=5, behind=4, poison=True)
    run_conv(rng, "f32", 70, 4, [1] * 12, single=True, state="inplace", pad=5, poison=True)
    run_scan(rng, "f32", 70, 16, [1] * 12, single=True, state="inplace", pad=5, poison=True)


@pytest.mark.parametrize("N", [5, 16])
@pytest.mark.parametrize("single", [False, True])
def test_an_infinity_stays_in_its_channel_and_sequence(N, single):
    """One infinite input, then one that is no number: every output and state of other channels, of other
    sequences and of the rows before it is bit for bit what it is without."""
    rng = np.random.default_rng(N)
    wh, Ch, lengths = hip(), 37, [1] * 6 if single else [30, 0, 400, 21]
    starts, T = (None, 6) if single else layout(lengths)
    n = len(lengths)
    x, dt, z = (normal(rng, (T, Ch), "f32", s) for s in (1, 0.3, 1))
    BC, w = [normal(rng, (T, N), "f32") for _ in range(2)], rng.normal(size=(Ch, 4)).astype(np.float32)
    A = -rng.uniform(0.1, 3, size=(Ch, N)).astype(np.float32)
    st = dev(starts) if starts is not None else None
    at, seq, c = (2, 2, 11) if single else (100, 2, 11)

    def run(v):
        x2 = x.copy()
        x2[at, c] = v
        rows = dict(dtype=0, tokens=T, channels=Ch, n_seq=n, n_slots=n, starts=st)
        u, y, hist, h = empty((T, Ch)), empty((T, Ch)), empty((n, 3, Ch)), empty((n, Ch, N))
        xb = dev(x2)
        wh.short_conv(xb, dev(w), u, taps=4, state_out=hist, **rows)
        need = 0 if single else wh.selective_scan_work(T, Ch, N, n)
        wh.selective_scan(xb, dev(dt), dev(A), dev(BC[0]), dev(BC[1]), y, n_state=N, z=dev(z), state_out=h,
                          work=empty(max(need, 16), np.uint8), work_bytes=need, **rows)
        return host(u), host(y), host(hist), host(h)
    want = run(x[at, c])
    end = at + 1 if single else int(starts[seq + 1])
    for v in (np.inf, -np.inf, NAN):
        for k, (got, ref) in enumerate(zip(run(v), want)):
            same = got.view(np.uint32) == ref.view(np.uint32)
            touched = np.zeros(same.shape, bool)
            if k < 2:
                touched[at:end, c] = True
            else:
                touched[(seq, slice(None), c) if k == 2 else (seq, c)] = True
            assert (same | touched).all()
            assert k == 0 or k == 2 or not np.isfinite(got[at, c] if k == 1 else got[seq, c]).any()
