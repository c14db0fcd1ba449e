"""The operators around a layer's recurrence and experts as a program runs
them: in a captured graph that is replayed, on two streams at once, a prompt
and then its tokens on the same states, many sequences in a batch, offsets
past 32 bits, and a layer of them together with the framework's router and
experts."""
import ctypes as C

import numpy as np
import pytest

import container as ct
import layer_ref as lr
from gpu_util import BALANCED, dev, empty, host, open_ctx
from test_gpu_layer_ops import hip, layout, normal, run_conv, run_scan

pytestmark = pytest.mark.gpu


class Stream:
    """A stream of the library's runtime (default priority)."""

    def __init__(self):
        from warp_amd.device import check, rt
        s = C.c_void_p()
        check(rt().hipStreamCreate(C.byref(s)), "hipStreamCreate")
        self.s = s.value

    def wait(self):
        from warp_amd.device import check, rt
        check(rt().hipStreamSynchronize(self.s), "hipStreamSynchronize")

    def close(self):
        from warp_amd.device import rt
        rt().hipStreamDestroy(C.c_void_p(self.s))


class Layer:
    """Buffers of one layer's operators for a packed batch, bf16 rows: convolution, scan, dispatch, combine and
    the combine's gradient, each on its predecessor's output (the experts are the identity)."""
    Ch, N, K, E, TAPS = 192, 16, 4, 24, 4

    def __init__(self, rng, lengths, single=False):
        self.n, self.single = len(lengths), single
        starts, self.T = (None, self.n) if single else layout(lengths)
        self.starts = dev(starts) if starts is not None else None
        self.w = dev((rng.normal(size=(self.Ch, self.TAPS)) * 0.5).astype(np.float32))
        self.A = dev(-(np.arange(1, self.N + 1) * rng.uniform(0.5, 1, size=(self.Ch, 1))).astype(np.float32))
        self.D = dev(rng.normal(size=self.Ch).astype(np.float32))
        self.x, self.dt, self.B, self.C = (empty((self.T, w), np.uint16) for w in (self.Ch, self.Ch, self.N, self.N))
        self.idx, self.wt = empty((self.T, self.K), np.int32), empty((self.T, self.K))
        self.hist = empty((self.n, self.TAPS - 1, self.Ch), np.uint16)
        self.h, self.h2, self.hist2 = empty((self.n, self.Ch, self.N)), empty((self.n, self.Ch, self.N)), empty(
            (self.n, self.TAPS - 1, self.Ch), np.uint16)
        self.u, self.y, self.out, self.dx = (empty((self.T, self.Ch), np.uint16) for _ in range(4))
        P = self.T * self.K
        self.offsets, self.perm, self.pos = empty(self.E + 1, np.int32), empty(P, np.int32), empty(P, np.int32)
        self.xs, self.dy, self.dw = empty((P, self.Ch), np.uint16), empty((P, self.Ch), np.uint16), empty((self.T, self.K))
        wh = hip()
        self.ns = 0 if single else wh.selective_scan_work(self.T, self.Ch, self.N, self.n)
        self.nd = wh.expert_dispatch_work(self.T, self.K, self.E)
        self.ws, self.wd = empty(max(self.ns, 16), np.uint8), empty(max(self.nd, 16), np.uint8)

    def inputs(self, seed):
        rng = np.random.default_rng(seed)
        for b in (self.x, self.dt, self.B, self.C, self.hist):
            b.upload(lr.pack(rng.normal(size=b.shape) * (0.05 if b is self.dt else 1), "bf16"))
        self.idx.upload(rng.integers(-1, self.E, size=self.idx.shape).astype(np.int32))
        self.wt.upload(rng.uniform(0.1, 1, size=self.wt.shape).astype(np.float32))
        self.h.upload(rng.normal(size=self.h.shape).astype(np.float32))
        for b in (self.perm, self.xs, self.dy):
            b.upload(np.zeros(b.shape, b.dtype))

    def run(self, stream):
        wh = hip()
        rows = dict(dtype=wh.BF16, tokens=self.T, channels=self.Ch, n_seq=self.n, n_slots=self.n, starts=self.starts,
                    stream=stream)
        moe = dict(dtype=wh.BF16, tokens=self.T, top_k=self.K, hidden=self.Ch, stream=stream)
        wh.short_conv(self.x, self.w, self.u, taps=self.TAPS, state_in=self.hist, state_out=self.hist2, **rows)
        wh.selective_scan(self.u, self.dt, self.A, self.B, self.C, self.y, n_state=self.N, D=self.D, z=self.x,
                          state_in=self.h, state_out=self.h2, work=self.ws, work_bytes=self.ns, **rows)
        wh.expert_dispatch(self.idx, self.offsets, self.perm, self.pos, n_experts=self.E, x=self.y, xs=self.xs,
                           work=self.wd, work_bytes=self.nd, **moe)
        wh.expert_combine(self.xs, self.pos, self.out, w=self.wt, resid=self.x, **moe)
        wh.expert_combine_backward(self.out, self.xs, self.pos, self.dy, self.dw, w=self.wt, **moe)
        wh.expert_combine(self.dy, self.pos, self.dx, **moe)

    def results(self):
        return [host(b).tobytes() for b in (self.u, self.hist2, self.y, self.h2, self.offsets, self.perm, self.pos, self.xs,
                                            self.out, self.dy, self.dw, self.dx)]


LENGTHS = [300, 0, 45, 700, 1, 150]


@pytest.mark.parametrize("single", [False, True])
def test_graph_replays_equal_eager(single):
    """A layer captured once and replayed on new inputs, with the same layer's eager calls and synchronisations
    between the replays: bit for bit what the eager calls give (which so are the same each time, too)."""
    from warp_amd.device import Graph, synchronize
    layer = Layer(np.random.default_rng(1), [1] * 9 if single else LENGTHS, single)
    st = Stream()
    eager = []
    for seed in range(3):
        layer.inputs(seed)
        synchronize()
        layer.run(st.s)
        st.wait()
        eager.append(layer.results())
    g = Graph(st.s, lambda: layer.run(st.s))
    try:
        for rep in range(6):
            layer.inputs(rep % 3)
            synchronize()
            g.launch()
            st.wait()
            assert layer.results() == eager[rep % 3], rep
            layer.inputs((rep + 1) % 3)
            synchronize()
            layer.run(st.s)
            st.wait()
            assert layer.results() == eager[(rep + 1) % 3], rep
    finally:
        g.free()
        st.close()


def test_two_streams_at_once():
    """Two layers on two streams, each with its own workspaces, queued without a wait: as one after the other."""
    from warp_amd.device import synchronize
    layers, streams = [Layer(np.random.default_rng(k), LENGTHS) for k in range(2)], [Stream(), Stream()]
    want = []
    for k, layer in enumerate(layers):
        layer.inputs(k)
        synchronize()
        layer.run(None)
        synchronize()
        want.append(layer.results())
        layer.inputs(k)
    synchronize()
    for _ in range(4):
        for layer, st in zip(layers, streams):
            layer.run(st.s)
    for st in streams:
        st.wait()
    assert [layer.results() for layer in layers] == want
    for st in streams:
        st.close()


@pytest.mark.parametrize("n", [63, 64, 65, 300, 5000])
def test_many_sequences(n):
    """As many sequences as a wave loads at once, and more than that, short and empty ones among them."""
    rng = np.random.default_rng(n)
    lengths = rng.integers(0, 4, size=n) * (rng.random(n) < 0.7)
    lengths[n // 2] = 150
    lengths = [int(v) for v in lengths]
    run_conv(rng, "f32", 12, 4, lengths, state="inplace", pad=n // 10, lead=2, behind=3)
    run_scan(rng, "f32", 6, 4, lengths, state="inplace", pad=n // 10, lead=2, behind=3)
    run_scan(rng, "f32", 6, 4, lengths, state="inplace", longest=0)


@pytest.mark.parametrize("longest", [0, 1, 40, 10 ** 9])
def test_results_hold_for_any_longest(longest):
    rng = np.random.default_rng(3)
    run_scan(rng, "f32", 70, 16, [200, 3, 90, 0, 41], state="inplace", longest=longest)
    run_scan(rng, "f32", 70, 16, [1] * 200, state="inplace", longest=longest)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_a_prompt_in_pieces_and_then_its_tokens(t):
    """Two sequences' rows in one call, in three, and token by token, on states that stay in their slots: the
    convolution's rows and states bit for bit, the scan's within its bound of the 64-bit statement of the whole."""
    rng = np.random.default_rng(11)
    wh, Ch, N, taps, n_slots = hip(), 66, 16, 4, 4
    x, dt = normal(rng, (2, 90, Ch), t), normal(rng, (2, 90, Ch), t, 0.5)
    B, Cc = normal(rng, (2, 90, 1, N), t), normal(rng, (2, 90, 1, N), t)
    w, A = rng.normal(size=(Ch, taps)).astype(np.float32), -rng.uniform(0.2, 9, size=(Ch, N)).astype(np.float32)
    bias, slots = rng.normal(size=Ch).astype(np.float32) - 3, np.array([2, 0], np.int32)
    hist0, h0 = normal(rng, (n_slots, taps - 1, Ch), t), rng.normal(size=(n_slots, Ch, N)).astype(np.float32)
    wd, Ad, bd, sd = dev(w), dev(A), dev(bias), dev(slots)
    cols = lambda v, a, b: dev(lr.pack(v[:, a:b].reshape(2 * (b - a), -1), t))

    def run(cuts):
        hist, h, ys = dev(lr.pack(hist0, t)), dev(h0), []
        for a, b in zip(cuts, cuts[1:]):
            T = 2 * (b - a)
            starts = dev(np.array([0, b - a, T], np.int32)) if b - a > 1 else None
            rows = dict(dtype=lr.TYPE[t], tokens=T, channels=Ch, n_seq=2, n_slots=n_slots, starts=starts, slots=sd)
            u, y = (empty((T, Ch), np.float32 if t == "f32" else np.uint16) for _ in range(2))
            wh.short_conv(cols(x, a, b), wd, u, taps=taps, state_in=hist, state_out=hist, **rows)
            need = wh.selective_scan_work(T, Ch, N, 2, b - a) if b - a > 1 else 0
            work = empty(max(need, 16), np.uint8)
            dtb, Bb, Cb = cols(dt, a, b), cols(B, a, b), cols(Cc, a, b)
            wh.selective_scan(u, dtb, Ad, Bb, Cb, y, n_state=N, dt_bias=bd, state_in=h, state_out=h, longest=b - a,
                              work=work, work_bytes=need, **rows)
            ys.append([host(v).reshape(2, b - a, Ch) for v in (u, y)])
        return [np.concatenate(v, 1) for v in zip(*ys)] + [host(hist), host(h)]
    whole = run([0, 90])
    u = lr.unpack(whole[0], t).reshape(180, Ch)
    y, ye, new, ne = lr.scan(u, dt.reshape(180, Ch), A, B.reshape(180, 1, N), Cc.reshape(180, 1, N), None, None, bias, True,
                             [(0, 90), (90, 180)], slots, h0, n_slots)
    for cuts in ([0, 90], [0, 37, 38, 90], list(range(91))):
        cu, cy, chist, ch = run(cuts)
        assert cu.tobytes() == whole[0].tobytes() and chist.tobytes() == whole[2].tobytes()
        lr.check(cy.reshape(180, Ch), y, ye, t)
        lr.check(ch, new, ne, "f32", h0)


def test_offsets_past_32_bits():
    """Rows, states and places whose offsets in elements, and in bytes, pass 2^31 and 2^32."""
    from warp_amd.device import D2D, check, mem_info, rt
    if mem_info()[0] < 100 << 30:
        pytest.skip("not enough device memory")
    rng = np.random.default_rng(2)
    wh, Ch, N, far = hip(), 64, 16, 5 << 28       # a stride of 1.3 G elements: the fourth row is past 2^32 bytes of bf16
    T = 5
    big = empty((T - 1) * far + Ch, np.uint16)    # 10.7 GB

    def scatter(a):
        for r in range(a.shape[0]):
            check(rt().hipMemcpy(big.ptr + 2 * r * far, a[r].ctypes.data, a[r].nbytes, 1), "hipMemcpy")
    x, dt, B, Cc = (normal(rng, (T, w), "bf16", s) for w, s in ((Ch, 1), (Ch, 0.1), (N, 1), (N, 1)))
    w, A = rng.normal(size=(Ch, 4)).astype(np.float32), -rng.uniform(0.2, 2, size=(Ch, N)).astype(np.float32)
    starts, one = dev(np.array([0, T], np.int32)), dev(np.array([0], np.int32))
    scatter(lr.pack(x, "bf16"))
    outs = [empty((T, Ch), np.uint16) for _ in range(4)]
    xb, dtb, Bb, Cb, wb, Ab = dev(lr.pack(x, "bf16")), dev(lr.pack(dt, "bf16")), dev(lr.pack(B, "bf16")), dev(lr.pack(Cc, "bf16")), dev(w), dev(A)
    seq = dict(dtype=1, tokens=T, channels=Ch, n_seq=1, n_slots=1, starts=starts, slots=one)
    # the same from near rows and from far ones, bit for bit
    wh.short_conv(xb, wb, outs[0], taps=4, **seq)
    wh.short_conv(big, wb, outs[1], taps=4, ldx=far, **seq)
    wh.selective_scan(xb, dtb, Ab, Bb, Cb, outs[2], n_state=N, **seq)
    wh.selective_scan(big, dtb, Ab, Bb, Cb, outs[3], n_state=N, ldx=far, **seq)
    o = [host(v).tobytes() for v in outs]
    assert o[0] == o[1] and o[2] == o[3]
    # slots of which the last begins past 2^32 bytes
    n_slots = (5 << 30) // (Ch * N * 4) + 1
    slots = dev(np.array([n_slots - 1, 0], np.int32))
    states = empty((n_slots, Ch, N))
    h0 = rng.normal(size=(2, Ch, N)).astype(np.float32)
    at = [states.ptr + (n_slots - 1) * Ch * N * 4, states.ptr]
    for k in range(2):
        check(rt().hipMemcpy(at[k], h0[k].ctypes.data, h0[k].nbytes, 1), "hipMemcpy")
    y, ye, new, ne = lr.scan(x[:2], dt[:2], A, B[:2, None], Cc[:2, None], None, None, None, True, [(0, 1), (1, 2)], [0, 1], h0, 2)
    wh.selective_scan(xb, dtb, Ab, Bb, Cb, outs[2], n_state=N, dtype=1, tokens=2, channels=Ch, n_seq=2, n_slots=n_slots,
                      slots=slots, state_in=states, state_out=states)
    got = [empty((Ch, N)) for _ in range(2)]
    for k in range(2):
        check(rt().hipMemcpy(got[k].ptr, at[k], Ch * N * 4, D2D), "hipMemcpy")
    lr.check(host(outs[2])[:2], y, ye, "bf16")
    lr.check(np.stack([host(g) for g in got]), new, ne, "f32")
    # pairs' places far apart
    K = 2
    idx = np.array([[1, 0], [0, 1]], np.int32)
    offsets, perm, pos = lr.dispatch(idx, 2)
    ob, pb, qb = empty(3, np.int32), empty(4, np.int32), empty(4, np.int32)
    moe = dict(dtype=1, tokens=2, top_k=K, hidden=Ch)
    wh.expert_dispatch(dev(idx), ob, pb, qb, n_experts=2, x=xb, xs=big, ldxs=far, work=empty(16, np.uint8), work_bytes=16, **moe)
    assert np.array_equal(host(pb), perm) and np.array_equal(host(qb), pos.reshape(-1))
    out, dy, dw = empty((2, Ch), np.uint16), empty((4, Ch), np.uint16), empty((2, K))
    wt = rng.uniform(0.5, 1, size=(2, K)).astype(np.float32)
    wh.expert_combine(big, qb, out, ldy=far, w=dev(wt), **moe)
    xs = x[perm // K]
    ref, err = lr.combine(xs, pos, wt, None)
    lr.check(host(out), ref, err, "bf16")
    wh.expert_combine_backward(xb, big, qb, dy, dw, ldy=far, w=dev(wt), **moe)
    rdy, rdw, rerr = lr.combine_backward(x[:2], xs, pos, wt)
    lr.check(host(dy), rdy, np.abs(rdy) * lr.EPS, "bf16")
    lr.check(host(dw), rdw, rerr, "f32")


def test_layer_with_the_frameworks_router_and_experts():
    """A ragged batch through convolution and scan, the framework's router, dispatch, experts (the records'
    decoded weights, on the host) and combine: what warp_hip_moe_chunk makes of the scan's rows, within the
    1e-4 of max that the framework's experts are held to."""
    import warp_amd
    spec = ct.Spec(hidden=256, inter=128, experts=16, top_k=4, layers=1, fmt="VQ3R", seed=41, shared_bits=0, **BALANCED)
    model = ct.build(spec)
    lengths = [9, 0, 14, 1, 8]
    starts, T = layout(lengths)
    H, I, E, K = spec.hidden, spec.inter, spec.experts, spec.top_k
    rng = np.random.default_rng(4)
    ctx, wh = open_ctx(model, max_tokens=T), hip()
    try:
        warp_amd.load_container_model(ctx, model)
        f = lambda *s: dev(rng.normal(size=s).astype(np.float32))
        x, w, u, y, st = f(T, H), f(H, 4), empty((T, H)), empty((T, H)), dev(starts)
        dt, A, B, Cc = f(T, H), dev(-rng.uniform(0.5, 4, size=(H, 16)).astype(np.float32)), f(T, 16), f(T, 16)
        rows = dict(dtype=wh.F32, tokens=T, channels=H, n_seq=len(lengths), n_slots=len(lengths), starts=st, stream=ctx.stream)
        need = wh.selective_scan_work(T, H, 16, len(lengths), max(lengths))
        work = empty(max(need, 16), np.uint8)
        wh.short_conv(x, w, u, taps=4, **rows)
        wh.selective_scan(u, dt, A, B, Cc, y, n_state=16, z=x, longest=max(lengths), work=work, work_bytes=need, **rows)
        want, logits = empty((T, H)), empty((T, E))
        idx, wt = empty((T, K), np.int32), empty((T, K))
        ctx.router_logits(0, y, T, logits)
        ctx.route(0, logits, T, idx, wt)
        offsets, perm, pos = empty(E + 1, np.int32), empty(T * K, np.int32), empty((T, K), np.int32)
        xs, ys, out = empty((T * K, H)), empty((T * K, H)), empty((T, H))
        nd = wh.expert_dispatch_work(T, K, E)
        moe = dict(dtype=wh.F32, tokens=T, top_k=K, hidden=H, stream=ctx.stream)
        wh.expert_dispatch(idx, offsets, perm, pos, n_experts=E, x=y, xs=xs, work=empty(max(nd, 16), np.uint8), work_bytes=nd, **moe)
        ctx.moe_chunk(0, y, want, T)
        ctx.sync()
        at, rows_in, made = host(offsets), host(xs).astype(np.float64), np.zeros((T * K, H), np.float32)
        assert at[0] == 0 and at[E] == T * K
        for e in range(E):
            if at[e] == at[e + 1]:
                continue
            W = [empty(s) for s in ((I, H), (I, H), (H, I))]
            for kind in range(3):
                ctx.decode_weights(0, kind, ctx.resident(0, e), W[kind])
            ctx.sync()
            g, up, down = (host(v).astype(np.float64) for v in W)
            r = rows_in[at[e]:at[e + 1]]
            a = r @ g.T
            made[at[e]:at[e + 1]] = (a / (1 + np.exp(-a)) * (r @ up.T)) @ down.T
        ys.upload(made)
        wh.expert_combine(ys, pos, out, w=wt, **moe)
        ctx.sync()
        got, ref = host(out), host(want)
        assert np.abs(got - ref).max() <= 1e-4 * np.abs(ref).max()
    finally:
        ctx.close()
