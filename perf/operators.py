"""The operators around a hybrid layer's recurrence and experts: a short
causal convolution, a selective state space scan, tokens sorted by expert and
brought back with their weights, and the gradient of that.

A case is a dict of plain values. prepare() makes what a program holds before
the call, run() is one pass through one operator (in plain torch, or through
warp_amd.hip where `own` is set), exact() the same in 64 bits, written apart.

Kinds:
  conv      short causal convolution over packed sequences with carried
            histories, or one token of each of several sequences
  scan      the selective scan over the same
  dispatch  tokens sorted by expert: offsets, order, places, and the rows
  combine   the experts' rows back to their tokens, weighted (or not: that
            is the gradient of dispatch)
  gradient  of combine: the rows' and the weights'

Convolution inputs are columns of a wider projection (a row stride above the
width), a scan's x, B and C are columns of one convolution's output and its
gate is columns of the projection, as such layers have them. Decay rates
A are -(1..N), time steps lie between 1e-3 and 1e-1 before what the token
adds. Experts are picked with Zipf(1.1) popularity where a case says so.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _conv(name, type, channels, tokens, seqs, **kw):
    return dict(dict(name=name, kind="conv", type=type, channels=channels, taps=4, tokens=tokens, seqs=seqs, single=False,
                     bias=True, silu=True, pad=0), **kw)


def _scan(name, type, channels, states, tokens, seqs, **kw):
    return dict(dict(name=name, kind="scan", type=type, channels=channels, states=states, groups=1, tokens=tokens,
                     seqs=seqs, single=False, gate=True, softplus=True, pad=0), **kw)


def _moe(name, kind, type, hidden, experts, top_k, tokens, **kw):
    return dict(dict(name=name, kind=kind, type=type, hidden=hidden, experts=experts, top_k=top_k, tokens=tokens, zipf=0.0,
                     drop=0.0, weights=True, residual=False), **kw)


def listed():
    return [
        # one token of each of eight sequences: a step of generation, mostly its launch
        _conv("conv-tokens", "bf16", 4640, 8, 8, single=True),
        # the q (or k, or v) rows of a delta-attention layer, 32 heads of 128, one prompt of an odd length
        _conv("conv-prompt", "f32", 4096, 1537, 1, bias=False),
        # a packed batch of ragged prompts through a wide mixer
        _conv("conv-packed", "bf16", 4640, 8191, 11),
        # one sequence's next token
        _scan("scan-token", "bf16", 4608, 16, 1, 1, single=True),
        # a batch of 256 sequences' next tokens, bound by their states
        _scan("scan-tokens", "bf16", 4608, 16, 256, 256, single=True),
        # one long prompt: no parallelism across sequences
        _scan("scan-prompt", "bf16", 4608, 16, 4096, 1),
        # packed ragged prompts, wide states in several groups, 32 bits, no gate
        _scan("scan-packed", "f32", 2304, 64, 1999, 13, groups=4, gate=False),
        # 32 sequences' tokens of one step through the widest layer
        _moe("dispatch-tokens", "dispatch", "bf16", 7168, 384, 16, 32),
        # a prompt's tokens on 256 experts of uneven popularity
        _moe("dispatch-prompt", "dispatch", "bf16", 2304, 256, 8, 4096, zipf=1.1),
        # a few tokens brought back onto their residual stream
        _moe("combine-tokens", "combine", "f32", 2304, 256, 8, 7, residual=True),
        # a large batch through the widest layer
        _moe("combine-prompt", "combine", "bf16", 7168, 384, 16, 4096, zipf=1.1),
        # a training step's backward pass
        _moe("gradient-prompt", "gradient", "bf16", 2304, 256, 8, 8192, zipf=1.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["conv", "scan", "scan", "dispatch", "combine", "gradient"])
    type = rng.choice(["f32", "bf16", "f16"])
    single = rng.random() < 0.35
    if kind == "conv":
        channels = _log(rng, 200, 16000)
        tokens = _log(rng, 1, 512) if single else _log(rng, 2, min(8191, 38_000_000 // channels))
        seqs = tokens if single else _log(rng, 1, min(64, tokens))
        case = _conv("", type, channels, tokens, seqs, taps=rng.choice([2, 3, 4, 4, 4, 5, 8]), single=single,
                     bias=rng.random() < 0.5, silu=rng.random() < 0.8)
    elif kind == "scan":
        states = rng.choice([4, 8, 12, 16, 16, 16, 23, 32, 64, 128])
        groups = rng.choice([1, 1, 2, 3, 8])
        channels = groups * _log(rng, 100 // groups, 7168 // groups)
        most = 300_000_000 // (channels * states)
        tokens = _log(rng, 1, min(256, most)) if single else _log(rng, 2, min(6000, most))
        seqs = tokens if single else _log(rng, 1, min(64, tokens))
        case = _scan("", type, channels, states, tokens, seqs, groups=groups, single=single, gate=rng.random() < 0.7,
                     softplus=rng.random() < 0.8)
    else:
        experts = _log(rng, 8, 896)
        top_k = min(experts // 2, rng.choice([1, 2, 4, 6, 8, 8, 16]))
        hidden = _log(rng, 250, 7168)
        tokens = _log(rng, 1, min(8192, 150_000_000 // (top_k * hidden)))
        case = _moe("", kind, type, hidden, experts, top_k, tokens, zipf=rng.choice([0.0, 1.1]),
                    drop=rng.choice([0.0, 0.0, 0.1]), weights=rng.random() < 0.7, residual=rng.random() < 0.5)
    if single:
        if "pad" in case:
            case["pad"] = rng.choice([0, 0, tokens // 4])
    del case["name"]
    return case


# ---- inputs, from the seed alone -------------------------------------------------------------------


def _gen(seed, tag):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + tag * 7919) & 0x7FFFFFFFFFFF)
    return g


def _normal(seed, tag, shape, std=1.0):
    return torch.randn(shape, generator=_gen(seed, tag), device="cuda") * std


def _uniform(seed, tag, shape, lo=0.0, hi=1.0):
    return torch.rand(shape, generator=_gen(seed, tag), device="cuda") * (hi - lo) + lo


def _sequences(case, seed):
    """Lengths on the host (as a scheduler has them), starts and slots on the device. Uneven lengths, some empty."""
    rng = np.random.default_rng((seed, 77))
    n, T = case["seqs"], case["tokens"]
    if case["single"]:
        lengths = np.ones(n, int)
    else:
        p = rng.exponential(size=n) * (rng.random(n) < 0.9) + 1e-9
        lengths = rng.multinomial(T, p / p.sum())
    slots = rng.permutation(n + 2)[:n].astype(np.int32)
    if case["pad"]:
        slots[n - case["pad"]:] = -1     # rows of a batch that is not full
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    return dict(lengths=[int(v) for v in lengths], starts=torch.from_numpy(starts).cuda(),
                slots=torch.from_numpy(slots).cuda(), n_slots=n + 2)


def _picks(case, seed):
    """[T][K] distinct experts of each token, by popularity; -1 where a pair is dropped."""
    T, E, K = case["tokens"], case["experts"], case["top_k"]
    pop = -case["zipf"] * torch.log(1.0 + torch.randperm(E, generator=_gen(seed, 20), device="cuda"))
    u = _uniform(seed, 21, (T, E), 1e-9, 1.0)
    idx = (pop - torch.log(-torch.log(u))).topk(K, 1).indices.int()
    if case["drop"]:
        idx = torch.where(_uniform(seed, 22, (T, K)) < case["drop"], -1, idx)
    return idx.contiguous()


def prepare(case, seed):
    kind, T, t = case["kind"], case["tokens"], TYPES[case["type"]]
    s = dict(case=case)
    if kind == "conv":
        C, K = case["channels"], case["taps"]
        s.update(_sequences(case, seed))
        s["x"] = _normal(seed, 1, (T, C + 64)).to(t)[:, 32:32 + C]
        s["w"] = _normal(seed, 2, (C, K), K ** -0.5)
        s["bias"] = _normal(seed, 3, (C,), 0.1) if case["bias"] else None
        s["history"] = _normal(seed, 4, (s["n_slots"], K - 1, C)).to(t)
    elif kind == "scan":
        D, N, G = case["channels"], case["states"], case["groups"]
        s.update(_sequences(case, seed))
        wide = _normal(seed, 1, (T, D + 2 * G * N)).to(t)
        s["x"], s["B"], s["C"] = wide[:, :D], wide[:, D:D + G * N], wide[:, D + G * N:]
        s["z"] = _normal(seed, 2, (T, 2 * D)).to(t)[:, D:] if case["gate"] else None
        step = torch.exp(_uniform(seed, 3, (D,), math.log(1e-3), math.log(1e-1)))
        if case["softplus"]:
            s["dt"], s["dt_bias"] = _normal(seed, 4, (T, D), 0.5).to(t), torch.log(torch.expm1(step))
        else:
            s["dt"], s["dt_bias"] = (step * torch.exp(_normal(seed, 4, (T, D), 0.5))).to(t), None
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * _uniform(seed, 5, (D, 1), 0.8, 1.2)
        s["D"] = _normal(seed, 6, (D,), 0.1) + 1
        s["h"] = _normal(seed, 7, (s["n_slots"], D, N), 0.3)
    else:
        K, H = case["top_k"], case["hidden"]
        s["idx"] = _picks(case, seed)
        if kind == "dispatch":
            s["x"] = _normal(seed, 1, (T, H)).to(t)
        else:
            s["pos"] = _sort(s["idx"], case["experts"])[2]
            s["y"] = _normal(seed, 1, (T * K, H)).to(t)
            w = torch.sigmoid(_normal(seed, 2, (T, K)))
            s["w"] = 2.0 * w / w.sum(1, keepdim=True) if case["weights"] or kind == "gradient" else None
            s["resid"] = _normal(seed, 3, (T, H)).to(t) if case["residual"] and kind == "combine" else None
            s["dout"] = _normal(seed, 3, (T, H)).to(t) if kind == "gradient" else None
    return s


# ---- the operators in plain torch ------------------------------------------------------------------


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(torch.clamp(v, max=20))))


def _rows(s):
    """Each token's sequence and its place in it."""
    t = torch.arange(s["case"]["tokens"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    return t, seq, t - s["starts"].long()[seq]


def _plain_conv(s):
    T, K, C = s["case"]["tokens"], s["case"]["taps"], s["case"]["channels"]
    t, seq, at = _rows(s)
    slots = s["slots"].long()
    ext = torch.cat([s["x"], s["history"].reshape(-1, C)])
    back = K - 1 - torch.arange(K, device="cuda")
    src, hist = t[:, None] - back, T + slots.clamp(min=0)[seq][:, None] * (K - 1) + K - 1 + at[:, None] - back
    u = ext[torch.where(at[:, None] >= back, src, hist)].float()
    v = (u * s["w"].t()).sum(1)
    if s["bias"] is not None:
        v = v + s["bias"]
    if s["case"]["silu"]:
        v = v / (1 + torch.exp(-v))
    live = slots >= 0
    y = torch.where(live[seq][:, None], v, 0.0).to(s["x"].dtype)
    # the last taps - 1 inputs of each sequence
    begin, end = s["starts"].long()[:-1, None], s["starts"].long()[1:, None]
    r = end - begin - (K - 1) + torch.arange(K - 1, device="cuda")
    new = ext[torch.where(r >= 0, begin + r, T + slots.clamp(min=0)[:, None] * (K - 1) + K - 1 + r)]
    out = torch.zeros((s["n_slots"] + 1,) + tuple(s["history"].shape[1:]), dtype=y.dtype, device="cuda")
    out[torch.where(live, slots, s["n_slots"])] = new
    return y, out[:-1]


def _plain_scan(s):
    D, N, G = s["case"]["channels"], s["case"]["states"], s["case"]["groups"]
    t, seq, at = _rows(s)
    slots = s["slots"].long()
    live, slot = slots >= 0, slots.clamp(min=0)
    x, dt = s["x"].float(), s["dt"].float()
    if s["dt_bias"] is not None:
        dt = _softplus(dt + s["dt_bias"])
    B = s["B"].float().view(-1, G, 1, N).expand(-1, -1, D // G, -1).reshape(-1, D, N)
    a = torch.exp(dt[:, :, None] * s["A"])
    b = (dt * x)[:, :, None] * B
    begin, end = s["starts"].long()[:-1], s["starts"].long()[1:]
    some, first = end > begin, begin.clamp(max=len(t) - 1)
    b.index_add_(0, first, torch.where(some[:, None, None], a[first] * s["h"][slot], 0.0))
    a = torch.where((at == 0)[:, None, None], 0.0, a)
    step = 1
    while step < max(s["lengths"]):      # each row takes in twice as many before it
        b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    C = s["C"].float().view(-1, G, 1, N).expand(-1, -1, D // G, -1).reshape(-1, D, N)
    y = (b * C).sum(-1) + s["D"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * (z / (1 + torch.exp(-z)))
    y = torch.where(live[seq][:, None], y, 0.0).to(s["x"].dtype)
    h = torch.zeros((s["n_slots"] + 1, D, N), device="cuda")
    h[torch.where(live, slots, s["n_slots"])] = torch.where(some[:, None, None], b[(end - 1).clamp(min=0)], s["h"][slot])
    return y, h[:-1]


def _sort(idx, experts):
    flat = torch.where((idx >= 0) & (idx < experts), idx, experts).reshape(-1)
    key, order = torch.sort(flat, stable=True)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device="cuda", dtype=key.dtype)).int()
    kept = key < experts
    pos = torch.empty_like(order)
    pos[order] = torch.where(kept, torch.arange(len(order), device="cuda"), -1)
    return offsets, torch.where(kept, order, 0).int(), pos.int().view(idx.shape), kept


def _plain_dispatch(s):
    offsets, perm, pos, kept = _sort(s["idx"], s["case"]["experts"])
    xs = torch.where(kept[:, None], s["x"][perm.long() // s["case"]["top_k"]], 0.0)
    return offsets, perm, pos, xs.to(s["x"].dtype)


def _taken(s):
    live = s["pos"] >= 0
    return live, torch.where(live[:, :, None], s["y"][s["pos"].long().clamp(min=0)], 0.0).float()


def _plain_combine(s):
    _, rows = _taken(s)
    out = (rows if s["w"] is None else rows * s["w"][:, :, None]).sum(1)
    if s["resid"] is not None:
        out = out + s["resid"].float()
    return out.to(s["y"].dtype)


def _plain_gradient(s):
    live, rows = _taken(s)
    d = s["dout"].float()[:, None, :]
    dw = torch.where(live, (rows * d).sum(-1), 0.0)
    dy = torch.zeros((s["y"].shape[0] + 1, s["y"].shape[1]), dtype=s["y"].dtype, device="cuda")
    dy[torch.where(live, s["pos"], s["y"].shape[0]).long()] = (s["w"][:, :, None] * d).to(dy.dtype)
    return dy[:-1], dw


# ---- and by the framework's kernels ----------------------------------------------------------------


def _buffers(s):
    """Outputs and workspace that a program keeps for its calls."""
    from warp_amd import hip
    case, k = s["case"], s.get("kept")
    if k is None:
        k = s["kept"] = dict(type=dict(f32=hip.F32, bf16=hip.BF16, f16=hip.F16)[case["type"]])
        T, K, H = case["tokens"], case.get("top_k"), case.get("hidden")
        if case["kind"] in ("conv", "scan"):
            k["y"] = torch.zeros((T, case["channels"]), dtype=s["x"].dtype, device="cuda")
            k["state"] = torch.zeros_like(s["history"] if case["kind"] == "conv" else s["h"])
        elif case["kind"] == "dispatch":
            k["offsets"] = torch.empty(case["experts"] + 1, dtype=torch.int32, device="cuda")
            k["perm"], k["pos"] = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (T * K, (T, K)))
            k["xs"] = torch.zeros((T * K, H), dtype=s["x"].dtype, device="cuda")
        else:
            k["out"] = torch.empty((T, H), dtype=s["y"].dtype, device="cuda")
            k["dy"], k["dw"] = torch.zeros_like(s["y"]), torch.empty((T, K), device="cuda")
        n = 0
        if case["kind"] == "scan" and not case["single"]:
            n = hip.selective_scan_work(T, case["channels"], case["states"], case["seqs"], max(s["lengths"]))
        elif case["kind"] == "dispatch":
            n = hip.expert_dispatch_work(T, K, case["experts"])
        k["work"] = torch.empty(n, dtype=torch.uint8, device="cuda") if n else None
    return hip, k


def _own(s):
    hip, k = _buffers(s)
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    kind = case["kind"]
    if kind in ("conv", "scan"):
        rows = dict(dtype=k["type"], tokens=case["tokens"], channels=case["channels"], n_seq=case["seqs"],
                    starts=None if case["single"] else s["starts"], slots=s["slots"], n_slots=s["n_slots"],
                    state_out=k["state"], ldx=s["x"].stride(0), stream=stream)
        if kind == "conv":
            hip.short_conv(s["x"], s["w"], k["y"], taps=case["taps"], bias=s["bias"], silu=case["silu"],
                           state_in=s["history"], **rows)
        else:
            z, w = s["z"], k["work"]
            hip.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], k["y"], n_state=case["states"],
                               groups=case["groups"], D=s["D"], z=z, dt_bias=s["dt_bias"], softplus=case["softplus"],
                               state_in=s["h"], ldbc=s["B"].stride(0), ldz=z.stride(0) if z is not None else 0,
                               longest=max(s["lengths"]), work=w, work_bytes=w.numel() if w is not None else 0, **rows)
        return k["y"], k["state"]
    if kind == "dispatch":
        hip.expert_dispatch(s["idx"], k["offsets"], k["perm"], k["pos"], tokens=case["tokens"], top_k=case["top_k"],
                            n_experts=case["experts"], x=s["x"], xs=k["xs"], dtype=k["type"], hidden=case["hidden"],
                            work=k["work"], work_bytes=k["work"].numel() if k["work"] is not None else 0, stream=stream)
        return k["offsets"], k["perm"], k["pos"], k["xs"]
    sizes = dict(dtype=k["type"], tokens=case["tokens"], top_k=case["top_k"], hidden=case["hidden"], w=s["w"],
                 stream=stream)
    if kind == "combine":
        hip.expert_combine(s["y"], s["pos"], k["out"], resid=s["resid"], **sizes)
        return k["out"]
    hip.expert_combine_backward(s["dout"], s["y"], s["pos"], k["dy"], k["dw"], **sizes)
    return k["dy"], k["dw"]


def run(state):
    if own:
        return _own(state)
    return dict(conv=_plain_conv, scan=_plain_scan, dispatch=_plain_dispatch, combine=_plain_combine,
                gradient=_plain_gradient)[state["case"]["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    T, e = case["tokens"], 4 if case["type"] == "f32" else 2
    if case["kind"] == "conv":
        C, K = case["channels"], case["taps"]
        return {"bytes": 2 * e * C * (T + case["seqs"] * (K - 1)) + 4 * C * (K + 1), "flops": T * C * (2 * K + 4)}
    if case["kind"] == "scan":
        D, N = case["channels"], case["states"]
        rows = T * ((4 if case["gate"] else 3) * D + 2 * case["groups"] * N)
        return {"bytes": e * rows + 8 * case["seqs"] * D * N + 4 * D * (N + 2), "flops": T * D * (7 * N + 8)}
    K, H = case["top_k"], case["hidden"]
    kept = T * K * (1 - case["drop"])
    if case["kind"] == "dispatch":
        return {"bytes": e * H * (T + kept) + 4 * (3 * T * K + case["experts"]), "flops": 0}
    if case["kind"] == "combine":
        return {"bytes": e * H * (kept + T * (2 if case["residual"] else 1)) + 8 * T * K, "flops": 2 * kept * H}
    return {"bytes": e * H * (2 * kept + T) + 12 * T * K, "flops": 3 * kept * H}


# ---- the same in 64 bits ---------------------------------------------------------------------------


def _exact_conv(s):
    K, x, w, out = s["case"]["taps"], s["x"].double(), s["w"].double(), []
    new = torch.zeros(s["history"].shape, dtype=torch.float64, device="cuda")
    begin = 0
    for n, slot in zip(s["lengths"], s["slots"].tolist()):
        u = torch.cat([s["history"][max(slot, 0)].double(), x[begin:begin + n]])
        begin += n
        v = sum(w[:, j] * u[j:j + n] for j in range(K))
        v = v if s["bias"] is None else v + s["bias"].double()
        v = v * torch.sigmoid(v) if s["case"]["silu"] else v
        out.append(v if slot >= 0 else torch.zeros_like(v))
        if slot >= 0:
            new[slot] = u[n:]
    return torch.cat(out), new


def _exact_scan(s):
    D, N, G = s["case"]["channels"], s["case"]["states"], s["case"]["groups"]
    x, dt = s["x"].double(), s["dt"].double()
    if s["dt_bias"] is not None:
        dt = torch.nn.functional.softplus(dt + s["dt_bias"].double(), threshold=60)
    A, B, C = s["A"].double(), s["B"].double().view(-1, G, N), s["C"].double().view(-1, G, N)
    group = torch.arange(D, device="cuda") // (D // G)
    y, new = torch.zeros_like(x), torch.zeros(s["h"].shape, dtype=torch.float64, device="cuda")
    if s["case"]["single"]:              # a step of every sequence at once
        live = (s["slots"] >= 0).nonzero()[:, 0]
        slot = s["slots"][live].long()
        h = torch.exp(dt[live, :, None] * A) * s["h"][slot].double() + (dt * x)[live, :, None] * B[live][:, group]
        y[live], new[slot] = (h * C[live][:, group]).sum(-1), h
    else:
        t = 0
        for n, slot in zip(s["lengths"], s["slots"].tolist()):
            h = s["h"][slot].double()
            for t in range(t, t + n):
                h = torch.addcmul((dt[t] * x[t])[:, None] * B[t][group], torch.exp(dt[t][:, None] * A), h)
                y[t] = (h * C[t][group]).sum(-1)
            t += n > 0
            new[slot] = h
    y = y + s["D"].double() * x
    if s["z"] is not None:
        y = y * torch.nn.functional.silu(s["z"].double())
    if s["case"]["single"]:
        y[s["slots"] < 0] = 0
    return y, new


def _exact_moe(s):
    kind, K, E = s["case"]["kind"], s["case"]["top_k"], s["case"]["experts"]
    idx = s["idx"].cpu().numpy().reshape(-1)
    order = np.concatenate([np.flatnonzero(idx == e) for e in range(E)])
    if kind == "dispatch":
        xs = torch.zeros((len(idx), s["x"].shape[1]), dtype=torch.float64, device="cuda")
        xs[:len(order)] = s["x"].double()[torch.from_numpy(order // K).cuda()]
        return None, None, None, xs
    token, pair = torch.from_numpy(order // K).cuda(), torch.from_numpy(order).cuda()
    w = s["w"].double().reshape(-1)[pair] if s["w"] is not None else torch.ones(len(order), dtype=torch.float64, device="cuda")
    y = s["y"][:len(order)].double()     # in the order of the experts
    if kind == "combine":
        out = torch.zeros((s["case"]["tokens"], y.shape[1]), dtype=torch.float64, device="cuda")
        out = out if s["resid"] is None else s["resid"].double()
        return out.index_add(0, token, y * w[:, None])
    d = s["dout"].double()[token]
    dy, dw = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda"), torch.zeros(len(idx), dtype=torch.float64, device="cuda")
    dy[:len(order)] = d * w[:, None]
    dw[pair] = torch.einsum("ij,ij->i", d, y)
    return dy, dw.view(-1, K)


def exact(case, seed):
    s = prepare(case, seed)
    return dict(conv=_exact_conv, scan=_exact_scan).get(case["kind"], _exact_moe)(s)
