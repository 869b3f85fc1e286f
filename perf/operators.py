"""Workloads of the rotary positions, the short causal convolution and the selective scan, with
their plain forms in elementary torch operations and their definitions in 64 bits.

``run`` computes the plain form where ``own`` is false and calls the framework's operators where it
is true, on the same state.  Sizes: heads 16 / 32 of 64 / 128 features, batches and lengths are
those of the framework's own benchmarks (B8-H16-D64 up to T=32768, B4-H32-D128), the channel
counts of the convolution and the scan are the same models' heads x features."""
import math
import os
import sys

import torch
import torch.nn.functional as F

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one new token of each of 64 requests, every request at a position of its own: decoding
        dict(name="rotary_token", op="rotary", B=64, L=1, H=16, Hk=16, D=64, R=64, dtype="bf16", layout="blhd",
             interleaved=False, scaling="none", positions="far", grad=False),
        # a prompt of a long-context model: shared key heads, positions stretched eight times
        dict(name="rotary_prompt", op="rotary", B=2, L=8192, H=32, Hk=8, D=128, R=128, dtype="bf16", layout="blhd",
             interleaved=False, scaling="yarn", positions="far", grad=False),
        # training with part of a head rotated, odd batch, heads and length
        dict(name="rotary_train_partial", op="rotary", B=3, L=1537, H=5, Hk=5, D=80, R=48, dtype="f16", layout="bhld",
             interleaved=True, scaling="none", positions="none", grad=True),
        # training at the framework's headline size: the rotary inputs of decoupled_la
        dict(name="rotary_train_large", op="rotary", B=8, L=32768, H=16, Hk=16, D=64, R=64, dtype="bf16",
             layout="bhld", interleaved=True, scaling="none", positions="none", grad=True),
        # one new token of each of 64 requests through the convolution, the history carried in place
        dict(name="conv_token", op="conv_step", B=64, C=2048, W=4, dtype="bf16", silu=True, bias=True),
        # a training step's convolution
        dict(name="conv_train", op="conv", B=8, T=4096, C=2048, W=4, dtype="bf16", silu=True, bias=True, seqs=0,
             state=False, grad=True),
        # packed sequences of uneven lengths, full precision, no activation
        dict(name="conv_packed", op="conv", B=1, T=7001, C=1003, W=3, dtype="f32", silu=False, bias=False, seqs=13,
             state=False, grad=True),
        # one new token of each of 64 requests through the scan, the state carried in place
        dict(name="scan_token", op="scan_step", B=64, C=2048, N=16, G=1, dtype="bf16", gate=True),
        # a long prompt: the whole sequence at once, its last state kept for decoding
        dict(name="scan_prompt", op="scan", B=1, T=8192, C=4096, N=16, G=1, dtype="bf16", gate=True, seqs=0,
             state=True, grad=False),
        # a training step's scan
        dict(name="scan_train", op="scan", B=8, T=4096, C=2048, N=16, G=1, dtype="bf16", gate=True, seqs=0,
             state=False, grad=True),
        # one long sequence: few channels, many tokens
        dict(name="scan_train_long", op="scan", B=1, T=16384, C=1024, N=16, G=1, dtype="f16", gate=True, seqs=0,
             state=False, grad=True),
        # packed sequences of uneven lengths, full precision, two groups, odd channels, small states
        dict(name="scan_packed", op="scan", B=1, T=5003, C=1010, N=8, G=2, dtype="f32", gate=False, seqs=11,
             state=False, grad=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    op = rng.choice(["rotary", "rotary", "conv", "conv", "conv_step", "scan", "scan", "scan", "scan_step"])
    if op == "rotary":
        D = rng.choice([32, 48, 64, 64, 80, 96, 128, 128, 256])
        R = rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)])
        Hk = _log(rng, 1, 32)
        H = Hk * rng.choice([1, 1, 2, 4])
        L = _log(rng, 1, 32768)
        B = _log(rng, 1, max(1, min(128, (1 << 27) // (L * H * D))))
        return dict(op=op, B=B, L=L, H=H, Hk=Hk, D=D, R=R, dtype=dtype, layout=rng.choice(["bhld", "blhd"]),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    positions=rng.choice(["none", "far"]), grad=rng.random() < 0.6)
    if op == "conv_step":
        return dict(op=op, B=_log(rng, 1, 512), C=_log(rng, 64, 8192), W=rng.randint(2, 4), dtype=dtype,
                    silu=rng.random() < 0.7, bias=rng.random() < 0.7)
    if op == "scan_step":
        G = rng.choice([1, 1, 2])
        return dict(op=op, B=_log(rng, 1, 512), C=G * _log(rng, 32, 4096), N=rng.choice([8, 16, 16, rng.randint(1, 32)]),
                    G=G, dtype=dtype, gate=rng.random() < 0.7)
    T = _log(rng, 1, 16384)
    G = rng.choice([1, 1, 2]) if op == "scan" else 1
    C = G * _log(rng, 64 // G, 4096 // G)
    seqs = rng.randint(1, 24) if rng.random() < 0.35 else 0
    case = dict(op=op, B=1, T=T, C=C, dtype=dtype, seqs=seqs, state=not seqs and rng.random() < 0.4,
                grad=rng.random() < 0.7)
    N = rng.choice([8, 16, 16, rng.randint(1, 32)])
    if not seqs:
        case["B"] = _log(rng, 1, max(1, min(64, (1 << 30) // (T * C * (N if op == "scan" else 16)))))
    if op == "conv":
        return dict(case, W=rng.randint(2, 4), silu=rng.random() < 0.7, bias=rng.random() < 0.7)
    return dict(case, N=N, G=G, gate=rng.random() < 0.7)


# ---- inputs ---------------------------------------------------------------------------------------

def _frequencies(case):
    """Radians per position of every pair, and the factor on the rotated features."""
    P = case["R"] // 2
    i = torch.arange(P, dtype=torch.float64, device="cuda")
    base, s, factor = 10000.0, 8.0, 1.0
    if case["scaling"] == "ntk" and P > 1:
        base *= s ** (P / (P - 1))
    f = base ** (-i / P)
    if case["scaling"] == "linear":
        f = f / s
    elif case["scaling"] == "yarn":
        keep = ((4096 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
        f = f * keep + f / s * (1 - keep)
        factor = 0.1 * math.log(s) + 1.0
    return f, factor


def _bounds(case, rng_cpu):
    """Sequence boundaries of a packed batch: uneven, ending at the last token."""
    T, n = case["T"], min(case["seqs"], case["T"])
    cuts = torch.randperm(T - 1, generator=rng_cpu)[:n - 1].sort().values + 1 if n > 1 else torch.empty(0, dtype=torch.long)
    return [0] + cuts.tolist() + [T]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def randn(*shape, to=dt, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(to)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=g, device="cuda") * (hi - lo) + lo

    s = {"case": dict(case)}
    op = case["op"]
    if op == "rotary":
        B, L, H, Hk, D = (case[k] for k in ("B", "L", "H", "Hk", "D"))
        shape = (lambda h: (B, h, L, D)) if case["layout"] == "bhld" else (lambda h: (B, L, h, D))
        s["q"], s["k"] = randn(*shape(H)), randn(*shape(Hk))
        s["freqs"], s["factor"] = _frequencies(case)
        s["positions"] = None
        if case["positions"] == "far":      # every row starts at a position of its own
            start = torch.randint(0, 32768, (B, 1), generator=g, device="cuda")
            s["positions"] = start + torch.arange(L, device="cuda")
        if case["grad"]:
            s["dq"], s["dk"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
            for d in (s["dq"], s["dk"]):
                d.copy_(randn(*d.shape))
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        return s
    C = case["C"]
    if op in ("conv", "conv_step"):
        W = case["W"]
        s["w"] = uniform(-W ** -0.5, W ** -0.5, C, W).to(dt)
        s["b"] = uniform(-W ** -0.5, W ** -0.5, C).to(dt) if case["bias"] else None
        if op == "conv_step":
            s["x"], s["hist"] = randn(case["B"], C), randn(case["B"], W - 1, C)
            return s
        s["hist"] = randn(case["B"], W - 1, C) if case["state"] else None
    else:
        N, G, B = case["N"], case["G"], case["B"]
        n = torch.arange(1, N + 1, device="cuda", dtype=torch.float32)
        s["A"] = -n * torch.exp(uniform(-0.3, 0.3, C, N))           # negative: decays from slow to fast
        step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), C))
        s["bias"] = step + torch.log(-torch.expm1(-step))           # softplus of it is the usual step
        s["D"] = 1.0 + 0.1 * randn(C, to=torch.float32)
        if op == "scan_step":
            s["x"], s["dt"] = randn(B, C), randn(B, C, scale=0.5)
            s["Bm"], s["Cm"] = (randn(B, G, N) for _ in range(2))
            s["z"] = randn(B, C) if case["gate"] else None
            s["h"] = randn(B, C, N, to=torch.float32, scale=0.2)
            return s
        s["hist"] = randn(B, C, N, to=torch.float32, scale=0.2) if case["state"] else None
    T, B = case["T"], case["B"]
    lead = (T,) if case["seqs"] else (B, T)
    # x and the gate are the two halves of one projection's output, as in the block they come from
    xz = randn(*lead, 2 * C)
    s["x"] = xz[..., :C]
    s["cu"], s["start"] = None, None
    if case["seqs"]:
        bounds = _bounds(case, gc)
        s["bounds"] = bounds
        s["cu"] = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    leaves = ["x", "w", "b"]
    if op == "scan":
        s["z"] = xz[..., C:] if case["gate"] else None
        s["dt"] = randn(*lead, C, scale=0.5)
        bc = randn(*lead, 2 * G * N)
        s["Bm"], s["Cm"] = (h.unflatten(-1, (G, N)) for h in bc.split(G * N, -1))
        leaves = ["x", "dt", "A", "Bm", "Cm", "D", "z", "bias"]
    if case["state"]:
        leaves.append("hist")
    s["leaves"] = [k for k in leaves if s.get(k) is not None]
    if case["grad"]:
        s["dy"] = randn(*lead, C)
        for k in s["leaves"]:
            s[k] = s[k].detach().requires_grad_()
        if case["state"]:
            s["dstate"] = randn(*s["hist"].shape, to=s["hist"].dtype)
    return s


# ---- the framework's operators --------------------------------------------------------------------

def _run_own(s):
    pkg = os.path.join(_ROOT, "flash-bidirectional-linear-attention_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    c = s["case"]
    op = c["op"]
    if op == "rotary":
        from flash_bla.ops.rotary.fused import rotary_embedding
        out = rotary_embedding(s["q"], s["k"], s["freqs"], s["positions"], factor=s["factor"],
                               interleaved=c["interleaved"], layout=c["layout"])
        if not c["grad"]:
            return out
        return [o.detach() for o in out] + list(torch.autograd.grad(out, (s["q"], s["k"]), (s["dq"], s["dk"])))
    act = "silu" if c.get("silu") else None
    if op == "conv_step":
        from flash_bla.ops.selective_scan.conv import causal_conv1d_step
        return causal_conv1d_step(s["x"], s["hist"], s["w"], s["b"], activation=act), s["hist"]
    if op == "scan_step":
        from flash_bla.ops.selective_scan.scan import selective_scan_step
        return selective_scan_step(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], s["h"], s["D"], s["z"], s["bias"],
                                   dt_softplus=True), s["h"]
    keep = dict(initial_state=s["hist"], return_final_state=True) if c["state"] else {}
    if op == "conv":
        from flash_bla.ops.selective_scan.conv import causal_conv1d
        out = causal_conv1d(s["x"], s["w"], s["b"], activation=act, cu_seqlens=s["cu"], **keep)
    else:
        from flash_bla.ops.selective_scan.scan import selective_scan
        out = selective_scan(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], s["D"], s["z"], s["bias"], dt_softplus=True,
                             cu_seqlens=s["cu"], **keep)
    out = out if c["state"] else (out,)
    if not c["grad"]:
        return [o.detach() for o in out]
    grads = torch.autograd.grad(out, [s[k] for k in s["leaves"]], [s["dy"]] + ([s["dstate"]] if c["state"] else []))
    return [o.detach() for o in out] + list(grads)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end -------------------------

def _rotate(x, cos, sin, R, interleaved):
    x = x.float()
    r, rest = x[..., :R], x[..., R:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :R // 2], r[..., R // 2:])
    u, v = a * cos - b * sin, a * sin + b * cos
    r = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((r, rest), -1)


def _plain_rotary(s):
    c = s["case"]
    pos = s["positions"] if s["positions"] is not None else torch.arange(c["L"], device="cuda")
    ang = pos[..., None].double() * s["freqs"]                      # far positions: the angle in 64 bits
    cos, sin = (f(ang).float() * s["factor"] for f in (torch.cos, torch.sin))
    if cos.dim() == 2:
        cos, sin = cos[None], sin[None]
    cos, sin = (t.unsqueeze(1 if c["layout"] == "bhld" else 2) for t in (cos, sin))
    turn = lambda x, sn: _rotate(x.detach(), cos, sn, c["R"], c["interleaved"]).to(x.dtype)  # noqa: E731
    out = [turn(s["q"], sin), turn(s["k"], sin)]
    if c["grad"]:
        out += [turn(s["dq"], -sin), turn(s["dk"], -sin)]
    return out


def _silu_slope(p):
    sg = torch.sigmoid(p)
    return sg * (1 + p * (1 - sg))


def _starts(s, T):
    """First token of every token's own sequence."""
    if s["cu"] is None:
        return torch.zeros(T, dtype=torch.long, device="cuda")
    cu = s["cu"].long()
    return cu[torch.searchsorted(cu, torch.arange(T, device="cuda"), right=True) - 1]


def _plain_conv(s):
    c = s["case"]
    W, T, dt = c["W"], c["T"], s["x"].dtype
    x = s["x"].detach().float().reshape(-1, T, c["C"])
    B = x.shape[0]
    hist = s["hist"].detach().float() if c["state"] else x.new_zeros(B, W - 1, c["C"])
    full = torch.cat((hist, x), 1)                                  # token t is row t + W - 1
    t = torch.arange(T, device="cuda")
    far = torch.arange(W, device="cuda") - (W - 1)                  # tap j looks at token t + far[j]
    ok = (t[:, None] + far >= _starts(s, T)[:, None]) if c["seqs"] else torch.ones(T, W, dtype=torch.bool, device="cuda")
    win = full.unfold(1, W, 1) * ok[None, :, None, :]               # (B, T, C, W)
    w = s["w"].detach().float()
    p = (win * w).sum(-1)
    if c["bias"]:
        p = p + s["b"].detach().float()
    y = p * torch.sigmoid(p) if c["silu"] else p
    last = full[:, T:]
    out = [y.to(dt).reshape(s["x"].shape)] + ([last.to(dt)] if c["state"] else [])
    if not c["grad"]:
        return out
    g = s["dy"].float().reshape(B, T, -1)
    if c["silu"]:
        g = g * _silu_slope(p)
    gw = g[..., None] * w * ok[None, :, None, :]                    # what token t sends to token t + far[j]
    dfull = F.pad(gw, (0, 0, 0, 0, W - 1, W - 1))                   # rows -(W-1) .. T+W-2 of t
    # row r of `full` receives tap j of token t = r - j
    r = torch.arange(T + W - 1, device="cuda")[:, None] - torch.arange(W, device="cuda") + W - 1
    dfull = dfull.permute(0, 1, 3, 2)[:, r, torch.arange(W, device="cuda")].sum(2)
    if c["state"]:
        dfull[:, T:] += s["dstate"].float()
    out.append(dfull[:, W - 1:].to(dt).reshape(s["x"].shape))
    out.append((g[..., None] * win).sum((0, 1)).to(dt))
    if c["bias"]:
        out.append(g.sum((0, 1)).to(dt))
    if c["state"]:
        out.append(dfull[:, :W - 1].to(dt))
    return out


def _plain_conv_step(s):
    x = s["x"].float()
    full = torch.cat((s["hist"].float(), x[:, None]), 1)            # (B, W, C)
    p = (full * s["w"].float().t()).sum(1)
    if s["b"] is not None:
        p = p + s["b"].float()
    y = p * torch.sigmoid(p) if s["case"]["silu"] else p
    s["hist"].copy_(full[:, 1:])
    return y.to(s["x"].dtype), s["hist"]


def _recurrence(a, u, h0):
    """h[t] = a[t] h[t-1] + u[t] along dim 0: blocks of about sqrt(T) steps side by side, then block after block."""
    T = a.shape[0]
    Q = max(1, math.isqrt(T))
    K = -(-T // Q)
    if K * Q > T:
        a = torch.cat((a, a.new_ones(K * Q - T, *a.shape[1:])))
        u = torch.cat((u, u.new_zeros(K * Q - T, *u.shape[1:])))
    a, h = a.view(K, Q, *a.shape[1:]).clone(), u.view(K, Q, *u.shape[1:]).clone()
    for q in range(1, Q):                                           # inside all blocks at once
        h[:, q].addcmul_(a[:, q], h[:, q - 1])
        a[:, q] *= a[:, q - 1]                                      # decay from the block's start
    h[0].addcmul_(a[0], h0)
    for k in range(1, K):
        h[k].addcmul_(a[k], h[k - 1, -1])
    return h.flatten(0, 1)[:T]


def _plain_scan(s):
    c = s["case"]
    T, C, N, G, dt = c["T"], c["C"], c["N"], c["G"], s["x"].dtype
    tf = lambda v: v.detach().float().reshape(-1, T, *v.shape[v.dim() - 1:]).transpose(0, 1)         # noqa: E731  (T, B, .)
    tn = lambda v: v.detach().float().reshape(-1, T, G, N).transpose(0, 1)                           # noqa: E731
    wide = lambda v: v.repeat_interleave(C // G, 2)                                                  # noqa: E731  (T, B, C, N)
    x, raw, A, D = tf(s["x"]), tf(s["dt"]), s["A"].detach(), s["D"].detach()
    raw = raw + s["bias"].detach()
    d = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20))))
    Bm, Cm = tn(s["Bm"]), tn(s["Cm"])
    a = torch.exp(d[..., None] * A)
    first = (_starts(s, T) == torch.arange(T, device="cuda")) if c["seqs"] else None
    if first is not None:
        a = a * (~first)[:, None, None, None]
    B = x.shape[1]
    h0 = s["hist"].detach() if c["state"] else x.new_zeros(B, C, N)
    u = (d * x)[..., None] * wide(Bm)
    h = _recurrence(a, u, h0)
    y = (h * wide(Cm)).sum(-1) + D * x
    z = tf(s["z"]) if c["gate"] else None
    o = y * z * torch.sigmoid(z) if c["gate"] else y
    back = lambda v, like: v.transpose(0, 1).reshape(like.shape).to(like.dtype)                      # noqa: E731
    out = [back(o, s["x"])] + ([h[-1].clone()] if c["state"] else [])
    if not c["grad"]:
        return out
    dy = tf(s["dy"])
    e = dy * z * torch.sigmoid(z) if c["gate"] else dy
    seed = e[..., None] * wide(Cm)
    if c["state"]:
        seed[-1] += s["dstate"]
    nxt = torch.cat((a[1:], a.new_zeros(1, *a.shape[1:])))
    dh = _recurrence(nxt.flip(0), seed.flip(0), torch.zeros_like(h0)).flip(0)
    del seed, nxt
    dCm = (e[..., None] * h).unflatten(2, (G, C // G)).sum(3)
    dBm = ((d * x)[..., None] * dh).unflatten(2, (G, C // G)).sum(3)
    dhB = (dh * wide(Bm)).sum(-1)
    dx = d * dhB + D * e
    kept = dh * torch.cat((h0[None], h[:-1])) * a                   # dh a h[t-1]
    dA = (kept * d[..., None]).sum((0, 1))
    dd = (kept * A).sum(-1) + x * dhB
    draw_ = torch.where(raw > 20, dd, dd * torch.sigmoid(raw))
    out += [back(dx, s["x"]), back(draw_, s["dt"]), dA, back(dBm, s["Bm"]), back(dCm, s["Cm"]), (e * x).sum((0, 1))]
    if c["gate"]:
        out.append(back(dy * y * _silu_slope(z), s["z"]))
    out.append(draw_.sum((0, 1)))
    if c["state"]:
        out.append(a[0] * dh[0])
    return out


def _plain_scan_step(s):
    x, raw = s["x"].float(), s["dt"].float() + s["bias"]
    C, G = s["case"]["C"], s["case"]["G"]
    d = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw.clamp(max=20))))
    wide = lambda v: v.float().repeat_interleave(C // G, 1)         # noqa: E731
    h = s["h"] * torch.exp(d[..., None] * s["A"]) + (d * x)[..., None] * wide(s["Bm"])
    y = (h * wide(s["Cm"])).sum(-1) + s["D"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z * torch.sigmoid(z)
    s["h"].copy_(h)
    return y.to(s["x"].dtype), s["h"]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan,
                "scan_step": _plain_scan_step}[state["case"]["op"]](state)


# ---- the definitions in 64 bits, written token by token and tap by tap ------------------------------

def _exact_rotary(s):
    c = s["case"]
    R, P = c["R"], c["R"] // 2
    pos = (s["positions"] if s["positions"] is not None else torch.arange(c["L"], device="cuda").expand(c["B"], -1)).double()

    def turned(x, sign):
        o = x.detach().double()
        o = o.transpose(1, 2).contiguous() if c["layout"] == "bhld" else o.clone()       # (B, L, H, D)
        for i in range(P):
            m, n = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + P)
            w = torch.polar(torch.full_like(pos, s["factor"]), sign * pos * s["freqs"][i])[:, :, None]
            v = torch.complex(o[..., m], o[..., n]) * w
            o[..., m], o[..., n] = v.real, v.imag
        return o.transpose(1, 2).contiguous() if c["layout"] == "bhld" else o

    out = [turned(s["q"], 1.0), turned(s["k"], 1.0)]
    return out + [turned(s["dq"], -1.0), turned(s["dk"], -1.0)] if c["grad"] else out


def _rows(s, T):
    """(first token, end) of every run of tokens that is one sequence (in every row of the batch)."""
    return list(zip(s["bounds"][:-1], s["bounds"][1:])) if s["cu"] is not None else [(0, T)]


def _exact_conv(s):
    c = s["case"]
    W, T, C = c["W"], c["T"], c["C"]
    x = s["x"].detach().double().reshape(-1, T, C)
    w = s["w"].detach().double()
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    dw, db = torch.zeros_like(w), w.new_zeros(C)
    dy = s["dy"].double().reshape(x.shape) if c["grad"] else None
    last = dhist = None
    for lo, hi in _rows(s, T):
        n = hi - lo
        before = s["hist"].detach().double() if c["state"] else x.new_zeros(x.shape[0], W - 1, C)
        f = torch.cat((before, x[:, lo:hi]), 1)
        p = s["b"].detach().double().expand(x.shape[0], n, -1).clone() if c["bias"] else x.new_zeros(x.shape[0], n, C)
        for j in range(W):
            p += f[:, j:j + n] * w[:, j]
        sg = torch.sigmoid(p)
        y[:, lo:hi] = p * sg if c["silu"] else p
        last = f[:, n:]
        if c["grad"]:
            g = dy[:, lo:hi] * (sg + p * sg * (1 - sg) if c["silu"] else 1)
            df = torch.zeros_like(f)
            for j in range(W):
                df[:, j:j + n] += g * w[:, j]
                dw[:, j] += (g * f[:, j:j + n]).sum((0, 1))
            if c["state"]:
                df[:, n:] += s["dstate"].double()
            dx[:, lo:hi], dhist = df[:, W - 1:], df[:, :W - 1]
            db += g.sum((0, 1))
    out = [y.reshape(s["x"].shape)] + ([last] if c["state"] else [])
    if c["grad"]:
        out += [dx.reshape(s["x"].shape), dw] + ([db] if c["bias"] else []) + ([dhist] if c["state"] else [])
    return out


def _exact_conv_step(s):
    f = torch.cat((s["hist"].double(), s["x"].double()[:, None]), 1)
    p = torch.einsum("bwc,cw->bc", f, s["w"].double())
    if s["b"] is not None:
        p = p + s["b"].double()
    return (p * torch.sigmoid(p) if s["case"]["silu"] else p), f[:, 1:].contiguous()


def _exact_scan(s):
    c = s["case"]
    T, C, N, G = c["T"], c["C"], c["N"], c["G"]
    dbl = lambda v, *tail: v.detach().double().reshape(-1, T, *tail)                                 # noqa: E731
    x, raw = dbl(s["x"], C), dbl(s["dt"], C) + s["bias"].detach().double()
    Bm, Cm = dbl(s["Bm"], G, N), dbl(s["Cm"], G, N)
    A, D = s["A"].detach().double(), s["D"].detach().double()
    d = F.softplus(raw)                                             # beyond 20 it is the value itself, as defined
    z = dbl(s["z"], C) if c["gate"] else None
    gate = z * torch.sigmoid(z) if c["gate"] else torch.ones_like(x)
    y, grad = torch.zeros_like(x), c["grad"]
    e = dbl(s["dy"], C) * gate if grad else None
    dx, dd = torch.zeros_like(x), torch.zeros_like(x)
    dB, dC, dA = torch.zeros_like(Bm), torch.zeros_like(Cm), torch.zeros_like(A)
    last = dhist = None
    spread = lambda v: v.repeat_interleave(C // G, 1)                                                # noqa: E731
    for lo, hi in _rows(s, T):
        h = s["hist"].detach().double() if c["state"] else x.new_zeros(x.shape[0], C, N)
        before = x.new_empty(hi - lo, *h.shape) if grad else None
        for t in range(lo, hi):
            if grad:
                before[t - lo] = h
            h = h * torch.exp(d[:, t, :, None] * A) + (d[:, t] * x[:, t])[..., None] * spread(Bm[:, t])
            y[:, t] = (h * spread(Cm[:, t])).sum(-1)
        last = h
        if not grad:
            continue
        dh = s["dstate"].double().clone() if c["state"] else torch.zeros_like(h)
        for t in range(hi - 1, lo - 1, -1):
            Bt, dtt, xt = spread(Bm[:, t]), d[:, t, :, None], x[:, t, :, None]
            am = torch.exp(dtt * A)
            kept = before[t - lo] * am
            now = kept + dtt * xt * Bt
            dh = dh + e[:, t, :, None] * spread(Cm[:, t])
            dC[:, t] = (e[:, t, :, None] * now).unflatten(1, (G, C // G)).sum(2)
            dB[:, t] = (dh * dtt * xt).unflatten(1, (G, C // G)).sum(2)
            dx[:, t] = (dh * dtt * Bt).sum(-1)
            kept = dh * kept
            dd[:, t] = (kept * A + dh * xt * Bt).sum(-1)
            dA += (kept * dtt).sum(0)
            dh = dh * am
        dhist = dh
    plain = y + D * x
    out = [(plain * gate).reshape(s["x"].shape)] + ([last] if c["state"] else [])
    if not grad:
        return out
    dd = torch.where(raw > 20, dd, dd * torch.sigmoid(raw))
    out += [(dx + D * e).reshape(s["x"].shape), dd.reshape(s["dt"].shape), dA, dB.reshape(s["Bm"].shape),
            dC.reshape(s["Cm"].shape), (e * x).sum((0, 1))]
    if c["gate"]:
        sg = torch.sigmoid(z)
        out.append((dbl(s["dy"], C) * plain * (sg + z * sg * (1 - sg))).reshape(s["z"].shape))
    return out + [dd.sum((0, 1))] + ([dhist] if c["state"] else [])


def _exact_scan_step(s):
    x, raw = s["x"].double(), s["dt"].double() + s["bias"].double()
    d, wide = F.softplus(raw), lambda v: v.double().repeat_interleave(s["case"]["C"] // s["case"]["G"], 1)
    h = torch.exp(d[..., None] * s["A"].double()) * s["h"].double() + d[..., None] * x[..., None] * wide(s["Bm"])
    y = torch.einsum("bcn,bcn->bc", h, wide(s["Cm"])) + s["D"].double() * x
    if s["z"] is not None:
        y = y * F.silu(s["z"].double())
    return y, h


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        return {"rotary": _exact_rotary, "conv": _exact_conv, "conv_step": _exact_conv_step, "scan": _exact_scan,
                "scan_step": _exact_scan_step}[case["op"]](s)


# ---- what one pass cannot do without ---------------------------------------------------------------

def work(case):
    c, e = case, _TYPES[case["dtype"]].itemsize
    op = c["op"]
    if op == "rotary":
        n = c["B"] * c["L"] * (c["H"] + c["Hk"])
        times = 2 if c["grad"] else 1
        by = times * 2 * n * c["D"] * e + c["R"] // 2 * 8 + (c["B"] * c["L"] * 8 if c["positions"] == "far" else 0)
        return {"bytes": by, "flops": times * 3 * n * c["R"]}
    if op == "conv_step":
        n = c["B"] * c["C"]
        return {"bytes": (2 * n + 2 * n * (c["W"] - 1) + c["C"] * (c["W"] + bool(c["bias"]))) * e,
                "flops": n * (2 * c["W"] + 4 * c["silu"])}
    if op == "scan_step":
        n = c["B"] * c["C"]
        return {"bytes": (3 + c["gate"]) * n * e + 2 * c["B"] * c["G"] * c["N"] * e + 8 * n * c["N"]
                + c["C"] * (c["N"] + 2) * 4, "flops": n * (7 * c["N"] + 10)}
    n = c["B"] * c["T"] * c["C"]
    if op == "conv":
        par, hist = c["C"] * (c["W"] + bool(c["bias"])), c["B"] * c["C"] * (c["W"] - 1) if c["state"] else 0
        big = 4 if c["grad"] else 2                                 # x, y; dy, dx
        return {"bytes": (big * n + (2 * par if c["grad"] else par) + (4 if c["grad"] else 2) * hist) * e,
                "flops": n * (2 * c["W"] + 4 * c["silu"]) * (3 if c["grad"] else 1)}
    bc = 2 * c["B"] * c["T"] * c["G"] * c["N"]
    par, hist = c["C"] * (c["N"] + 2) * 4, c["B"] * c["C"] * c["N"] * 4 if c["state"] else 0
    big = (3 + c["gate"]) * (2 if c["grad"] else 1)                 # x, dt, z, y; their gradients
    return {"bytes": (big * n + bc * (2 if c["grad"] else 1)) * e + par * (2 if c["grad"] else 1)
            + hist * (4 if c["grad"] else 2), "flops": n * c["N"] * (27 if c["grad"] else 7)}
