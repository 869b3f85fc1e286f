"""Selective scan: formulas and refusals on the CPU, the kernels on the GPU.

Tolerances, in fp32 roundings (2^-24) relative to the sum of the absolute terms.  A decay a = exp(d A) has
the error of d (softplus: 4 units, weighted by |d A| a <= 0.37), of the product, and of the exponential
(2^-22 at most): 6; with the rounding of h itself 7, and d x B three: a state that remembers L tokens is
within 8 L + 8, and a gradient, which runs through the states and back, within twice that.  y adds N
products and sums and the gate (the sigmoid is good to 2^-21: 8 units): N + 16.  dB, dC add one per channel
summed, dA, dD and dbias one per token."""
import pytest
import torch

from oracle import seq_oracle as Q
from seq_helpers import DTYPES, cuda, leaf, randn, within

from flash_bla.ops.selective_scan.naive import by_sequence, naive_selective_scan
from flash_bla.ops.selective_scan.scan import selective_scan, selective_scan_step

NAMES = ("x", "dt", "A", "B", "C", "D", "z", "bias", "init")
GRADS = ("dx", "ddt", "dA", "dB", "dC", "dD", "dz", "dbias", "dinit")


def inputs(seed, lead, C, G, N, dtype, rows, D=True, z=True, bias=True, state=True):
    rn = randn(seed)
    t = dict(x=rn(*lead, C, dtype=dtype), dt=rn(*lead, C, dtype=dtype, scale=0.5, shift=0.0 if bias else -3.0),
             A=-torch.exp(rn(C, N, scale=0.8)), B=rn(*lead, G, N, dtype=dtype), C=rn(*lead, G, N, dtype=dtype),
             D=rn(C) if D else None, z=rn(*lead, C, dtype=dtype) if z else None, bias=rn(C, shift=-3.0) if bias else None,
             init=rn(rows, C, N) if state else None)
    return t, rn(*lead, C, dtype=dtype), rn(rows, C, N)


# ---- CPU ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cu", [None, [0, 1, 1, 4, 11]])
@pytest.mark.parametrize("softplus", [False, True])
def test_oracle_matches_autograd_and_differences(cu, softplus):
    T, C, G, N = 11, 6, 2, 3
    rows = 2 if cu is None else len(cu) - 1
    t, dy, df = inputs(0, (2, T) if cu is None else (T,), C, G, N, torch.float64, rows)
    t = {k: v.double().requires_grad_() for k, v in t.items()}
    df = df.double()
    order = ("x", "dt", "B", "C", "z")

    def fwd(t):
        if cu is None:
            return naive_selective_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], t["D"], t["z"], t["bias"], softplus, t["init"])
        return by_sequence(lambda v, s: naive_selective_scan(v[0], v[1], t["A"], v[2], v[3], t["D"], v[4], t["bias"], softplus, s),
                           torch.tensor(cu), [t[k] for k in order], t["init"])

    y, f = fwd(t)
    grads = torch.autograd.grad((y, f), [t[k] for k in NAMES], (dy, df))
    lift = (lambda v: v) if cu is None else (lambda v: v[None])
    ref = Q.scan(lift(t["x"]), lift(t["dt"]), t["A"], lift(t["B"]), lift(t["C"]), t["D"], lift(t["z"]), t["bias"], softplus, t["init"],
                 lift(dy), df, None if cu is None else torch.tensor(cu))
    assert torch.allclose(lift(y), ref["y"], atol=1e-11) and torch.allclose(f, ref["final"], atol=1e-11)
    for got, name, key in zip(grads, NAMES, GRADS):
        assert torch.allclose(lift(got) if name in order else got, ref[key], atol=1e-10), key
    e = torch.zeros_like(t["A"])
    e[1, 2] = 1e-6
    num = sum(((p - m) * g).sum() for p, m, g in zip(fwd(dict(t, A=t["A"] + e)), fwd(dict(t, A=t["A"] - e)), (dy, df))) / 2e-6
    # Rounding: both sums are within 100 roundings (8 per token and the sum's own) of 2^-53 of their absolute
    # terms, whose difference is divided by 2e-6.  Truncation: the third derivative is at most (sum d)^2 < 40^2
    # times the first, by 1e-12 / 6.  Without softplus a negative step size lets a state grow without bound, and
    # the terms with it, so neither is an absolute number.
    terms = sum((v.abs() * g.abs()).sum() for v, g in zip((y, f), (dy, df))).item()
    assert abs(num.item() - ref["dA"][1, 2].item()) < 100 * 2.0 ** -53 * 2 * terms / 2e-6 + 1e-9 * abs(ref["dA"][1, 2].item())


def test_refusals_on_cpu():
    t, _, _ = inputs(1, (2, 5), 6, 2, 4, torch.float32, 2)

    def refused(exc, match, step=False, **kw):
        a = dict(t, **{k: v for k, v in kw.items() if k in t})
        kw = {k: v for k, v in kw.items() if k not in t}
        with pytest.raises(exc, match=match):
            selective_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["bias"], initial_state=a["init"], **kw)

    refused(RuntimeError, "CUDA")
    refused(ValueError, "shape", x=t["x"][0])
    refused(TypeError, "dtype", x=t["x"].double())
    refused(ValueError, "dt must", dt=t["dt"][:, :4])
    refused(ValueError, "z must", z=t["z"].half())
    refused(ValueError, "A must", A=t["A"].half())
    refused(ValueError, "A must", A=t["A"][:5])
    refused(ValueError, "states", A=torch.zeros(6, 33))
    refused(ValueError, "B must", B=t["B"][..., :3])
    refused(ValueError, "C must", C=t["C"].half())
    refused(ValueError, "same shape", C=t["C"][:, :, :1])
    refused(ValueError, "groups", B=torch.zeros(2, 5, 4, 4), C=torch.zeros(2, 5, 4, 4))
    refused(ValueError, "groups", B=torch.zeros(2, 5, 0, 4), C=torch.zeros(2, 5, 0, 4))
    refused(ValueError, "D must", D=t["D"].half())
    refused(ValueError, "dt_bias must", bias=t["bias"][:5])
    refused(ValueError, "initial_state", init=t["init"][:1])
    refused(ValueError, "initial_state", init=t["init"].double())
    refused(ValueError, "no channels", x=t["x"][..., :0])
    refused(ValueError, "shape", cu_seqlens=torch.tensor([0, 5], dtype=torch.int32))

    def step_refused(exc, match, **kw):
        a = dict(x=t["x"][:, 0], dt=t["dt"][:, 0], A=t["A"], B=t["B"][:, 0], C=t["C"][:, 0], state=t["init"])
        with pytest.raises(exc, match=match):
            selective_scan_step(**dict(a, **kw))

    step_refused(RuntimeError, "CUDA")
    step_refused(ValueError, "shape", x=t["x"])
    step_refused(ValueError, "state", state=t["init"][:1])
    step_refused(ValueError, "contiguous", state=torch.zeros(2, 4, 6).transpose(1, 2))
    step_refused(ValueError, "aligned", state=torch.zeros(2 * 6 * 4 + 1)[1:].view(2, 6, 4))
    step_refused(RuntimeError, "gradient", A=t["A"].clone().requires_grad_())


def test_library_refuses_without_a_device():
    import ctypes
    from flash_bla import _C
    L = _C.lib()
    ok = lambda: _C.ScanProblem(1, 2, 64, 16, 1, 1, 0, 0, 100)      # noqa: E731
    p = ok()
    assert L.fbla_selective_scan_checkpoint_floats(ctypes.byref(p)) > 0
    assert L.fbla_selective_scan_workspace_bytes(ctypes.byref(p), 1) > 0
    assert L.fbla_selective_scan_fwd(ctypes.byref(p), *[None] * 13, 0, None) == 1 and b"NULL" in L.fbla_last_error()
    for field, value, word in (("states", 33, b"states"), ("states", 0, b"states"), ("groups", 3, b"groups"), ("dtype", 5, b"dtype"),
                               ("channels", 0, b"channels"), ("seq_len", -1, b"seq_len"), ("batch", 70000, b"batch")):
        bad = ok()
        setattr(bad, field, value)
        assert L.fbla_selective_scan_workspace_bytes(ctypes.byref(bad), 0) == -1 and word in L.fbla_last_error()
    a = [16] * 10
    assert L.fbla_selective_scan_step(ctypes.byref(p), *a[:8], 8, 16, None) == 1 and b"aligned" in L.fbla_last_error()


# ---- GPU ------------------------------------------------------------------------------------------
gpu = pytest.mark.gpu


def run(t, dy, df, softplus, cu=None):
    v = {k: leaf(x) for k, x in t.items()}
    y, f = selective_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], dt_softplus=softplus,
                          initial_state=v["init"], return_final_state=True, cu_seqlens=cuda(cu))
    torch.autograd.backward((y, f), (dy.cuda(), df.cuda()))
    return dict(y=y, final=f, **{g: None if v[k] is None else v[k].grad for k, g in zip(NAMES, GRADS)})


def compare(got, t, dy, df, softplus, cu=None):
    packed = cu is not None
    lift = lambda v: v[None] if packed and v is not None else v     # noqa: E731
    args = (lift(t["x"]), lift(t["dt"]), t["A"], lift(t["B"]), lift(t["C"]), t["D"], lift(t["z"]), t["bias"], softplus, t["init"],
            lift(dy), df, cu)
    ref, major = Q.scan(*args), Q.scan(*args, absolute=True)
    T, (C, N) = lift(t["x"]).shape[1], t["A"].shape
    tokens = t["x"].numel() // C
    st = 8 * T + 8
    k = dict(y=st + N + 16, final=st, dx=2 * st + N + 32, ddt=2 * st + N + 32, dA=2 * st + tokens + 32, dB=2 * st + C + 32,
             dC=st + C + 32, dD=tokens + 32, dz=st + N + 32, dbias=2 * st + N + tokens + 32, dinit=2 * st + 32)
    for key, n in k.items():
        if got.get(key) is not None:
            r, m = (d[key][0] if packed and key in ("y", "dx", "ddt", "dB", "dC", "dz") else d[key] for d in (ref, major))
            within(got[key], r, m, n, key)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,C,G,N", [(1, 1, 1, 1, 1), (2, 3, 8, 1, 16), (2, 33, 70, 1, 16), (1, 64, 130, 2, 8), (3, 31, 64, 1, 5),
                                       (1, 45, 24, 3, 32), (2, 19, 65, 1, 20), (1, 257, 16, 1, 3)])
def test_forward_and_backward(dtype, B, T, C, G, N):
    t, dy, df = inputs(T, (B, T), C, G, N, dtype, B)
    compare(run(t, dy, df, True), t, dy, df, True)


@gpu
@pytest.mark.parametrize("missing", [("D",), ("z",), ("bias",), ("init",), ("D", "z", "bias", "init")])
@pytest.mark.parametrize("softplus", [False, True])
def test_optional_arguments(missing, softplus):
    t, dy, df = inputs(5, (2, 40), 24, 1, 16, torch.bfloat16, 2, **{"state" if k == "init" else k: False for k in missing})
    if not softplus:                    # step sizes are positive in earnest
        t["dt"] = t["dt"].abs() * 0.2
        t["bias"] = None if t["bias"] is None else t["bias"].abs() * 0.02
    compare(run(t, dy, df, softplus), t, dy, df, softplus)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1024, 1000])
def test_segments(dtype, T):
    """Few channels and many tokens: the tokens are cut into segments."""
    t, dy, df = inputs(6, (1, T), 72, 1, 16, dtype, 1)
    compare(run(t, dy, df, True), t, dy, df, True)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [16, 8, 24])
@pytest.mark.parametrize("cu", [[0, 1, 3, 6, 10, 47], [0, 0, 2, 2, 130, 131, 131], [0, 200], [2, 9, 40], [0, 300, 301, 700, 1000]])
@pytest.mark.parametrize("state", [False, True])
def test_packed(dtype, N, cu, state):
    T = cu[-1] + 5                      # five tokens behind the last sequence
    t, dy, df = inputs(T, (T,), 24, 1, N, dtype, len(cu) - 1, state=state)
    t["B"][-3:] = float("nan")          # nothing of theirs may show anywhere
    t["dt"][-2:] = float("inf")
    cu = torch.tensor(cu, dtype=torch.int32)
    got = run(t, dy, df, True, cu)
    clean = dict(t, B=t["B"].nan_to_num(0.0), dt=t["dt"].nan_to_num(posinf=0.0))
    compare(got, clean, dy, df, True, cu)
    for key in ("y", "dx", "ddt", "dB", "dC", "dz"):
        assert not got[key][:cu[0]].any() and not got[key][cu[-1]:].any(), key


@gpu
@pytest.mark.parametrize("off", [0, 1, 8])
def test_strided_inputs_and_gradient(off):
    """x and z as slices of one projection, B and C of another, at any offset; an expanded gradient."""
    t, _, _ = inputs(8, (2, 50), 32, 1, 16, torch.bfloat16, 2, state=False)
    xz = torch.cat((torch.zeros(2, 50, off, dtype=torch.bfloat16), t["x"], t["z"]), -1).cuda()
    bc = torch.cat((torch.zeros(2, 50, 3, dtype=torch.bfloat16), t["B"].flatten(2), t["C"].flatten(2)), -1).cuda()
    v = {k: leaf(x) for k, x in t.items()}
    v["x"], v["z"] = (xz[..., off + i * 32:off + (i + 1) * 32].requires_grad_() for i in range(2))
    v["B"], v["C"] = (bc[..., 3 + i * 16:19 + i * 16].requires_grad_() for i in range(2))      # no group dimension
    g = randn(1)(2, 1, 32, dtype=torch.bfloat16)
    y = selective_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], dt_softplus=True)
    y.backward(g.cuda().expand(2, 50, 32))
    got = dict(y=y, **{gr: v[k].grad for k, gr in zip(NAMES, GRADS) if v[k] is not None})
    for k in ("dB", "dC"):
        got[k] = got[k].unflatten(-1, (1, 16))
    compare(got, t, g.expand(2, 50, 32), None, True)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,C,G,N", [(1, 1, 1, 1), (3, 70, 1, 16), (2, 64, 2, 8), (2, 24, 1, 30)])
def test_steps_continue_a_prompt(dtype, B, C, G, N):
    T, n = 21, 4
    t, _, _ = inputs(C, (B, T + n), C, G, N, dtype, B)
    ref = Q.scan(t["x"], t["dt"], t["A"], t["B"], t["C"], t["D"], t["z"], t["bias"], True, t["init"])
    major = Q.scan(t["x"], t["dt"], t["A"], t["B"], t["C"], t["D"], t["z"], t["bias"], True, t["init"], absolute=True)
    k = 8 * (T + n) + 8
    part = lambda lo, hi: {n_: cuda(v) if v is None or n_ in ("A", "D", "bias", "init") else v[:, lo:hi].cuda() for n_, v in t.items()}  # noqa: E731
    v = part(0, T)
    with torch.no_grad():
        _, state = selective_scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["bias"], dt_softplus=True,
                                  initial_state=v["init"], return_final_state=True)
        for i in range(T, T + n):
            v = {n_: x if n_ in ("A", "D", "bias", "init") else x[:, 0] for n_, x in part(i, i + 1).items()}
            y = selective_scan_step(v["x"], v["dt"], v["A"], v["B"], v["C"], state, v["D"], v["z"], v["bias"], dt_softplus=True)
            within(y, ref["y"][:, i], major["y"][:, i], k + N + 16, f"token {i}")
    within(state, ref["final"], major["final"], k, "state")


@gpu
def test_slow_decays_do_not_drift():
    """A state that forgets almost nothing over 4096 tokens: the decays' errors must not add up one way.
    Every factor is within one rounding of fp32 of its value (2^-24) and so is every step of the state, so
    4096 steps are within 2 * 4096 roundings; a biased exponential (2^-22 each) would be four times that
    and is seen here as a relative error of the state beyond 2^-24 * 4096."""
    T = 4096
    x = torch.zeros(1, T, 64)
    x[0, 0] = 1.0
    dt = torch.full((1, T, 64), 1.0)
    A = -torch.logspace(-6, -3.5, 64)[:, None]
    one = torch.ones(1, T, 1)
    _, end = selective_scan(x.cuda(), dt.cuda(), A.cuda(), one.cuda(), one.cuda(), return_final_state=True)
    ref = torch.exp(A.double() * (T - 1))
    assert ((end[0].cpu().double() - ref).abs() <= 2.0 ** -24 * T * ref).all()


@gpu
def test_large_steps_and_masked_tokens():
    """A step size far beyond 20 (softplus is the identity), one that underflows, infinities in x of one channel."""
    t, dy, df = inputs(9, (1, 37), 16, 1, 16, torch.float32, 1)
    t["dt"][0, 3] = 60.0
    t["dt"][0, 4] = -200.0
    compare(run(t, dy, df, True), t, dy, df, True)
    t["x"][0, 5, 2] = float("inf")
    y = selective_scan(*(cuda(t[k]) for k in NAMES[:8]), dt_softplus=True).cpu()
    rest = torch.arange(16) != 2
    assert y[0, :, rest].isfinite().all() and y[0, :5].isfinite().all() and not y[0, 5:, 2].isfinite().any()


@gpu
def test_same_bits_on_every_run_and_empty_inputs():
    t, dy, df = inputs(10, (2, 515), 72, 1, 16, torch.float32, 2)
    a, b = (run(t, dy, df, True) for _ in range(2))
    assert all(torch.equal(a[k], b[k]) for k in a)
    e = {k: (v if k in ("A", "D", "bias", "init") else v[:, :0]) for k, v in t.items()}
    got = run(e, dy[:, :0], df, True)
    assert got["y"].shape == (2, 0, 72) and torch.equal(got["final"], t["init"].cuda()) and torch.equal(got["dinit"], df.cuda())
    assert not got["dA"].any() and not got["dD"].any() and not got["dbias"].any()
    e = {k: (v if k in ("A", "D", "bias") else v[:0]) for k, v in t.items()}
    got = run(e, dy[:0], df[:0], True)
    assert got["y"].shape == (0, 515, 72) and not got["dA"].any()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("C,G,N", [(23, 1, 16), (42, 2, 7), (136, 1, 16), (67, 1, 30)])
@pytest.mark.parametrize("cu", [[0, 33, 33, 34, 200], [3, 64, 96, 640]])
def test_packed_channel_counts(dtype, C, G, N, cu):
    """Rows that start off boundaries, and boundaries of sequences on and inside tiles, with segments."""
    T = cu[-1] + 2
    t, dy, df = inputs(T + C, (T,), C, G, N, dtype, len(cu) - 1)
    cu = torch.tensor(cu, dtype=torch.int32)
    compare(run(t, dy, df, True, cu), t, dy, df, True, cu)


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^32 elements: the last tokens are what they are on their own from the state before them."""
    T, C, N = 1_050_000, 4096, 4
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.empty(1, T, C, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    dt = torch.empty(1, T, C, dtype=torch.bfloat16, device="cuda").uniform_(0.01, 0.2, generator=g)
    Bm = torch.randn(1, T, N, device="cuda", generator=g).bfloat16()
    A = -torch.rand(C, N, device="cuda", generator=g) - 0.5
    y, end = selective_scan(x, dt, A, Bm, Bm, return_final_state=True)
    lo = T - 64                         # exp(-0.5 * 0.1 * 5000) leaves nothing of what came before the last 5000 tokens
    part = lambda v, a: v[:, a:].clone()                                # noqa: E731
    tail, end2 = selective_scan(part(x, lo - 6000), part(dt, lo - 6000), A, part(Bm, lo - 6000), part(Bm, lo - 6000), return_final_state=True)
    # sums of the same terms in other segments: 8 roundings for each of the 400 tokens that matter, of terms below 64
    assert (y[:, lo:].float() - tail[:, -64:].float()).abs().max() <= 2.0 ** -8 * y[:, lo:].float().abs().max() + 3200 * 2.0 ** -24 * 64
    assert (end - end2).abs().max() <= 3200 * 2.0 ** -24 * 64


@gpu
def test_many_short_sequences_and_no_token_at_all():
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 3, (500,), generator=g)
    cu = torch.cat((torch.zeros(1, dtype=torch.long), lengths.cumsum(0))).int()
    t, dy, df = inputs(12, (int(cu[-1]),), 12, 1, 16, torch.float32, 500)
    compare(run(t, dy, df, True, cu), t, dy, df, True, cu)
    none = torch.zeros(4, dtype=torch.int32)
    e = {k: v if k in ("A", "D", "bias") else v[:3] if k == "init" else v[:0] for k, v in t.items()}
    got = run(e, dy[:0], df[:3], True, none)
    assert got["y"].shape == (0, 12) and torch.equal(got["final"].cpu(), t["init"][:3]) and torch.equal(got["dinit"].cpu(), df[:3])
    assert not got["dA"].any() and not got["dD"].any() and not got["dbias"].any()


@gpu
def test_only_the_final_state_or_only_the_output_is_used():
    """A gradient that reaches one of the two results alone."""
    t, dy, df = inputs(13, (2, 40), 24, 1, 16, torch.float32, 2)
    zero = torch.zeros_like
    for use in ("y", "final"):
        v = {k: leaf(x) for k, x in t.items()}
        y, f = selective_scan(*(v[k] for k in NAMES[:8]), dt_softplus=True, initial_state=v["init"], return_final_state=True)
        (y * dy.cuda()).sum().backward() if use == "y" else (f * df.cuda()).sum().backward()
        got = dict(y=y, final=f, **{g: v[k].grad for k, g in zip(NAMES, GRADS)})
        compare(got, t, dy if use == "y" else zero(dy), df if use == "final" else zero(df), True)


@gpu
def test_a_second_derivative_is_refused():
    t, dy, _ = inputs(14, (1, 9), 8, 1, 4, torch.float32, 1)
    v = {k: leaf(x) for k, x in t.items()}
    y = selective_scan(*(v[k] for k in NAMES[:8]), dt_softplus=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, v["x"], dy.cuda(), create_graph=True)


# ---- the address of A -----------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("N", [8, 16, 32, 7])
def test_parameters_at_any_offset_of_a_flat_buffer(off, N):
    """A, D and dt_bias as views of one buffer, as an optimizer that keeps its parameters flat has them."""
    C, T = 24, 40
    t, dy, df = inputs(15 + N, (2, T), C, 1, N, torch.float32, 2)
    want = run(t, dy, df, True)
    flat = torch.cat([torch.zeros(off)] + [t[k].flatten() for k in ("A", "D", "bias")]).cuda().requires_grad_()
    at = [off, off + C * N, off + C * N + C, off + C * N + 2 * C]
    A, D, bias = (flat[lo:hi] for lo, hi in zip(at, at[1:]))
    A = A.view(C, N)
    assert A.data_ptr() % 16 and A.is_contiguous()
    v = {k: leaf(t[k]) for k in ("x", "dt", "B", "C", "z", "init")}
    y, f = selective_scan(v["x"], v["dt"], A, v["B"], v["C"], D, v["z"], bias, dt_softplus=True, initial_state=v["init"],
                          return_final_state=True)
    torch.autograd.backward((y, f), (dy.cuda(), df.cuda()))
    assert torch.equal(y, want["y"]) and torch.equal(f, want["final"])
    assert torch.equal(flat.grad[off:], torch.cat([want[k].flatten() for k in ("dA", "dD", "dbias")]))
    assert all(torch.equal(v[k].grad, want[g]) for k, g in zip(NAMES, GRADS) if k in v)
    with torch.no_grad():
        a = {k: cuda(x) if k in ("A", "D", "bias", "init") else x[:, 0].cuda() for k, x in t.items()}
        ends = [a["init"].clone() for _ in range(2)]
        ys = [selective_scan_step(a["x"], a["dt"], r, a["B"], a["C"], h, d, a["z"], b, dt_softplus=True)
              for h, (r, d, b) in zip(ends, ((a["A"], a["D"], a["bias"]), (A, D, bias)))]
    assert torch.equal(*ys) and torch.equal(*ends)


@gpu
def test_segments_whose_total_decay_leaves_the_range():
    """Three segments of 128 tokens with d A = 1 or -1: a whole segment's factor e^128 or e^-128 is beyond fp32 while
    its product with the state (zero, or 1e30) is not; the same for what comes back from behind."""
    T, C, N = 384, 64, 16
    rn = randn(20)
    up, down = slice(0, 32), slice(32, 64)
    t = dict(x=torch.zeros(1, T, C), dt=torch.full((1, T, C), 0.125), A=torch.full((C, N), 8.0), B=rn(1, T, 1, N), C=rn(1, T, 1, N),
             D=None, z=None, bias=None, init=torch.zeros(1, C, N))
    dy, df = torch.zeros(1, T, C), torch.zeros(1, C, N)
    t["A"][down] = -8.0
    t["x"][:, 340:, up], dy[:, :40, up] = rn(1, 44, 32), rn(1, 40, 32)          # nothing before it grows, or behind it
    t["init"][:, down], df[:, down] = rn(1, 32, N, scale=1e30), rn(1, 32, N, scale=1e30)
    got = run(t, dy, df, False)
    args = [t[k] for k in NAMES[:8]] + [False, t["init"], dy, df]
    ref, major = Q.scan(*args), Q.scan(*args, absolute=True)
    # As in compare(), the largest of its counts for all; beside it what underflow takes: values run down from 1e30 to
    # nothing, a state, a product or a partial sum below 2^-126 is 0, so each loses up to that, times a factor |B|, |C| < 6
    # or |A| = 8 at most, in sums of no more than T terms (N per y, dx and ddt, C per dB and dC, T per dA)
    floor = 8 * T * 2.0 ** -126
    for key in ("y", "final", "dx", "ddt", "dA", "dB", "dC", "dinit"):
        err = (got[key].detach().cpu().double() - ref[key]).abs()
        assert (err <= Q.bounds(ref[key], major[key], torch.float32, 2 * (8 * T + 8) + T + 32) + floor).all(), key
    t["init"][0, 40, 5] = float("inf")
    y = selective_scan(*(cuda(t[k]) for k in NAMES[:5]), initial_state=cuda(t["init"])).cpu()
    rest = torch.arange(C) != 40
    assert y[0, :, 40].isinf().all() and y[0, :, rest].isfinite().all()


@gpu
def test_backward_offsets_beyond_32_bits():
    """More than 2^31 elements, 2^32 floats of checkpoints and 2^31 of sums over channels: gradients of the last tokens are
    what they are on their own from the state before them.  exp(-0.5 * 0.1 * 6000) leaves nothing of what came before."""
    T, C, N, n, back = 1_050_000, 2048, 32, 64, 6000
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.empty(1, T, C, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    dt = torch.empty(1, T, C, dtype=torch.bfloat16, device="cuda").uniform_(0.01, 0.2, generator=g)
    Bm, Cm = (torch.randn(1, T, N, device="cuda", generator=g).bfloat16() for _ in range(2))
    A = -torch.rand(C, N, device="cuda", generator=g) - 0.5
    dy = torch.zeros_like(x)
    dy[:, -n:].normal_(generator=g)

    def grads(*t):
        *t, dy = (v.detach().requires_grad_() for v in t)
        y = selective_scan(t[0], t[1], A, *t[2:])
        return (y.detach(),) + torch.autograd.grad(y, t, dy.detach())

    whole = [v[:, -n:].clone() for v in grads(x, dt, Bm, Cm, dy)]
    short = [v[:, -n - back:].clone() for v in (x, dt, Bm, Cm, dy)]
    alone = [v[:, -n:].float() for v in grads(*short)]
    # the same sums with every term positive; ddt = sum A r + x sum G B has a negative part, and dx = d sum G B
    size = [v[:, -n:] for v in grads(*(v.float() if v is short[1] else v.float().abs() for v in short))]
    size[2] = 2 * short[0][:, -n:].float().abs() * size[1] / short[1][:, -n:].float() - size[2]
    for what, k, a, b, m in zip(("y", "dx", "ddt", "dB", "dC"), (1, 0, 2, 0, 1), whole, alone, size):
        # dx and dB take nothing from before: the same operations on the same numbers.  The others are sums from states
        # formed in other segments: 8 roundings for each of the 400 tokens that matter on either side, twice that for a
        # product with G, and one step of bf16 where the roundings fall apart
        err = (a.float() - b).abs()
        assert (err <= (2.0 ** -7 * b.abs() + 2 * k * 3200 * 2.0 ** -24 * m if k else torch.zeros_like(err))).all(), what


@gpu
@pytest.mark.parametrize("bad", ["nan", "-inf"])
@pytest.mark.parametrize("where", [30, 280, 310, 500])
def test_a_step_size_that_is_no_number_stays_in_its_sequence(bad, where):
    """Packed sequences over several segments (128 tokens each): a NaN or infinite step size in one of them, in the segment
    in which the next one begins too, shows in no output and no gradient of the others."""
    cu = [0, 20, 300, 305, 560, 900]
    t, dy, df = inputs(30, (cu[-1],), 24, 1, 16, torch.float32, len(cu) - 1)
    t["dt"], t["bias"] = t["dt"].abs() * 0.1, t["bias"].abs() * 0.01
    lens = torch.tensor(cu, dtype=torch.int32)
    want = run(t, dy, df, False, lens)
    t["dt"][where] = float(bad)
    got = run(t, dy, df, False, lens)
    own = max(i for i, lo in enumerate(cu) if lo <= where)
    for key in ("y", "dx", "ddt", "dB", "dC", "dz"):
        for lo, hi in (z for i, z in enumerate(zip(cu, cu[1:])) if i != own):
            assert torch.equal(got[key][lo:hi], want[key][lo:hi]), (key, lo)
    rest = torch.arange(len(cu) - 1) != own
    assert torch.equal(got["final"][rest], want["final"][rest]) and torch.equal(got["dinit"][rest], want["dinit"][rest])
    assert not got["y"][where].isfinite().any()


@gpu
@pytest.mark.parametrize("bad", ["x", "init", "dt"])
@pytest.mark.parametrize("N", [8, 16, 30])
def test_gradients_behind_the_last_sequence_stay_zero(bad, N):
    """Its last state is still in the registers there, and 0 times an infinite one is not 0."""
    cu = torch.tensor([0, 7, 40], dtype=torch.int32)
    t, dy, df = inputs(31, (75,), 24, 1, N, torch.float32, 2)
    if bad == "init":
        t["init"][1, 3, 2] = float("inf")
    else:
        t[bad][38, 3] = float("nan")
    got = run(t, dy, df, True, cu)
    assert not got["y"][38:40].isfinite().all() and not got["dC"][38:40].isfinite().all()
    for key in ("y", "dx", "ddt", "dB", "dC", "dz"):
        assert not got[key][40:].any() and got[key][:7].isfinite().all(), key
