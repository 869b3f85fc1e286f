"""Short causal convolution: formulas and refusals on the CPU, the kernels on the GPU.

Tolerances, in fp32 roundings relative to the sum of the absolute terms: W products and sums and the bias
round W + 1 times; the sigmoid is good to 2^-21 (8 roundings) and passes on its argument's error (slope at
most 1.1): forward 16.  g = dy y'(p) has that and three products: 24; dx adds W more: 32.  dw and dbias add
one per token summed."""
import pytest
import torch

from oracle import seq_oracle as Q
from seq_helpers import DTYPES, cuda, leaf, randn, within

from flash_bla.ops.selective_scan.conv import causal_conv1d, causal_conv1d_step
from flash_bla.ops.selective_scan.naive import by_sequence, naive_causal_conv1d

FWD, BWD = 16, 32


# ---- CPU ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("cu", [None, [0, 1, 1, 4, 11]])
def test_oracle_matches_autograd_and_differences(silu, cu):
    rn = randn(1)
    C, W, T = 5, 4, 11
    B = 2 if cu is None else 1
    n = B if cu is None else len(cu) - 1
    x, w, b, init = (rn(*s, dtype=torch.float64).requires_grad_() for s in ((B, T, C), (C, W), (C,), (n, W - 1, C)))
    dy, df = rn(B, T, C, dtype=torch.float64), rn(n, W - 1, C, dtype=torch.float64)
    act = "silu" if silu else None

    def fwd(x, w, b, init):
        if cu is None:
            return naive_causal_conv1d(x, w, b, act, init)
        y, f = by_sequence(lambda ts, s: naive_causal_conv1d(ts[0], w, b, act, s), torch.tensor(cu), [x[0]], init)
        return y[None], f

    y, f = fwd(x, w, b, init)
    grads = torch.autograd.grad((y, f), (x, w, b, init), (dy, df))
    ref = Q.conv(x, w, b, silu, init, dy, df, None if cu is None else torch.tensor(cu))
    for got, key in zip((y, f) + grads, ("y", "final", "dx", "dw", "db", "dinit")):
        assert torch.allclose(got, ref[key], atol=1e-11), key
    e = torch.zeros_like(w)
    e[2, 1] = 1e-6
    num = sum(((p - m) * g).sum() for p, m, g in zip(fwd(x, w + e, b, init), fwd(x, w - e, b, init), (dy, df))) / 2e-6
    assert abs(num.item() - ref["dw"][2, 1].item()) < 1e-6


def test_refusals_on_cpu():
    x, w, b = torch.zeros(2, 5, 6), torch.zeros(6, 4), torch.zeros(6)
    cu = torch.tensor([0, 5], dtype=torch.int32)

    def refused(exc, match, x=x, w=w, b=b, **kw):
        with pytest.raises(exc, match=match):
            causal_conv1d(x, w, b, **kw)

    refused(RuntimeError, "CUDA")
    refused(ValueError, "shape", x=x[0])
    refused(ValueError, "shape", cu_seqlens=cu)
    refused(ValueError, "channels", w=w[:5], b=None)
    refused(ValueError, "width", w=torch.zeros(6, 5))
    refused(ValueError, "width", w=torch.zeros(6, 1))
    refused(TypeError, "dtype", x=x.double())
    refused(TypeError, "weight", w=w.half())
    refused(ValueError, "bias", b=b[:5])
    refused(ValueError, "bias", b=b.half())
    refused(ValueError, "activation", activation="relu")
    refused(ValueError, "initial_state", initial_state=torch.zeros(2, 4, 6))
    refused(ValueError, "initial_state", initial_state=torch.zeros(2, 3, 6).half())
    refused(ValueError, "int32", x=x[0], cu_seqlens=cu.long())
    refused(ValueError, "int32", x=x[0], cu_seqlens=cu[:1])
    refused(ValueError, "channels", x=x[..., :0], w=w[:0], b=None)

    def step_refused(exc, match, x=x[:, 0], s=torch.zeros(2, 3, 6), w=w, b=b, **kw):
        with pytest.raises(exc, match=match):
            causal_conv1d_step(x, s, w, b, **kw)

    step_refused(RuntimeError, "CUDA")
    step_refused(ValueError, "shape", x=x)
    step_refused(ValueError, "state", s=torch.zeros(2, 4, 6))
    step_refused(ValueError, "state", s=torch.zeros(2, 3, 6).half())
    step_refused(ValueError, "contiguous", s=torch.zeros(2, 6, 3).transpose(1, 2))
    step_refused(RuntimeError, "gradient", w=w.clone().requires_grad_())


def test_library_refuses_without_a_device():
    import ctypes
    from flash_bla import _C
    L = _C.lib()
    p = _C.ConvProblem(0, 0, 2, 8, 4, 0, 0, 0, 16)
    assert L.fbla_causal_conv_workspace_bytes(ctypes.byref(p)) > 0
    assert L.fbla_causal_conv_fwd(ctypes.byref(p), *[None] * 7) == 1 and b"NULL" in L.fbla_last_error()
    for field, value, word in (("width", 5, b"width"), ("dtype", 3, b"dtype"), ("weight_dtype", 2, b"weight_dtype"),
                               ("channels", 0, b"channels"), ("seq_len", -1, b"seq_len"), ("batch", 65536, b"batch")):
        bad = _C.ConvProblem(0, 0, 2, 8, 4, 0, 0, 0, 16)
        setattr(bad, field, value)
        assert L.fbla_causal_conv_workspace_bytes(ctypes.byref(bad)) == -1 and word in L.fbla_last_error()
    p.cu_seqlens = 16                   # packed rows want batch 1; nothing is read from the address
    assert L.fbla_causal_conv_workspace_bytes(ctypes.byref(p)) == -1 and b"packed" in L.fbla_last_error()
    p = _C.ConvProblem(0, 0, 2, 8, 4, 0, 0, 0, 16)
    assert L.fbla_causal_conv_bwd(ctypes.byref(p), 16, 16, None, None, 16, None, 16, 16, None, None, None, 0, None) == 4


# ---- GPU ------------------------------------------------------------------------------------------
gpu = pytest.mark.gpu


def run(x, w, b, act, init, dy, df, cu=None):
    """The operator's outputs and gradients, keyed as the oracle keys them."""
    xs = [leaf(t) for t in (x, w, b, init)]
    y, f = causal_conv1d(xs[0], xs[1], xs[2], activation=act, initial_state=xs[3], return_final_state=True,
                         cu_seqlens=cuda(cu))
    torch.autograd.backward((y, f), (dy.cuda(), df.cuda()))
    grads = [None if t is None else t.grad for t in xs]
    return dict(zip(("y", "final", "dx", "dw", "db", "dinit"), [y, f] + grads))


def compare(got, x, w, b, act, init, dy, df, cu=None):
    packed = cu is not None
    lift = (lambda t: t[None]) if packed else (lambda t: t)
    args = (lift(x), w, b, act == "silu", init, lift(dy), df, cu)
    ref, major = Q.conv(*args), Q.conv(*args, absolute=True)
    tokens = x.numel() // x.shape[-1]
    for key, k in (("y", FWD), ("final", 0), ("dx", BWD), ("dw", BWD + tokens), ("db", BWD + tokens), ("dinit", BWD)):
        if got[key] is not None:
            r, m = (d[key][0] if packed and key in ("y", "dx") else d[key] for d in (ref, major))
            within(got[key], r, m, k, key)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,C,W", [(1, 1, 1, 4), (2, 2, 8, 4), (3, 5, 17, 3), (2, 67, 64, 2), (1, 300, 40, 4), (5, 33, 520, 3)])
@pytest.mark.parametrize("act,bias,state", [("silu", True, True), (None, False, False), ("silu", False, True)])
def test_forward_and_backward(dtype, B, T, C, W, act, bias, state):
    rn = randn(B * 100 + T)
    x, w, dy = rn(B, T, C, dtype=dtype), rn(C, W, dtype=dtype), rn(B, T, C, dtype=dtype)
    b = rn(C, dtype=dtype) if bias else None
    init, df = rn(B, W - 1, C, dtype=dtype) if state else None, rn(B, W - 1, C, dtype=dtype)
    compare(run(x, w, b, act, init, dy, df), x, w, b, act, init, dy, df)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cu", [[0, 1, 3, 6, 10, 47], [0, 0, 2, 2, 130, 131], [0, 200], [2, 9, 40]])
@pytest.mark.parametrize("state", [False, True])
def test_packed(dtype, cu, state):
    rn = randn(len(cu))
    W, C, tail = 4, 24, 5                               # five tokens behind the last sequence
    T, n = cu[-1] + tail, len(cu) - 1
    x, w, b, dy = rn(T, C, dtype=dtype), rn(C, W), rn(C), rn(T, C, dtype=dtype)     # fp32 filters beside 16-bit inputs
    init, df = rn(n, W - 1, C, dtype=dtype) if state else None, rn(n, W - 1, C, dtype=dtype)
    cu = torch.tensor(cu, dtype=torch.int32)
    got = run(x, w, b, "silu", init, dy, df, cu)
    compare(got, x, w, b, "silu", init, dy, df, cu)
    for key in ("y", "dx"):
        assert not got[key][:cu[0]].any() and not got[key][cu[-1]:].any()


@gpu
@pytest.mark.parametrize("off", [0, 1, 8])
def test_strided_input_and_gradient(off):
    """x as a slice of a wider projection, at any offset; a gradient that is expanded over the tokens."""
    rn = randn(9)
    wide = rn(2, 20, 3 * 16 + 8, dtype=torch.bfloat16)
    x, w, g = wide[..., off:off + 16], rn(16, 4, dtype=torch.bfloat16), rn(2, 1, 16, dtype=torch.bfloat16)
    xd = wide.cuda()[..., off:off + 16].requires_grad_()
    wd = leaf(w)
    y = causal_conv1d(xd, wd)
    y.backward(g.cuda().expand(2, 20, 16))
    zero = torch.zeros(2, 3, 16)
    compare(dict(y=y, final=None, dx=xd.grad, dw=wd.grad, db=None, dinit=None), x, w, None, None, None, g.expand(2, 20, 16), zero)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,C,W", [(1, 1, 4), (3, 17, 3), (7, 256, 4), (2, 40, 2)])
def test_steps_continue_a_prompt(dtype, B, C, W):
    """A prompt and then single tokens give what the whole sequence gives, and leave its final state."""
    rn = randn(C)
    T, n = 9, 5
    x, w, b = rn(B, T + n, C, dtype=dtype), rn(C, W, dtype=dtype), rn(C, dtype=dtype)
    whole, end = causal_conv1d(x.cuda(), w.cuda(), b.cuda(), activation="silu", return_final_state=True)
    y, state = causal_conv1d(x[:, :T].cuda(), w.cuda(), b.cuda(), activation="silu", return_final_state=True)
    ref = Q.conv(x, w, b, True)
    major = Q.conv(x, w, b, True, absolute=True)
    for i in range(n):
        got = causal_conv1d_step(x[:, T + i].cuda(), state, w.cuda(), b.cuda(), activation="silu")
        within(got, ref["y"][:, T + i], major["y"][:, T + i], FWD, f"step {i}")
    assert torch.equal(state, end)
    assert torch.equal(y, whole[:, :T])


@gpu
def test_same_bits_on_every_run_and_empty_inputs():
    rn = randn(11)
    x, w, b, dy, df = rn(3, 515, 72), rn(72, 4), rn(72), rn(3, 515, 72), rn(3, 3, 72)
    a, c = (run(x, w, b, "silu", None, dy, df) for _ in range(2))
    assert all(torch.equal(a[k], c[k]) for k in ("y", "dx", "dw", "db"))
    xs = [leaf(t) for t in (x[:, :0], w, b, rn(3, 3, 72))]
    y, f = causal_conv1d(*xs[:3], initial_state=xs[3], return_final_state=True)
    (y.sum() + (f * df.cuda()).sum()).backward()
    assert y.shape == (3, 0, 72) and torch.equal(f, xs[3]) and torch.equal(xs[3].grad, df.cuda())
    assert not xs[1].grad.any() and not xs[2].grad.any()
    assert causal_conv1d_step(x[:0, 0].cuda(), torch.zeros(0, 3, 72, device="cuda"), w.cuda()).shape == (0, 72)


@gpu
def test_old_infinities_stay_in_their_window():
    x = torch.ones(1, 12, 4)
    x[0, 3, 1] = float("inf")
    y = causal_conv1d(x.cuda(), torch.ones(4, 3).cuda()).cpu()
    assert y[0, 3:6, 1].isinf().all() and int(y.isfinite().logical_not().sum()) == 3


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [22, 30, 257])
@pytest.mark.parametrize("cu", [None, [0, 3, 70, 71]])
def test_channel_counts_between_the_packs(dtype, C, cu):
    """Two channels at a time, or one, in the fixed and the packed layout."""
    rn = randn(C)
    W, n = 4, 2 if cu is None else len(cu) - 1
    lead = (2, 71) if cu is None else (71,)
    x, w, b, dy = rn(*lead, C, dtype=dtype), rn(C, W, dtype=dtype), rn(C, dtype=dtype), rn(*lead, C, dtype=dtype)
    init, df = rn(n, W - 1, C, dtype=dtype), rn(n, W - 1, C, dtype=dtype)
    cu = None if cu is None else torch.tensor(cu, dtype=torch.int32)
    compare(run(x, w, b, "silu", init, dy, df, cu), x, w, b, "silu", init, dy, df, cu)


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^32 elements: the last tokens are what they are on their own, with the inputs before them as state."""
    T, C, W = 2_200_000, 2048, 4
    x = torch.empty(1, T, C, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(0))
    w = torch.randn(C, W, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    y, end = causal_conv1d(x, w, activation="silu", return_final_state=True)
    lo = T - 50
    tail, end2 = causal_conv1d(x[:, lo:].clone(), w, activation="silu", initial_state=x[:, lo - W + 1:lo].clone(), return_final_state=True)
    assert torch.equal(y[:, lo:], tail) and torch.equal(end, end2)


@gpu
def test_many_short_sequences_and_no_token_at_all():
    """Sequences shorter than the filter, many of them empty; then packed rows without a single token."""
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 3, (700,), generator=g)
    cu = torch.cat((torch.zeros(1, dtype=torch.long), lengths.cumsum(0))).int()
    rn = randn(12)
    T, C, n = int(cu[-1]), 12, 700
    x, w, b, dy, init, df = rn(T, C), rn(C, 4), rn(C), rn(T, C), rn(n, 3, C), rn(n, 3, C)
    compare(run(x, w, b, "silu", init, dy, df, cu), x, w, b, "silu", init, dy, df, cu)
    none = torch.zeros(4, dtype=torch.int32)
    got = run(x[:0], w, b, None, init[:3], dy[:0], df[:3], none)
    assert got["y"].shape == (0, C) and torch.equal(got["final"].cpu(), init[:3]) and torch.equal(got["dinit"].cpu(), df[:3])
    assert not got["dw"].any() and not got["db"].any()


@gpu
def test_backward_offsets_beyond_32_bits():
    """More than 2^31 elements: gradients of the last tokens are what they are on their own.  dy is zero but for the first
    and the last 50 tokens, so the filter's gradient is the sum of two short calls'."""
    T, C, W, n = 1_060_000, 2048, 4, 50
    g = torch.Generator("cuda").manual_seed(2)
    x = torch.empty(1, T, C, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = torch.randn(C, W, device="cuda", generator=g)
    dy = torch.zeros_like(x)
    for part in (dy[:, :n], dy[:, -n:]):
        part.normal_(generator=g)

    def grads(x, dy, state=None):
        x, v = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = causal_conv1d(x, v, activation="silu", initial_state=state)
        return torch.autograd.grad(y, (x, v), dy)

    dx, dw = grads(x, dy)
    tail, dw_tail = grads(x[:, -n:].clone(), dy[:, -n:].clone(), x[:, -n - W + 1:-n].clone())
    head, dw_head = grads(x[:, :n].clone(), dy[:, :n].clone())
    assert torch.equal(dx[:, -n:], tail) and torch.equal(dx[:, :n], head)
    # 2 n terms g x, |g| at most 1.1 |dy|, each product and each sum rounded once, on both sides
    size = 1.1 * (dy[0, :n].abs().float().sum(0) + dy[0, -n:].abs().float().sum(0)) * x.abs().max().float()
    assert ((dw - dw_head - dw_tail).abs() <= 2 * (2 * n + 1) * 2.0 ** -24 * size[:, None]).all()
