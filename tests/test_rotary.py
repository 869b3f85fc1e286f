"""Rotary positions: formulas and refusals on the CPU, the kernel on the GPU.

Tolerance: the angle is exact to 2^-25 turns of half a circle (pi 2^-25 < 4 units of 2^-24 with the
rounding of the sine and cosine, 2 units more, and the factor's), the two products and their sum round
three times: 12 units of 2^-24 relative to factor (|x0| + |x1|), then one rounding to the output type."""
import math

import pytest
import torch

from oracle import seq_oracle as Q
from seq_helpers import DTYPES, randn, within

from flash_bla.ops.rotary.fused import rotary_embedding, rotary_frequencies
from flash_bla.ops.rotary.naive import naive_rotary

ROUNDINGS = 12


def freqs_of(pairs, base=1e4):
    return base ** (-torch.arange(pairs, dtype=torch.float64) / pairs)


# ---- CPU ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes", [1, 2])
def test_oracle_matches_the_naive_statement_and_its_gradient(interleaved, axes):
    rn = randn(0)
    x = rn(2, 3, 7, 14, dtype=torch.float64).requires_grad_()
    f = freqs_of(6)
    pos = torch.arange(7 * axes).view(7, axes) * 5 - 9 if axes > 1 else torch.arange(7) * 1000
    y = naive_rotary(x, f, pos, 1.3, interleaved, axes)
    assert torch.allclose(y, Q.rotary(x, f, pos, 1.3, interleaved, axes), atol=1e-12)
    dy = rn(2, 3, 7, 14, dtype=torch.float64)
    dx, = torch.autograd.grad(y, x, dy)
    assert torch.allclose(dx, Q.rotary(dy, f, pos, 1.3, interleaved, axes, inverse=True), atol=1e-12)
    # differences
    e = torch.zeros_like(x)
    e[1, 2, 3, 4] = 1e-6
    num = ((naive_rotary(x + e, f, pos, 1.3, interleaved, axes) - naive_rotary(x - e, f, pos, 1.3, interleaved, axes)) * dy).sum() / 2e-6
    assert abs(num.item() - dx[1, 2, 3, 4].item()) < 1e-7


def test_frequencies():
    f, m = rotary_frequencies(16, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0 and torch.allclose(f, freqs_of(8), rtol=1e-14)
    g, m = rotary_frequencies(16, scaling="linear", scale=4, device="cpu")
    assert torch.allclose(g, f / 4) and m == 1.0
    g, m = rotary_frequencies(16, scaling="ntk", scale=4, device="cpu")
    assert g[0] == f[0] and math.isclose(g[-1].item(), f[-1].item() / 4, rel_tol=1e-12) and m == 1.0
    g, m = rotary_frequencies(128, scaling="yarn", scale=8, original_length=4096, device="cpu")
    f = freqs_of(64)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.equal(g[turns <= 1], f[turns <= 1] / 8)
    assert ((g <= f) & (g >= f / 8 * (1 - 1e-12))).all() and m == 0.1 * math.log(8) + 1
    g, _ = rotary_frequencies(16, axes=2, device="cpu")
    assert torch.allclose(g, freqs_of(4).repeat(2))
    assert torch.equal(rotary_frequencies(2, scaling="ntk", scale=2, device="cpu")[0], torch.ones(1, dtype=torch.float64))


@pytest.mark.parametrize("kw", [dict(dim=3), dict(dim=0), dict(dim=8, axes=3), dict(dim=8, scaling="other"),
                                dict(dim=8, scaling="linear", scale=0.5), dict(dim=8, scaling="yarn", scale=2),
                                dict(dim=8, scaling="yarn", scale=2, original_length=64, ramp=(3.0, 3.0))])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        rotary_frequencies(**kw, device="cpu")


def test_refusals_on_cpu():
    q, f = torch.zeros(2, 3, 5, 8), freqs_of(4)
    pos = torch.arange(5)

    def refused(exc, match, q=q, k=None, f=f, p=None, **kw):
        with pytest.raises(exc, match=match):
            rotary_embedding(q, k, f, p, **kw)

    refused(RuntimeError, "CUDA")
    refused(ValueError, "layout", layout="hbld")
    refused(ValueError, "dimensions", q=q[0])
    refused(TypeError, "dtype", q=q.double())
    refused(ValueError, "agree", k=q[:1])
    refused(ValueError, "agree", k=q[..., :6])
    refused(ValueError, "same dtype", k=q.half())
    refused(ValueError, "no heads", k=q[:, :0])
    refused(TypeError, "float64", f=f.float())
    refused(ValueError, "pairs", f=freqs_of(5))
    refused(ValueError, "pairs", f=freqs_of(0))
    refused(ValueError, "axes", axes=3, p=pos)
    refused(ValueError, "axes", axes=2)
    refused(TypeError, "int64", p=pos.float())
    refused(ValueError, "positions", p=pos[:4])
    refused(ValueError, "positions", p=pos.expand(3, 5))
    refused(ValueError, "positions", p=pos, axes=2)
    refused(ValueError, "offset", p=pos, offset=3)
    refused(ValueError, "dimensions", cu_seqlens=torch.tensor([0, 5], dtype=torch.int32))
    refused(ValueError, "int32", q=q[0], cu_seqlens=torch.tensor([0, 5]))


def test_frequencies_that_want_a_gradient_are_refused():
    """They get none: refused, where they would otherwise stay as they are without a word."""
    q, f = torch.zeros(2, 3, 5, 8), freqs_of(4).requires_grad_()
    with pytest.raises(RuntimeError, match="freqs"):
        rotary_embedding(q, None, f)
    fw = torch.autograd.forward_ad
    with fw.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="freqs"):
        rotary_embedding(q, None, fw.make_dual(f.detach(), torch.ones(4, dtype=torch.float64)))
    for frequencies in (f.detach(), f):
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            rotary_embedding(q, None, frequencies)


def test_library_refuses_without_a_device():
    import ctypes
    from flash_bla import _C
    f = _C.lib().fbla_rotary
    p = _C.RotaryProblem(0, 1, 1, 0, 8, 4, 1)
    p.seq_len = 3
    assert f(ctypes.byref(p), None, None, None, None, None) == 1 and b"freqs" in _C.lib().fbla_last_error()
    p.freqs = 16
    assert f(ctypes.byref(p), None, None, None, None, None) == 1 and b"NULL" in _C.lib().fbla_last_error()
    p.pairs = 5
    assert f(ctypes.byref(p), None, None, None, None, None) == 1 and b"pairs" in _C.lib().fbla_last_error()
    p.pairs, p.dtype = 4, 7
    assert f(ctypes.byref(p), None, None, None, None, None) == 1 and b"dtype" in _C.lib().fbla_last_error()


# ---- GPU ------------------------------------------------------------------------------------------
gpu = pytest.mark.gpu

#        B  L   H  Hk  D    R   layout  interleaved
SHAPES = [(1, 1, 1, 1, 64, 64, "bhld", False),
          (2, 1, 16, 4, 64, 64, "blhd", True),
          (3, 37, 5, 5, 80, 48, "bhld", True),
          (3, 37, 5, 2, 80, 48, "blhd", False),
          (1, 130, 2, 1, 128, 128, "bhld", False),
          (2, 9, 3, 3, 10, 6, "bhld", False),       # pairs of 3: element by element
          (2, 9, 3, 1, 9, 8, "blhd", True),         # an odd number of features
          (1, 5, 2, 2, 7, 2, "bhld", False),
          (1, 33, 1, 1, 512, 512, "blhd", True)]    # all heads' features turned as one


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("positions", ["none", "shared", "rows32"])
def test_forward_and_backward(shape, dtype, positions):
    B, L, H, Hk, D, R, layout, inter = shape
    rn = randn(B * 1000 + L)
    dims = lambda h: (B, h, L, D) if layout == "bhld" else (B, L, h, D)     # noqa: E731
    q, k, dq, dk = rn(*dims(H), dtype=dtype), rn(*dims(Hk), dtype=dtype), rn(*dims(H), dtype=dtype), rn(*dims(Hk), dtype=dtype)
    f = freqs_of(R // 2)
    pos, kw = torch.arange(L) + 11, dict(offset=11)
    if positions == "shared":
        pos, kw = torch.arange(L) * 977 - 5, {}
    elif positions == "rows32":
        pos, kw = (torch.arange(B)[:, None] * 1000003 + torch.arange(L)).int(), {}
    given = None if positions == "none" else pos.cuda()
    qd, kd = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    qo, ko = rotary_embedding(qd, kd, f.cuda(), given, factor=1.25, interleaved=inter, layout=layout, **kw)
    torch.autograd.backward((qo, ko), (dq.cuda(), dk.cuda()))
    wide = pos if pos.dim() == 1 else pos[:, None]
    if layout == "blhd":
        ref = lambda x, **a: Q.rotary(x.transpose(1, 2), f, wide, 1.25, inter, **a).transpose(1, 2)     # noqa: E731
    else:
        ref = lambda x, **a: Q.rotary(x, f, wide, 1.25, inter, **a)         # noqa: E731
    for got, x, inv, what in ((qo, q, False, "q"), (ko, k, False, "k"), (qd.grad, dq, True, "dq"), (kd.grad, dk, True, "dk")):
        within(got, ref(x, inverse=inv), ref(x, absolute=True), ROUNDINGS, what)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_positions_keep_their_angle(dtype):
    """A position of 2^40 leaves nothing of an angle formed in fp32."""
    q = randn(3)(1, 2, 6, 32, dtype=dtype)
    pos = torch.tensor([0, 1, 10 ** 6, 2 ** 31 + 7, 2 ** 40 + 1, -5])
    f = freqs_of(16)
    # 2^40 f itself carries 2^-53 relative error in 64 bits, 2^-13 radians: integer frequencies have none
    f[1] = 1.0
    f[2] = 0.5
    got = rotary_embedding(q.cuda(), None, f.cuda(), pos.cuda())
    ref, major = Q.rotary(q, f, pos, 1.0, False), Q.rotary(q, f, pos, 1.0, False, absolute=True)
    near = pos.abs() < 2 ** 21              # there 64 bits hold the angle to 2^-31 on both sides
    within(got[:, :, near], ref[:, :, near], major[:, :, near], ROUNDINGS, "near")
    # beyond, both sides form pos * f and divide by 2 pi in 64 bits: three roundings of 2^-53 of the angle
    err = (got.cpu().double() - ref).abs()
    lim = major * (3 * 2.0 ** -53 * pos.abs().double()[:, None] + 16 * Q.U + torch.finfo(dtype).eps / 2)
    assert (err <= lim).all()


@gpu
def test_axes():
    """A grid: the first half of the pairs turns with the row, the second with the column."""
    q = randn(4)(2, 3, 12, 16)
    f, _ = rotary_frequencies(16, axes=2)
    pos = torch.stack((torch.arange(12) // 4, torch.arange(12) % 4), -1)
    for p in (pos, pos.expand(2, 12, 2).contiguous()):
        got = rotary_embedding(q.cuda(), None, f, p.cuda(), axes=2, interleaved=True)
        ref = Q.rotary(q, f.cpu(), pos, 1.0, True, 2)
        within(got, ref, Q.rotary(q, f.cpu(), pos, 1.0, True, 2, absolute=True), ROUNDINGS, "axes")


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_packed_sequences_start_over(interleaved):
    rn = randn(5)
    cu = torch.tensor([0, 1, 1, 8, 20], dtype=torch.int32)
    q, dq = rn(23, 4, 24), rn(23, 4, 24)                # three tokens behind the last sequence
    f = freqs_of(10)
    qd = q.cuda().requires_grad_()
    got = rotary_embedding(qd, None, f.cuda(), offset=3, interleaved=interleaved, cu_seqlens=cu.cuda())
    got.backward(dq.cuda())
    pos = torch.cat([torch.arange(n) + 3 for n in (1, 7, 12)])
    for g, x, inv in ((got, q, False), (qd.grad, dq, True)):
        ref = Q.rotary(x[:20].transpose(0, 1), f, pos, 1.0, interleaved, inverse=inv).transpose(0, 1)
        major = Q.rotary(x[:20].transpose(0, 1), f, pos, 1.0, interleaved, absolute=True).transpose(0, 1)
        within(g[:20], ref, major, ROUNDINGS, "packed")
        assert not g[20:].any()


@gpu
@pytest.mark.parametrize("off", [0, 1, 4])
def test_strided_and_unaligned_inputs(off):
    """q and k as slices of one projection's output, at any offset; a gradient that is expanded."""
    rn = randn(6)
    buf = rn(2, 9, 3 * 4 * 16 + 8, dtype=torch.bfloat16).cuda()
    q, k = (buf[..., off + i * 64:off + (i + 1) * 64].unflatten(-1, (4, 16)) for i in range(2))
    f = freqs_of(8)
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    qo, ko = rotary_embedding(q, k, f.cuda(), layout="blhd")
    (qo.float().sum() + ko.float().sum() * 2).backward()
    pos = torch.arange(9)
    for got, x in ((qo, q), (ko, k), (q.grad, torch.ones_like(q)), (k.grad, 2 * torch.ones_like(k))):
        inv = got is q.grad or got is k.grad
        x = x.detach().cpu().transpose(1, 2)
        within(got.transpose(1, 2), Q.rotary(x, f, pos, 1.0, False, inverse=inv), Q.rotary(x, f, pos, 1.0, False, absolute=True),
               ROUNDINGS, "strided")


@gpu
def test_nan_stays_in_its_pair_and_empty_inputs():
    q = randn(7)(1, 2, 4, 8)
    q[0, 1, 2, 3] = float("nan")
    got = rotary_embedding(q.cuda(), None, freqs_of(4).cuda()).cpu()
    assert got[0, 1, 2, [3, 7]].isnan().all() and int(got.isnan().sum()) == 2
    for shape in ((0, 2, 4, 8), (2, 2, 0, 8)):
        assert rotary_embedding(torch.zeros(shape, device="cuda"), None, freqs_of(4).cuda()).shape == shape


@gpu
def test_one_gradient_alone_and_graph_capture():
    rn = randn(8)
    q, k, d = rn(2, 3, 10, 32), rn(2, 1, 10, 32), rn(2, 1, 10, 32)
    f, pos = freqs_of(16), torch.arange(10)
    kd = k.cuda().requires_grad_()
    _, ko = rotary_embedding(q.cuda(), kd, f.cuda())
    ko.backward(d.cuda())
    within(kd.grad, Q.rotary(d, f, pos, 1.0, False, inverse=True), Q.rotary(d, f, pos, 1.0, False, absolute=True), ROUNDINGS, "dk alone")
    x, fd = q.cuda(), f.cuda()
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rotary_embedding(x, None, fd)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(g):
        out = rotary_embedding(x, None, fd)
    x.copy_(rn(2, 3, 10, 32))
    g.replay()
    assert torch.equal(out, rotary_embedding(x, None, fd))


@gpu
def test_offsets_beyond_32_bits():
    L, H, D = 1_050_000, 32, 128
    q = torch.empty(1, L, H, D, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(0))
    f = freqs_of(64).cuda()
    got = rotary_embedding(q, None, f, layout="blhd")
    tail = rotary_embedding(q[:, -40:].clone(), None, f, offset=L - 40, layout="blhd")
    assert torch.equal(got[:, -40:], tail)
