"""The rotary positions, the convolution and the scan as they are used together and beside the
framework's other operators."""
import pytest
import torch
import torch.nn.functional as F

from oracle import bla_oracle as O
from oracle import seq_oracle as Q
from helpers import check
from seq_helpers import randn

from flash_bla.ops.linear_attn.decoupled import decoupled_la, rotary_decoupled_la
from flash_bla.ops.rotary.fused import rotary_embedding, rotary_frequencies
from flash_bla.ops.selective_scan.conv import causal_conv1d, causal_conv1d_step
from flash_bla.ops.selective_scan.naive import naive_causal_conv1d, naive_selective_scan
from flash_bla.ops.selective_scan.scan import selective_scan, selective_scan_step

pytestmark = pytest.mark.gpu


def block_weights(seed, width, C, N, R, dtype):
    rn = randn(seed)
    return dict(w_in=rn(2 * C, width, dtype=dtype, scale=width ** -0.5), conv_w=rn(C, 4, dtype=dtype, scale=0.5),
                conv_b=rn(C, dtype=dtype, scale=0.1), w_x=rn(R + 2 * N, C, dtype=dtype, scale=C ** -0.5),
                w_dt=rn(C, R, dtype=dtype, scale=R ** -0.5), dt_bias=rn(C, shift=-3.0), A=-torch.exp(rn(C, N, scale=0.5)), D=rn(C),
                w_out=rn(width, C, dtype=dtype, scale=C ** -0.5))


def block(w, u, conv, scan, N):
    """The block around the scan: projection, convolution, the scan's inputs from its output, gate, projection."""
    C, R = w["w_dt"].shape
    xz = u @ w["w_in"].t()
    x = conv(xz[..., :C])
    p = x @ w["w_x"].t()
    dt = p[..., :R] @ w["w_dt"].t()
    y = scan(x, dt, p[..., R:R + N], p[..., R + N:], xz[..., C:])
    return y @ w["w_out"].t()


def test_block_trains_and_decodes():
    width, C, N, R, B, T = 32, 64, 16, 8, 2, 100
    w = block_weights(0, width, C, N, R, torch.float32)
    u = randn(1)(B, T, width)
    dy = randn(2)(B, T, width)

    def whole(w, u):
        return block(w, u, lambda x: causal_conv1d(x, w["conv_w"], w["conv_b"], activation="silu"),
                     lambda x, dt, Bm, Cm, z: selective_scan(x, dt, w["A"], Bm, Cm, w["D"], z, w["dt_bias"], dt_softplus=True), N)

    def plain(w, u):
        return block(w, u, lambda x: naive_causal_conv1d(x, w["conv_w"], w["conv_b"], "silu")[0],
                     lambda x, dt, Bm, Cm, z: naive_selective_scan(x, dt, w["A"], Bm[:, :, None], Cm[:, :, None], w["D"], z, w["dt_bias"],
                                                                   True)[0], N)

    allow = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        wg, ug = {k: v.cuda().requires_grad_() for k, v in w.items()}, u.cuda().requires_grad_()
        out = whole(wg, ug)
        out.backward(dy.cuda())
        wd, ud = {k: v.double().requires_grad_() for k, v in w.items()}, u.double().requires_grad_()
        ref = plain(wd, ud)
        ref.backward(dy.double())
        # fp32 throughout: 100 tokens' states at 8 roundings each, two projections of up to 72 terms on both ways
        # (4 * 72), the sum over 200 tokens of a weight's gradient: about 2000 roundings of 2^-24 = 1.2e-4
        for what, got, want in [("out", out, ref), ("du", ug.grad, ud.grad)] + [(k, wg[k].grad, wd[k].grad) for k in w]:
            err = (got.detach().cpu().double() - want.detach()).norm() / want.detach().norm()
            assert err < 1.2e-4, (what, err.item())
        # a prompt, its states kept, then token by token
        with torch.no_grad():
            w = {k: v.detach() for k, v in wg.items()}
            states = {}

            def conv_prompt(x):
                y, states["conv"] = causal_conv1d(x, w["conv_w"], w["conv_b"], activation="silu", return_final_state=True)
                return y

            def scan_prompt(x, dt, Bm, Cm, z):
                y, states["scan"] = selective_scan(x, dt, w["A"], Bm, Cm, w["D"], z, w["dt_bias"], dt_softplus=True,
                                                   return_final_state=True)
                return y

            got = [block(w, u[:, :90].cuda(), conv_prompt, scan_prompt, N)]
            for t in range(90, T):
                got.append(block(w, u[:, t].cuda(), lambda x: causal_conv1d_step(x, states["conv"], w["conv_w"], w["conv_b"], activation="silu"),
                                 lambda x, dt, Bm, Cm, z: selective_scan_step(x, dt, w["A"], Bm, Cm, states["scan"], w["D"], z, w["dt_bias"],
                                                                              dt_softplus=True), N)[:, None])
            got = torch.cat(got, 1).cpu().double()
            assert (got - ref.detach()).norm() / ref.detach().norm() < 1.2e-4
    finally:
        torch.backends.cuda.matmul.allow_tf32 = allow


def test_steps_replay_from_a_graph():
    """Decoding captured once and replayed: the states move on in place."""
    B, C, N = 4, 128, 16
    rn = randn(3)
    w = {k: v.cuda() for k, v in block_weights(4, 32, C, N, 8, torch.bfloat16).items()}
    xs = rn(6, B, C, dtype=torch.bfloat16).cuda()
    Bm, Cm = rn(6, B, N, dtype=torch.bfloat16).cuda(), rn(6, B, N, dtype=torch.bfloat16).cuda()

    def token(x, Bt, Ct, conv, scan):
        h = causal_conv1d_step(x, conv, w["conv_w"], w["conv_b"], activation="silu")
        return selective_scan_step(h, h, w["A"], Bt, Ct, scan, w["D"], x, w["dt_bias"], dt_softplus=True)

    fresh = lambda: (torch.zeros(B, 3, C, dtype=torch.bfloat16, device="cuda"), torch.zeros(B, C, N, device="cuda"))     # noqa: E731
    conv, scan = fresh()
    want = [token(xs[i], Bm[i], Cm[i], conv, scan).clone() for i in range(6)]
    conv2, scan2 = fresh()
    x, Bt, Ct = xs[0].clone(), Bm[0].clone(), Cm[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token(x, Bt, Ct, conv2, scan2)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = token(x, Bt, Ct, conv2, scan2)
    conv2.zero_()
    scan2.zero_()
    for i in range(6):
        x.copy_(xs[i])
        Bt.copy_(Bm[i])
        Ct.copy_(Cm[i])
        graph.replay()
        assert torch.equal(y, want[i]), i
    assert torch.equal(conv, conv2) and torch.equal(scan, scan2)


def test_training_step_replays_from_a_graph():
    """Forward and backward of convolution and scan in one captured graph, as often as it is replayed."""
    B, T, C, N = 2, 70, 64, 16
    rn = randn(5)
    leaves = [t.cuda().requires_grad_() for t in (rn(B, T, C, dtype=torch.bfloat16), rn(C, 4, dtype=torch.bfloat16),
                                                  -torch.exp(rn(C, N)), rn(B, T, N, dtype=torch.bfloat16))]
    dy = rn(B, T, C, dtype=torch.bfloat16).cuda()

    def step():
        x, w, A, Bm = leaves
        h = causal_conv1d(x, w, activation="silu")
        y = selective_scan(h, h, A, Bm, Bm, dt_softplus=True)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (6, 7):
        with torch.no_grad():
            leaves[0].copy_(randn(seed)(B, T, C, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64])
def test_rotary_decoupled_la(dtype, D):
    """The rotary inputs of decoupled_la made on the way, on a grid of positions, with gradients."""
    B, H, rows, cols = 2, 3, 9, 11
    L = rows * cols
    rn = randn(D)
    q, k = (F.elu(rn(B, H, L, D)).add(1).to(dtype) for _ in range(2))
    v, do = rn(B, H, L, D, dtype=dtype), rn(B, H, L, D, dtype=dtype)
    pos = torch.stack((torch.arange(L) // cols, torch.arange(L) % cols), -1)
    f, _ = rotary_frequencies(D, axes=2)
    xs = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = rotary_decoupled_la(*xs, f, pos.cuda(), axes=2)
    o.backward(do.cuda())
    # the same by hand: rotary_embedding, decoupled_la
    ys = [t.cuda().requires_grad_() for t in (q, k, v)]
    qr, kr = rotary_embedding(ys[0], ys[1], f, pos.cuda(), axes=2, interleaved=True)
    o2 = decoupled_la(ys[0], ys[1], qr, kr, ys[2])
    o2.backward(do.cuda())
    assert torch.equal(o, o2) and all(torch.equal(a.grad, b.grad) for a, b in zip(xs, ys))
    # against 64 bits, on the rotated inputs as the kernel rounds them
    rot = lambda t: Q.rotary(t, f.cpu(), pos, 1.0, True, 2).to(dtype)       # noqa: E731
    check(o, O.decoupled_la_fwd(q, k, rot(q), rot(k), v), dtype, "o")


def test_on_another_stream_and_at_once():
    """Two streams run the same operators at the same time: every call has a workspace of its own."""
    rn = randn(8)
    C, N, T = 96, 16, 2000                              # few channels: the scan's segments use the workspace
    sets = [[t.cuda() for t in (rn(1, T, C), rn(1, T, C).abs() * 0.1, -torch.exp(rn(C, N)), rn(1, T, N), rn(1, T, N))] for _ in range(2)]
    want = [selective_scan(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = selective_scan(*sets[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which", ["convolution", "scan"])
def test_a_step_on_a_state_that_a_backward_pass_needs_is_noticed(which):
    """The state of a call with gradients moved on by a token before its backward pass: an error, as of torch's own
    operations in place, and no wrong gradient."""
    B, T, C, N = 2, 12, 32, 16
    rn = randn(9)
    x, dt, A, Bm = rn(B, T, C).cuda(), rn(B, T, C).abs().cuda(), -torch.exp(rn(C, N)).cuda(), rn(B, T, N).cuda()
    w = rn(C, 4).cuda().requires_grad_()
    A.requires_grad_()
    if which == "convolution":
        state = rn(B, 3, C).cuda()
        whole = lambda: causal_conv1d(x, w, activation="silu", initial_state=state)             # noqa: E731
        step = lambda: causal_conv1d_step(x[:, 0], state, w)                                    # noqa: E731
    else:
        state = rn(B, C, N).cuda()
        whole = lambda: selective_scan(x, dt, A, Bm, Bm, initial_state=state)                   # noqa: E731
        step = lambda: selective_scan_step(x[:, 0], dt[:, 0], A, Bm[:, 0], Bm[:, 0], state)     # noqa: E731
    y = whole()
    before = state._version
    with torch.no_grad():
        step()
    versions = state._version - before
    assert versions == 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    y = whole()                         # in the other order nothing is in the way
    y.sum().backward()
    with torch.no_grad():
        step()
    with torch.inference_mode():        # a state made there has no version to move on
        held = state.clone()
        causal_conv1d_step(x[:, 0], held, w) if which == "convolution" else \
            selective_scan_step(x[:, 0], dt[:, 0], A, Bm[:, 0], Bm[:, 0], held)
    with torch.no_grad():
        step()
    assert torch.equal(held, state)


def test_forward_mode_derivatives_are_refused():
    """No operator has a forward-mode derivative: a dual input raises, under no_grad too, and so does a dual gradient."""
    fw = torch.autograd.forward_ad
    rn = randn(10)
    B, T, C, N = 2, 6, 16, 4
    x, w, dt, A, Bm = rn(B, T, C).cuda(), rn(C, 4).cuda(), rn(B, T, C).abs().cuda(), -torch.exp(rn(C, N)).cuda(), rn(B, T, N).cuda()
    q, f = rn(2, 3, 5, 8).cuda(), rotary_frequencies(8)[0]
    hist, state = rn(B, 3, C).cuda(), rn(B, C, N).cuda()
    calls = [(lambda v: rotary_embedding(v, None, f), q), (lambda v: rotary_embedding(q, v, f), q),
             (lambda v: rotary_decoupled_la(v, q, q, f), q), (lambda v: causal_conv1d(v, w), x), (lambda v: causal_conv1d(x, v), w),
             (lambda v: causal_conv1d(x, w, initial_state=v), hist), (lambda v: selective_scan(v, dt, A, Bm, Bm), x),
             (lambda v: selective_scan(x, dt, v, Bm, Bm), A), (lambda v: selective_scan(x, dt, A, Bm, v), Bm),
             (lambda v: selective_scan(x, dt, A, Bm, Bm, initial_state=v), state),
             (lambda v: causal_conv1d_step(v, hist, w), x[:, 0]), (lambda v: causal_conv1d_step(x[:, 0], v, w), hist),
             (lambda v: selective_scan_step(v, dt[:, 0], A, Bm[:, 0], Bm[:, 0], state), x[:, 0])]
    with fw.dual_level():
        for i, (call, v) in enumerate(calls):
            call(v)                     # an active level alone changes nothing
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="jvp|forward-mode"):
                    call(fw.make_dual(v, torch.ones_like(v)))
                    pytest.fail(f"call {i} went through")
    for call, v in (calls[0], calls[3], calls[6]):
        v = v.clone().requires_grad_()
        y = call(v)
        with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, v, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))
