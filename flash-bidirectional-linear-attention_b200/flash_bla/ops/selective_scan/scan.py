"""Selective state space scan: a state per channel that decays and is fed token by token, both by
amounts that depend on the token.  The causal relative of ``simple_la``: there every token adds
``k v^T`` to one state, here the state also decays between tokens.

    d = dt + dt_bias  (softplus'd when asked)
    h[c, n] <- exp(d A[c, n]) h[c, n] + d x[c] B[n],   y[c] = (sum_n C[n] h[c, n] + D[c] x[c]) * silu(z[c])

For whole sequences (with gradients), packed sequences, and single tokens with a carried state.
"""
import ctypes
from typing import Optional

import torch

from flash_bla import _C
from flash_bla.ops import _seq as S


def _check(x, dt, A, B, C, D, z, dt_bias, lead):
    """``lead``: the number of x's dimensions before the channels.  Returns the number of groups."""
    shape, dtype = x.shape, x.dtype
    ch = shape[-1]
    if dtype not in S.FLOATS:
        raise TypeError(f"dtype {dtype} is not supported (float16, bfloat16, float32)")
    if ch == 0:
        raise ValueError("x has no channels")
    if dt.shape != shape or dt.dtype != dtype:
        raise ValueError(f"dt must have the shape and the dtype of x, got {tuple(dt.shape)} {dt.dtype}")
    if z is not None and (z.shape != shape or z.dtype != dtype):
        raise ValueError(f"z must have the shape and the dtype of x, got {tuple(z.shape)} {z.dtype}")
    if A.dim() != 2 or A.shape[0] != ch or A.dtype != torch.float32:
        raise ValueError("A must be a float32 tensor of shape (channels, states)")
    N = A.shape[1]
    if not 1 <= N <= 32:
        raise ValueError(f"the number of states must be between 1 and 32, got {N}")
    bc = B.shape
    for name, t, s in (("B", B, bc), ("C", C, C.shape)):
        if t.dtype != dtype or len(s) not in (lead + 1, lead + 2) or s[:lead] != shape[:lead] or s[-1] != N:
            raise ValueError(f"{name} must have the dtype of x and shape (..., states) or (..., groups, states), got {tuple(s)}")
    if C.shape != bc:
        raise ValueError("B and C must have the same shape")
    groups = bc[lead] if len(bc) == lead + 2 else 1
    if groups < 1 or ch % groups:
        raise ValueError(f"{groups} groups do not divide {ch} channels")
    for name, t in (("D", D), ("dt_bias", dt_bias)):
        if t is not None and (t.shape != (ch,) or t.dtype != torch.float32):
            raise ValueError(f"{name} must be a float32 tensor of shape (channels,)")
    return groups


def _s2(t):
    """(batch, token) strides of x and the like; a packed tensor has no batch."""
    if t is None:
        return 0, 0
    s = t.stride()
    return (s[0], s[1]) if len(s) == 3 else (0, s[0])


def _s3(t, lead):
    """(batch, token, group) strides of B, C."""
    s = t.stride()
    group = s[lead] if len(s) == lead + 2 else 0
    return (s[0], s[1], group) if lead == 2 else (0, s[0], group)


def _problem(x, dt, A, B, C, z, softplus, cu, dy=None):
    shape = x.shape
    lead = len(shape) - 1
    groups = B.shape[lead] if B.dim() == lead + 2 else 1
    return _C.ScanProblem(_C.dtype_code(x.dtype), shape[0] if lead == 2 else 1, shape[-1], A.shape[1], groups, softplus,
                          0 if cu is None else cu.numel() - 1, 0, shape[lead - 1], *_s2(x), *_s2(dt), *_s2(z),
                          *_s2(dy), *_s3(B, lead), *_s3(C, lead), _C.ptr(cu))


def _forward(x, dt, A, B, C, D, z, dt_bias, state, softplus, want_final, cu, checkpoints=False):
    L = _C.lib()
    prob = _problem(x, dt, A, B, C, z, softplus, cu)
    y = S.new(x)
    rows = prob.batch if cu is None else prob.num_seqs
    final = torch.empty(rows, *A.shape, dtype=torch.float32, device=x.device) if want_final else None
    ckpt = None
    if checkpoints:
        ckpt = torch.empty(L.fbla_selective_scan_checkpoint_floats(ctypes.byref(prob)), dtype=torch.float32, device=x.device)
    ws, n = S.scratch(L.fbla_selective_scan_workspace_bytes(ctypes.byref(prob), 0), x)
    S.call(L.fbla_selective_scan_fwd, prob, x, x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), _C.ptr(D),
           _C.ptr(z), _C.ptr(dt_bias), _C.ptr(state), y.data_ptr(), _C.ptr(final), _C.ptr(ckpt), _C.ptr(ws), n)
    return y, final, ckpt


class SelectiveScanFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, state, softplus, want_final, cu):
        y, final, ckpt = _forward(x, dt, A, B, C, D, z, dt_bias, state, softplus, want_final, cu, checkpoints=True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, state, cu, ckpt)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    def backward(ctx, dy, dfinal):
        S.refuse_second_order("selective_scan", dy, dfinal)
        x, dt, A, B, C, D, z, dt_bias, state, cu, ckpt = ctx.saved_tensors
        dy = torch.zeros_like(x) if dy is None else S.rows(dy)
        dfinal = S.aligned(S.dense(dfinal))
        prob = _problem(x, dt, A, B, C, z, ctx.softplus, cu, dy)
        dx, ddt, dA, dB, dC, dD, dz, dbias = map(S.new, (x, dt, A, B, C, D, z, dt_bias))
        dstate = S.new(state) if ctx.needs_input_grad[8] else None
        L = _C.lib()
        ws, n = S.scratch(L.fbla_selective_scan_workspace_bytes(ctypes.byref(prob), 1), x)
        S.call(L.fbla_selective_scan_bwd, prob, x, x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(), _C.ptr(D),
               _C.ptr(z), _C.ptr(dt_bias), _C.ptr(state), ckpt.data_ptr(), dy.data_ptr(), _C.ptr(dfinal), dx.data_ptr(),
               ddt.data_ptr(), dA.data_ptr(), dB.data_ptr(), dC.data_ptr(), _C.ptr(dD), _C.ptr(dz), _C.ptr(dbias),
               _C.ptr(dstate), _C.ptr(ws), n)
        return dx, ddt, dA, dB, dC, dD, dz, dbias, dstate, None, None, None


def selective_scan(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: Optional[torch.Tensor] = None,
    z: Optional[torch.Tensor] = None,
    dt_bias: Optional[torch.Tensor] = None,
    *,
    dt_softplus: bool = False,
    initial_state: Optional[torch.Tensor] = None,
    return_final_state: bool = False,
    cu_seqlens: Optional[torch.Tensor] = None,
):
    r"""
    Args:
        x, dt: inputs and step sizes `(B, T, C)`, or packed `(total_tokens, C)` with `cu_seqlens`.
        A: decay rates `(C, N)` float32, `N` up to 32; negative for a state that forgets.
        B, C: input and output projections `(B, T, N)`, or `(B, T, G, N)` for `G` groups of channels
            (packed: without the first dimension).
        D: skip weight `(C,)` float32, or `None`.
        z: gate of the shape of `x`, or `None`: `y` is multiplied by `silu(z)`.
        dt_bias: `(C,)` float32, or `None`, added to `dt`.
        dt_softplus: pass `dt + dt_bias` through softplus.
        initial_state: `(B, C, N)` float32 -- one row per sequence when packed; `None`: zeros.
        return_final_state: also return the states behind the last tokens in the same form.
        cu_seqlens: int32 cumulative lengths of packed sequences, starting at zero and not decreasing;
            tokens behind the last one come out as zeros.
    x, dt, z, B, C share one dtype and are read with any strides as long as their last dimension is
    contiguous.  States and sums are float32.
    Returns `y` of the shape and dtype of `x`, or `(y, final_state)`.
    """
    if x.dim() != (3 if cu_seqlens is None else 2):
        raise ValueError("x must have shape (B, T, C), or (total_tokens, C) with cu_seqlens, "
                         f"got {tuple(x.shape)}")
    _check(x, dt, A, B, C, D, z, dt_bias, x.dim() - 1)
    rows = x.shape[0]
    if cu_seqlens is not None:
        cu_seqlens = S.check_cu_seqlens(cu_seqlens)
        rows = cu_seqlens.numel() - 1
    if rows > 65535:
        raise ValueError(f"at most 65535 sequences, got {rows}")
    if initial_state is not None:
        if tuple(initial_state.shape) != (rows,) + tuple(A.shape) or initial_state.dtype != torch.float32:
            raise ValueError(f"initial_state must be a float32 tensor of shape {(rows,) + tuple(A.shape)}")
        initial_state = S.aligned(S.dense(initial_state))
    S.same_device(x, dt, A, B, C, D, z, dt_bias, initial_state, cu_seqlens)
    S.require_cuda(x)
    args = (S.rows(x), S.rows(dt), S.dense(A), S.rows(B), S.rows(C), S.dense(D), S.rows(z), S.dense(dt_bias), initial_state,
            bool(dt_softplus), bool(return_final_state), cu_seqlens)
    if S.wants_grad(x, dt, A, B, C, D, z, dt_bias, initial_state):
        y, final = SelectiveScanFunction.apply(*args)
    else:
        y, final, _ = _forward(*args)
    return (y, final) if return_final_state else y


def selective_scan_step(
    x: torch.Tensor,
    dt: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    state: torch.Tensor,
    D: Optional[torch.Tensor] = None,
    z: Optional[torch.Tensor] = None,
    dt_bias: Optional[torch.Tensor] = None,
    *,
    dt_softplus: bool = False,
) -> torch.Tensor:
    r"""One token of every row: `x`, `dt`, `z` `(B, C)`, `B`, `C` `(B, N)` or `(B, G, N)`, `state`
    `(B, C, N)` float32 as `selective_scan` returns it.  `state` is moved on by this token in place
    (contiguous, 16-byte aligned); no gradient.  Returns `y` `(B, C)`."""
    if x.dim() != 2:
        raise ValueError(f"x must have shape (B, C), got {tuple(x.shape)}")
    groups = _check(x, dt, A, B, C, D, z, dt_bias, 1)
    if state.shape != (x.shape[0],) + A.shape or state.dtype != torch.float32:
        raise ValueError(f"state must be a float32 tensor of shape {(x.shape[0],) + tuple(A.shape)}")
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("state is updated in place and must be contiguous and 16-byte aligned")
    if x.shape[0] > 65535:
        raise ValueError(f"at most 65535 rows, got {x.shape[0]}")
    S.same_device(x, dt, A, B, C, state, D, z, dt_bias)
    S.refuse_grad("selective_scan_step", x, dt, A, B, C, state, D, z, dt_bias)
    S.require_cuda(x)
    y = S.new(x)
    if y.numel() == 0:
        return y
    x, dt, B, C, z, A = S.rows(x), S.rows(dt), S.rows(B), S.rows(C), S.rows(z), S.dense(A)
    D, dt_bias = S.dense(D), S.dense(dt_bias)
    bs, cs = B.stride(), C.stride()
    prob = _C.ScanProblem(_C.dtype_code(x.dtype), x.shape[0], x.shape[1], A.shape[1], groups, dt_softplus, 0, 0, 1,
                          x.stride(0), 0, dt.stride(0), 0, 0 if z is None else z.stride(0), 0, 0, 0,
                          bs[0], 0, bs[1] if len(bs) == 3 else 0, cs[0], 0, cs[1] if len(cs) == 3 else 0)
    S.call(_C.lib().fbla_selective_scan_step, prob, x, x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(),
           _C.ptr(D), _C.ptr(z), _C.ptr(dt_bias), state.data_ptr(), y.data_ptr())
    S.moved(state)
    return y
