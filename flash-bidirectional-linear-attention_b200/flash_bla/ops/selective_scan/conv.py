"""Short causal convolution over tokens, one filter per channel: what a selective scan's inputs pass
through first.

    y[t, c] = act(bias[c] + sum_j weight[c, j] x[t - W + 1 + j, c])

For whole sequences (with gradients), packed sequences, and single tokens with a carried history.
"""
import ctypes
from typing import Optional

import torch

from flash_bla import _C
from flash_bla.ops import _seq as S


def _check_weight(x, weight, bias, activation):
    if x.dtype not in S.FLOATS:
        raise TypeError(f"dtype {x.dtype} is not supported (float16, bfloat16, float32)")
    if weight.dim() != 2 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"weight must have shape (channels, width), got {tuple(weight.shape)} for {x.shape[-1]} channels")
    if not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"width must be between 2 and 4, got {weight.shape[1]}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError("weight must have the dtype of x or float32")
    if bias is not None and (bias.shape != weight.shape[:1] or bias.dtype != weight.dtype):
        raise ValueError("bias must have shape (channels,) and the dtype of weight")
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")


def _lead(t):
    """(batch, token) strides; a packed tensor has no batch."""
    if t is None:
        return 0, 0
    s = t.stride()
    return (s[0], s[1]) if len(s) == 3 else (0, s[0])


def _problem(x, weight, silu, cu, dy=None):
    shape = x.shape
    return _C.ConvProblem(_C.dtype_code(x.dtype), _C.dtype_code(weight.dtype), shape[0] if len(shape) == 3 else 1, shape[-1],
                          weight.shape[1], silu, 0 if cu is None else cu.numel() - 1, 0, shape[-2], *_lead(x), *_lead(dy), _C.ptr(cu))


def _forward(x, weight, bias, state, silu, want_final, cu):
    y = S.new(x)
    prob = _problem(x, weight, silu, cu)
    rows = prob.batch if cu is None else prob.num_seqs
    final = torch.empty(rows, weight.shape[1] - 1, x.shape[-1], dtype=x.dtype, device=x.device) if want_final else None
    S.call(_C.lib().fbla_causal_conv_fwd, prob, x, x.data_ptr(), weight.data_ptr(), _C.ptr(bias), _C.ptr(state), y.data_ptr(),
           _C.ptr(final))
    return y, final


class CausalConv1dFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, state, silu, want_final, cu):
        y, final = _forward(x, weight, bias, state, silu, want_final, cu)
        ctx.save_for_backward(x, weight, bias, state, cu)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    def backward(ctx, dy, dfinal):
        S.refuse_second_order("causal_conv1d", dy, dfinal)
        x, weight, bias, state, cu = ctx.saved_tensors
        dy = torch.zeros_like(x) if dy is None else S.rows(dy)
        dfinal = S.dense(dfinal)
        prob = _problem(x, weight, ctx.silu, cu, dy)
        dx = S.new(x)
        dw = torch.empty_like(weight)
        db = None if bias is None else torch.empty_like(bias)
        dstate = torch.empty_like(state) if state is not None and ctx.needs_input_grad[3] else None
        L = _C.lib()
        ws, n = S.scratch(L.fbla_causal_conv_workspace_bytes(ctypes.byref(prob)), x)
        S.call(L.fbla_causal_conv_bwd, prob, x, x.data_ptr(), weight.data_ptr(), _C.ptr(bias), _C.ptr(state), dy.data_ptr(),
               _C.ptr(dfinal), dx.data_ptr(), dw.data_ptr(), _C.ptr(db), _C.ptr(dstate), _C.ptr(ws), n)
        return dx, dw, db, dstate, None, None, None


def causal_conv1d(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    activation: Optional[str] = None,
    initial_state: Optional[torch.Tensor] = None,
    return_final_state: bool = False,
    cu_seqlens: Optional[torch.Tensor] = None,
):
    r"""
    Args:
        x: `(B, T, C)`, or packed `(total_tokens, C)` with `cu_seqlens`.  Read with any strides as long as
            the channels are contiguous (a slice of a projection's output needs no copy).
        weight: `(C, W)`, `W` from 2 to 4 taps, the last one for the current token; dtype of `x` or float32.
        bias: `(C,)` of the dtype of `weight`, or `None`.
        activation: `None` or `"silu"`.
        initial_state: `(B, W - 1, C)` -- one row per sequence when packed --, the inputs before the first
            token, oldest first, of the dtype of `x`; `None`: zeros.
        return_final_state: also return the last `W - 1` inputs in the same form.
        cu_seqlens: int32 cumulative lengths of packed sequences, starting at zero and not decreasing;
            tokens behind the last one come out as zeros.
    Returns `y` of the shape of `x`, or `(y, final_state)`.
    """
    if x.dim() != (3 if cu_seqlens is None else 2):
        raise ValueError("x must have shape (B, T, C), or (total_tokens, C) with cu_seqlens, "
                         f"got {tuple(x.shape)}")
    _check_weight(x, weight, bias, activation)
    if x.shape[-1] == 0:
        raise ValueError("x has no channels")
    rows = x.shape[0]
    if cu_seqlens is not None:
        cu_seqlens = S.check_cu_seqlens(cu_seqlens)
        rows = cu_seqlens.numel() - 1
    if rows > 65535:
        raise ValueError(f"at most 65535 sequences, got {rows}")
    if initial_state is not None:
        if tuple(initial_state.shape) != (rows, weight.shape[1] - 1, x.shape[-1]) or initial_state.dtype != x.dtype:
            raise ValueError(f"initial_state must have shape {(rows, weight.shape[1] - 1, x.shape[-1])} and the dtype of x")
        initial_state = S.dense(initial_state)
    S.same_device(x, weight, bias, initial_state, cu_seqlens)
    S.require_cuda(x)
    args = (S.rows(x), S.dense(weight), S.dense(bias), initial_state, activation == "silu", bool(return_final_state), cu_seqlens)
    y, final = CausalConv1dFunction.apply(*args) if S.wants_grad(x, weight, bias, initial_state) else _forward(*args)
    return (y, final) if return_final_state else y


def causal_conv1d_step(
    x: torch.Tensor,
    state: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    activation: Optional[str] = None,
) -> torch.Tensor:
    r"""One token of every row: `x` `(B, C)`, `state` `(B, W - 1, C)` as `causal_conv1d` returns it.
    `state` is read and moved on by this token in place (contiguous, the dtype of `x`); no gradient.
    Returns `y` `(B, C)`."""
    if x.dim() != 2:
        raise ValueError(f"x must have shape (B, C), got {tuple(x.shape)}")
    _check_weight(x, weight, bias, activation)
    if state.shape != (x.shape[0], weight.shape[1] - 1, x.shape[1]) or state.dtype != x.dtype:
        raise ValueError(f"state must have shape {(x.shape[0], weight.shape[1] - 1, x.shape[1])} and the dtype of x")
    if not state.is_contiguous():
        raise ValueError("state is updated in place and must be contiguous")
    if x.shape[0] > 65535:
        raise ValueError(f"at most 65535 rows, got {x.shape[0]}")
    S.same_device(x, state, weight, bias)
    S.refuse_grad("causal_conv1d_step", x, state, weight, bias)
    S.require_cuda(x)
    x, weight, bias = S.rows(x), S.dense(weight), S.dense(bias)
    y = S.new(x)
    if y.numel() == 0:
        return y
    prob = _C.ConvProblem(_C.dtype_code(x.dtype), _C.dtype_code(weight.dtype), x.shape[0], x.shape[1], weight.shape[1],
                          activation == "silu", 0, 0, 1, x.stride(0))
    S.call(_C.lib().fbla_causal_conv_step, prob, x, x.data_ptr(), weight.data_ptr(), _C.ptr(bias),
           state.data_ptr(), y.data_ptr())
    S.moved(state)
    return y
