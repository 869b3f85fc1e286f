"""Rotary positions: what ``decoupled_la`` takes as ``q_rope`` and ``k_rope``.

    (x0, x1) -> factor * (x0 cos a - x1 sin a, x0 sin a + x1 cos a),   a = position * freqs[pair]

q and k are rotated by one kernel; the gradient is the same kernel with the opposite angle.  The
reference's layers rotate in torch (``flash_bla/layers/mlla.py``, ``rala.py``).
"""
import math
from typing import Optional, Tuple

import torch

from flash_bla import _C
from flash_bla.ops import _seq as S


def rotary_frequencies(
    dim: int,
    base: float = 10000.0,
    *,
    axes: int = 1,
    scaling: Optional[str] = None,
    scale: float = 1.0,
    original_length: Optional[int] = None,
    ramp: Tuple[float, float] = (1.0, 32.0),
    device="cuda",
) -> Tuple[torch.Tensor, float]:
    r"""Radians per position of every pair, and the factor that goes with them.

    Args:
        dim: number of rotated features (two per pair).
        base: pair `i` of `P` (per axis) turns by `base ** (-i / P)` per position.
        axes: number of position coordinates the pairs are shared out to (2 for an image grid).
        scaling: how positions beyond the trained length are brought in, by `scale` (>= 1):
            `None`; `"linear"`: all frequencies divided; `"ntk"`: the base raised to
            `base * scale ** (P / (P - 1))`, so that the slowest pair is divided and the fastest is not;
            `"yarn"`: a pair that turns less than `ramp[0]` times over `original_length` is divided, one
            that turns more than `ramp[1]` times is kept, a linear ramp in between, and the rotated
            features are multiplied by `0.1 ln(scale) + 1`.
    Returns `(freqs, factor)`: float64 `(dim / 2,)` on `device`, and a float, as `rotary_embedding` takes them.
    """
    if dim < 2 or dim % 2:
        raise ValueError(f"dim must be even and positive, got {dim}")
    pairs = dim // 2
    if axes < 1 or pairs % axes:
        raise ValueError(f"axes={axes} must divide the {pairs} pairs")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    if not scale >= 1.0:
        raise ValueError(f"scale must be at least 1, got {scale}")
    per = pairs // axes
    if scaling == "ntk" and per > 1:
        base = base * scale ** (per / (per - 1))
    freqs = float(base) ** (-torch.arange(per, dtype=torch.float64) / per)
    factor = 1.0
    if scaling == "linear":
        freqs = freqs / scale
    elif scaling == "yarn":
        if original_length is None or original_length < 1:
            raise ValueError("scaling='yarn' needs original_length")
        if not ramp[1] > ramp[0]:
            raise ValueError(f"ramp must be increasing, got {ramp}")
        keep = ((original_length * freqs / (2 * math.pi) - ramp[0]) / (ramp[1] - ramp[0])).clamp(0, 1)
        freqs = freqs * keep + freqs / scale * (1 - keep)
        factor = 0.1 * math.log(scale) + 1.0
    return freqs.repeat(axes).to(device), factor


# positions of (batch, head, token) among the tensor's dimensions; None: packed (total, heads, features)
_DIMS = {"bhld": (0, 1, 2), "blhd": (0, 2, 1)}


def _order(v, dims):
    """(batch, head, token) entries of a shape or of strides; a packed tensor has no batch."""
    if dims is None:
        return None, v[1], v[0]
    return v[dims[0]], v[dims[1]], v[dims[2]]


_ZERO3 = (0, 0, 0)


def _strides(v, dims):
    b, h, t = _order(v, dims)
    return b or 0, h, t


def _rotate(q, k, freqs, positions, offset, factor, interleaved, axes, dims, cu, inverse):
    """One launch; q or k may be None.  Outputs are contiguous in the layout of the inputs."""
    if q is None:
        return None, _rotate(k, None, freqs, positions, offset, factor, interleaved, axes, dims, cu, inverse)[0]
    q = S.rows(q)
    qo = S.new(q)
    B, H, L = _order(q.shape, dims)
    Hk, ko, ks, kos = 0, None, _ZERO3, _ZERO3
    if k is not None:
        k = S.rows(k)
        ko = S.new(k)
        Hk, ks, kos = _order(k.shape, dims)[1], _strides(k.stride(), dims), _strides(ko.stride(), dims)
    pos32, pstride, pptr = 0, (0, 0), None
    if positions is not None:
        pos32, pptr, ps = positions.dtype == torch.int32, positions.data_ptr(), positions.stride()
        if positions.dim() - (axes > 1) == 2:
            pstride = (ps[0] if positions.shape[0] > 1 else 0, ps[1])
        else:
            pstride = (0, ps[0])
    prob = _C.RotaryProblem(_C.dtype_code(q.dtype), 1 if B is None else B, H, Hk, q.shape[-1], freqs.numel(), axes, interleaved,
                            inverse, pos32, 0 if cu is None else cu.numel() - 1, factor, L, offset, *_strides(q.stride(), dims), *ks,
                            *_strides(qo.stride(), dims), *kos, *pstride, pptr, _C.ptr(cu), freqs.data_ptr())
    S.call(_C.lib().fbla_rotary, prob, q, q.data_ptr(), _C.ptr(k), qo.data_ptr(), _C.ptr(ko))
    return qo, ko


class RotaryFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, freqs, positions, offset, factor, interleaved, axes, dims, cu):
        ctx.save_for_backward(freqs, positions, cu)
        ctx.args = (offset, factor, interleaved, axes, dims)
        ctx.set_materialize_grads(False)
        return _rotate(q, k, freqs, positions, offset, factor, interleaved, axes, dims, cu, False)

    @staticmethod
    def backward(ctx, dq, dk):
        S.refuse_second_order("rotary_embedding", dq, dk)
        freqs, positions, cu = ctx.saved_tensors
        offset, factor, interleaved, axes, dims = ctx.args
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        if dq is not None or dk is not None:
            dq, dk = _rotate(dq, dk, freqs, positions, offset, factor, interleaved, axes, dims, cu, True)
        return (dq, dk) + (None,) * 8


def rotary_embedding(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    freqs: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    *,
    offset: int = 0,
    factor: float = 1.0,
    interleaved: bool = False,
    axes: int = 1,
    layout: str = "bhld",
    cu_seqlens: Optional[torch.Tensor] = None,
):
    r"""
    Args:
        q: queries `(B, H, L, D)`, with `layout="blhd"` `(B, L, H, D)`, with `cu_seqlens` packed
            `(total_tokens, H, D)`.  Read with any strides as long as the features are contiguous.
        k: keys of the same layout, dtype, batch, length and features (the number of heads may differ), or `None`.
        freqs: float64 `(P,)`, radians per position of each pair; the first `2 P <= D` features are
            rotated, the others copied.  They get no gradient and must not require one.  See `rotary_frequencies`.
        positions: int32 or int64 `(L,)` or `(B, L)`, packed `(total_tokens,)`; with `axes > 1` a last
            dimension of `axes` coordinates, and pair `i` turns with coordinate `i // (P / axes)`.
            `None`: `offset`, `offset + 1`, ... in every sequence.
        factor: multiplies the rotated features (the second result of `rotary_frequencies`).
        interleaved: pair `i` is features `(2 i, 2 i + 1)`; otherwise `(i, i + P)`.
        cu_seqlens: int32 cumulative lengths of packed sequences; tokens behind the last one come out
            as zeros.
    Returns `(q_rope, k_rope)`, contiguous; `q_rope` alone when `k` is `None`.
    """
    if cu_seqlens is not None:
        cu_seqlens, dims, rank = S.check_cu_seqlens(cu_seqlens), None, 3
    elif layout in _DIMS:
        dims, rank = _DIMS[layout], 4
    else:
        raise ValueError(f"layout must be 'bhld' or 'blhd', got {layout!r}")
    if q.dim() != rank:
        raise ValueError(f"expected q with {rank} dimensions in this layout, got shape {tuple(q.shape)}")
    if q.dtype not in S.FLOATS:
        raise TypeError(f"dtype {q.dtype} is not supported (float16, bfloat16, float32)")
    B, H, L = _order(q.shape, dims)
    if k is not None:
        if k.dim() != rank or k.shape[-1] != q.shape[-1] or _order(k.shape, dims)[0::2] != (B, L):
            raise ValueError(f"q and k must agree in all but the heads, got {tuple(q.shape)} and {tuple(k.shape)}")
        if k.dtype != q.dtype:
            raise ValueError("q and k must have the same dtype")
        if _order(k.shape, dims)[1] == 0:
            raise ValueError("k has no heads: pass None")
    if H == 0:
        raise ValueError("q has no heads")
    if freqs.dtype != torch.float64 or freqs.dim() != 1:
        raise TypeError("freqs must be a float64 tensor of shape (pairs,)")
    if S.wants_grad(freqs):
        raise RuntimeError("freqs get no gradient: detach them, or call under torch.no_grad()")
    pairs = freqs.numel()
    if not 1 <= pairs <= q.shape[-1] // 2:
        raise ValueError(f"{pairs} pairs do not fit {q.shape[-1]} features")
    if axes < 1 or pairs % axes:
        raise ValueError(f"axes={axes} must divide the {pairs} pairs")
    if positions is None:
        if axes > 1:
            raise ValueError("positions on several axes have to be given")
    else:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must be int32 or int64")
        if offset != 0:
            raise ValueError("offset goes with positions=None")
        tail = (axes,) if axes > 1 else ()
        if positions.shape not in ((L,) + tail, (B, L) + tail, (1, L) + tail):
            raise ValueError(f"positions of shape {tuple(positions.shape)} do not fit {B or 1} rows of {L} tokens on {axes} axes")
        if axes > 1:
            positions = S.rows(positions)
    S.same_device(q, k, freqs, positions, cu_seqlens)
    S.require_cuda(q)
    args = (S.dense(freqs), positions, int(offset), float(factor), bool(interleaved), int(axes), dims, cu_seqlens)
    if S.wants_grad(q, k):
        qo, ko = RotaryFunction.apply(q, k, *args)
    else:
        qo, ko = _rotate(q, k, *args, False)
    return qo if k is None else (qo, ko)
