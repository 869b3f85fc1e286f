"""Host-side helpers of the sequence operators beside the attention passes (rotary positions, the
short causal convolution, the selective scan)."""
import ctypes

import torch
from torch.autograd import forward_ad as _fw

from flash_bla import _C

FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def require_cuda(x):
    if not x.is_cuda:
        raise RuntimeError("flash_bla operators run on CUDA tensors only (there is no CPU path)")


def same_device(x, *others):
    d = x.device
    for t in others:
        if t is not None and t.device != d:
            raise ValueError(f"all tensors must be on one device, got {d} and {t.device}")


def check_cu_seqlens(cu):
    if not isinstance(cu, torch.Tensor) or cu.ndim != 1 or cu.numel() < 2 or cu.dtype != torch.int32:
        raise ValueError("cu_seqlens must be an int32 tensor of shape (num_sequences + 1,)")
    return cu.contiguous()


def rows(t):
    """The tensor with its last dimension contiguous; the others may have any stride."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def new(t):
    """A contiguous tensor of the shape, dtype and device of ``t``."""
    return None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)


def aligned(t):
    """States are read 16 bytes at a time: a view at an odd offset is copied."""
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone()


def is_dual(*tensors):
    """Whether one of them carries a forward-mode tangent, which a kernel would drop without a word."""
    if getattr(_fw, "_current_level", 0) < 0:           # no forward-mode level is active
        return False
    return any(isinstance(t, torch.Tensor) and _fw.unpack_dual(t).tangent is not None for t in tensors)


def wants_grad(*tensors):
    """Whether the call has to go through its autograd function.  A dual input does not ``require`` a gradient, but there
    it raises, with gradients switched off too."""
    if is_dual(*tensors):
        return True
    for t in tensors:
        if t is not None and t.requires_grad:
            return torch.is_grad_enabled()
    return False


def refuse_grad(what, *tensors):
    if wants_grad(*tensors):
        if is_dual(*tensors):
            raise RuntimeError(f"{what} has no forward-mode derivative")
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")


def refuse_second_order(what, *grads):
    """At the head of a backward pass: with ``create_graph=True`` its results would look like constants, and to a
    forward-mode level as well."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no second derivative: its backward pass cannot run with create_graph=True")
    if is_dual(*grads):
        raise RuntimeError(f"{what} has no second derivative: its backward pass has no forward-mode derivative")


def call(fn, prob, like, *args):
    """One library call on the current stream of ``like``'s device."""
    with _C.device_guard(like):
        _C.check(fn(ctypes.byref(prob), *args, _C.stream_of(like)))


# After a kernel has written a caller's state through its address: as torch's own operations in place do, tell autograd, so
# that a backward pass which still needs the old state raises instead of using the new one (0.2 us).
moved = torch.autograd.graph.increment_version


def scratch(nbytes, like):
    """(tensor or None, bytes) from torch's caching allocator: a workspace of this call alone."""
    if nbytes < 0:
        _C.check(1)
    return (torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None), nbytes
