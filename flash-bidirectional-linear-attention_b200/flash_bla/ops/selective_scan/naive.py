"""Plain torch statements of the short causal convolution and the selective scan (any device and float
type, differentiable by autograd); the CUDA operators never call them."""
import torch
import torch.nn.functional as F


def naive_causal_conv1d(x, weight, bias=None, activation=None, initial_state=None):
    """``x`` (B, T, C) -> (y, final_state)."""
    W, T = weight.shape[1], x.shape[1]
    if initial_state is None:
        initial_state = x.new_zeros(x.shape[0], W - 1, x.shape[2])
    full = torch.cat((initial_state, x), dim=1)
    y = sum(full[:, j:j + T] * weight[:, j] for j in range(W))
    if bias is not None:
        y = y + bias
    return (F.silu(y) if activation == "silu" else y), full[:, T:]


def naive_selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None):
    """``x``, ``dt``, ``z`` (B, T, C), ``B``, ``C`` (B, T, G, N) -> (y, final_state), token by token."""
    per = x.shape[2] // B.shape[2]
    B, C = (v.repeat_interleave(per, dim=2) for v in (B, C))            # (B, T, C, N)
    d = dt if dt_bias is None else dt + dt_bias
    if dt_softplus:
        d = F.softplus(d)
    h = x.new_zeros(x.shape[0], *A.shape) if initial_state is None else initial_state
    out = []
    for t in range(x.shape[1]):
        h = torch.exp(d[:, t, :, None] * A) * h + (d[:, t] * x[:, t])[..., None] * B[:, t]
        out.append((h * C[:, t]).sum(-1))
    y = torch.stack(out, dim=1) if out else torch.zeros_like(x)
    if D is not None:
        y = y + D * x
    return (y if z is None else y * F.silu(z)), h


def by_sequence(fn, cu_seqlens, tensors, states):
    """Runs ``fn(tensors of one sequence (1, len, ...), state (1, ...) or None) -> (y, state)`` over packed
    sequences; returns the packed results and the stacked states."""
    bounds = cu_seqlens.tolist()
    ys, ends = [], []
    for s, (lo, hi) in enumerate(zip(bounds[:-1], bounds[1:])):
        y, end = fn([None if t is None else t[None, lo:hi] for t in tensors], None if states is None else states[s:s + 1])
        ys.append(y[0])
        ends.append(end)
    return torch.cat(ys), torch.cat(ends)
