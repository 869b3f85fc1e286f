"""Plain torch statement of the rotary positions (any device and float type); the CUDA operator never
calls it."""
import torch


def naive_rotary(x, freqs, positions, factor=1.0, interleaved=False, axes=1):
    """``x`` (..., L, D) with ``positions`` (L,) -- (L, axes) on several axes -- or anything that
    broadcasts against the leading dimensions; angles in 64 bits."""
    pairs = freqs.numel()
    pos = positions.double()
    if axes > 1:
        pos = pos.repeat_interleave(pairs // axes, dim=-1)      # (..., L, pairs)
    else:
        pos = pos[..., None]
    angle = pos * freqs.double()
    cos, sin = torch.cos(angle).to(x.dtype) * factor, torch.sin(angle).to(x.dtype) * factor
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((turned, rest), dim=-1)
