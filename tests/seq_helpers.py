"""Shared by the tests of the rotary positions, the convolution and the scan."""
import torch

from oracle import seq_oracle as Q

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def within(got, ref, major, roundings, what):
    """Elementwise, in the type that ``got`` has."""
    assert got is not None, f"{what}: missing"
    g = got.detach().cpu()
    assert g.shape == ref.shape, f"{what}: shape {tuple(g.shape)}, expected {tuple(ref.shape)}"
    tol = Q.bounds(ref, major, g.dtype, roundings)
    err = (g.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(err / tol).nan_to_num(9e9).max():.2f} x the "
                           f"bound, at {tuple(bad.nonzero()[0].tolist())}: {g[tuple(bad.nonzero()[0])].item()} for "
                           f"{ref[tuple(bad.nonzero()[0])].item()}")


def randn(seed):
    g = torch.Generator().manual_seed(seed)
    return lambda *s, dtype=torch.float32, scale=1.0, shift=0.0: (torch.randn(*s, generator=g) * scale + shift).to(dtype)


def leaf(t):
    return None if t is None else t.cuda().requires_grad_()


def cuda(t):
    return None if t is None else t.cuda()
