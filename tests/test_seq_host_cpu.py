"""Host-side rules of the sequence operators that need no device."""
import pytest
import torch

from flash_bla.ops import _seq as S
from flash_bla.ops.selective_scan.conv import causal_conv1d_step
from flash_bla.ops.selective_scan.scan import selective_scan_step


def test_dual_tensors_want_a_derivative():
    fw = torch.autograd.forward_ad
    x = torch.ones(2, 3)
    assert not S.wants_grad(x, None) and S.wants_grad(x, x.clone().requires_grad_())
    with fw.dual_level():
        d = fw.make_dual(x, x)
        assert not S.wants_grad(x, None) and S.wants_grad(x, None, d)
        with torch.no_grad():
            assert S.wants_grad(d) and not S.wants_grad(x.clone().requires_grad_())
    assert not S.wants_grad(x)


@pytest.mark.parametrize("dual", ["x", "state", "weights"])
def test_steps_refuse_dual_tensors(dual):
    fw = torch.autograd.forward_ad
    t = dict(x=torch.ones(2, 6), state=torch.zeros(2, 3, 6), w=torch.ones(6, 4), h=torch.zeros(2, 6, 5), A=torch.ones(6, 5))
    Bm = torch.ones(2, 5)
    with fw.dual_level(), torch.no_grad():
        for k in {"x": ["x"], "state": ["state", "h"], "weights": ["w", "A"]}[dual]:
            t[k] = fw.make_dual(t[k], torch.ones_like(t[k]))
        for call in (lambda: causal_conv1d_step(t["x"], t["state"], t["w"]),
                     lambda: selective_scan_step(t["x"], torch.ones(2, 6), t["A"], Bm, Bm, t["h"])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
