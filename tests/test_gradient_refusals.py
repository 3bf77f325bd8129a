"""What the kernels cannot differentiate is refused, not dropped (host logic, no GPU)."""
import pytest
import torch
from torch.autograd import forward_ad


def test_forward_mode_tangents_are_refused():
    from onereel_b200.attention import _wants_grad
    x, w = torch.randn(3, 4), torch.randn(3, 4, requires_grad=True)
    assert not _wants_grad(x, None) and _wants_grad(x, w, None)
    with forward_ad.dual_level():
        assert not _wants_grad(x) and _wants_grad(x, w)
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for t in (dual, dual.view(4, 3)):
            with pytest.raises(NotImplementedError, match='forward-mode'):
                _wants_grad(w, t)
            with torch.no_grad(), pytest.raises(NotImplementedError, match='forward-mode'):
                _wants_grad(t)
    with pytest.raises(NotImplementedError, match='forward-mode'):
        torch.func.jvp(lambda t: t if _wants_grad(t) else t, (x,), (x,))
