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


def test_a_path_without_a_backward_pass_raises_in_it():
    """values and graph-free inference are untouched; backward and grad() through the path raise, also where the rest of the
    loss has a gradient of its own"""
    from onereel_b200.attention import no_gradients, without_gradient
    x, w = torch.randn(3, 4), torch.randn(4, requires_grad=True)
    q = x * w
    for values in (q.detach() * 2, (q.detach() * 2, None), (q.detach() * 2, x + 1)):
        with torch.no_grad():
            assert without_gradient('this path', values, q, None) is values
        assert without_gradient('this path', values, x, None) is values
        tied = without_gradient('this path', values, q, None)
        one = tied[0] if isinstance(tied, tuple) else tied
        assert torch.equal(one, q.detach() * 2) and one.requires_grad
        for t in tied if isinstance(tied, tuple) else (tied,):
            if t is not None:
                with pytest.raises(NotImplementedError, match='this path'):
                    (q.sum() + t.sum()).backward()
                with pytest.raises(NotImplementedError, match='this path'):
                    torch.autograd.grad(q.sum() + t.sum(), w)
        q = x * w
    kept = x * w                                         # already differentiable: handed on
    assert without_gradient('this path', kept, q) is kept

    class Path:
        @no_gradients('this path')
        def run(self, q, k=None):
            return q.detach() + 1, None
    out, none = Path().run(x, k=w)
    assert none is None and torch.equal(out, x + 1)
    with pytest.raises(NotImplementedError):
        out.sum().backward()


def test_overwritten_tensors_raise_in_the_backward_pass():
    """old values that a node saved are refused, new ones have no gradient; views, second targets and plain targets too;
    without a wish for gradients nothing is recorded"""
    from onereel_b200.attention import overwrites
    w = torch.randn(4, requires_grad=True)
    a, b = torch.exp(w), torch.zeros(4)                  # exp saves its result
    overwrites('this kernel', (a, b), torch.ones(4))
    assert a.requires_grad and b.requires_grad
    for t in (a, b):
        with pytest.raises(NotImplementedError, match='this kernel'):
            torch.autograd.grad(t.sum() + w.sum(), w, retain_graph=True)
    saved = torch.exp(w)
    kept = saved * 1
    overwrites('this kernel', (saved,))
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        kept.sum().backward()
    base = torch.exp(w)
    overwrites('this kernel', (base[1:3],))
    with pytest.raises(NotImplementedError, match='this kernel'):
        base.sum().backward()
    plain = torch.zeros(4)
    overwrites('this kernel', (plain,), torch.ones(4))
    with torch.no_grad():
        overwrites('this kernel', (plain, torch.exp(w)), w)
    assert not plain.requires_grad
    with pytest.raises(RuntimeError, match='leaf'):
        overwrites('this kernel', (w,))
