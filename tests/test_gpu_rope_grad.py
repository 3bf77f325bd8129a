"""The q/k RMSNorm + RoPE gradient kernel against float64 (B200 only). Everything up to the stored dx and dweight is fp32:
the bounds are one rounding to bf16 (u = 2^-8 of the value) and f = 2^-14 of the sums' absolute terms."""
import pytest
import torch

from tests.grad_ref import F, U, assert_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module', autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip('needs a B200')
    from onereel_b200.csrc.build import build
    build()


def make(rows, heads, dh, per_head, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (2 * torch.randn(rows, heads * dh, generator=g)).cuda().bfloat16()
    w = (1 + 0.2 * torch.randn(dh if per_head else heads * dh, generator=g)).cuda().bfloat16()
    ang = torch.randn(rows, dh // 2, generator=g) * 3
    cos, sin = ang.cos().repeat_interleave(2, -1).cuda(), ang.sin().repeat_interleave(2, -1).cuda()
    return x, w, cos, sin, torch.randn(rows, heads, dh, generator=g).cuda().bfloat16()


def reference(x, w, cos, sin, dy, heads, eps, per_head, shift):
    """(dx, bound), (dw, bound)"""
    rows, dh = x.shape[0], x.shape[1] // heads
    X, W, G = x.detach().double(), w.detach().double(), dy.double()
    X = X.view(rows, heads, dh) if per_head else X
    c, s = cos.double()[:, None, 0::2], sin.double()[:, None, shift::2]
    u = torch.stack([G[..., 0::2] * c + G[..., 1::2] * s, G[..., 1::2] * c - G[..., 0::2] * s], -1).reshape(X.shape)
    inv = ((X * X).mean(-1, keepdim=True) + eps).rsqrt()
    wu = W * u
    dx = inv * wu - X * inv ** 3 * (wu * X).mean(-1, keepdim=True)
    size = inv * wu.abs() + X.abs() * inv ** 3 * (wu * X).abs().mean(-1, keepdim=True)
    t = u * X * inv
    dims = (0, 1) if per_head else 0
    dw, dw_size = t.sum(dims), t.abs().sum(dims)
    return ((dx.reshape(rows, -1), (U * dx.abs() + F * size).reshape(rows, -1) + 1e-30),
            (dw, U * dw.abs() + F * dw_size + 1e-30))


@pytest.mark.parametrize('rows', [1, 2, 7, 1001, 5000])
@pytest.mark.parametrize('heads,dh,per_head', [(16, 128, True), (12, 128, False), (4, 64, True), (3, 64, False),
                                               (1, 64, False), (1, 8, True), (64, 128, False)])
def test_gradients(rows, heads, dh, per_head):
    check_gradients(rows, heads, dh, per_head)


@pytest.mark.parametrize('rows', [1, 149, 2003])
@pytest.mark.parametrize('heads,dh,per_head', [(40, 128, False), (40, 128, True), (13, 96, False), (60, 40, False),
                                               (3, 256, True), (5, 24, False), (1, 8192, False), (9, 256, False)])
def test_gradients_of_rows_over_several_warps_and_odd_heads(rows, heads, dh, per_head):
    check_gradients(rows, heads, dh, per_head)


def check_gradients(rows, heads, dh, per_head):
    from onereel_b200.rope import qk_norm_rope
    shift = 0 if per_head else 1
    x, w, cos, sin, dy = make(rows, heads, dh, per_head, seed=rows)
    with torch.no_grad():
        plain = qk_norm_rope(x, w, cos, sin, heads, 1e-6, per_head, shift)
    x.requires_grad_()
    w.requires_grad_()
    y = qk_norm_rope(x, w, cos, sin, heads, 1e-6, per_head, shift)
    assert torch.equal(y, plain)
    dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    again = torch.autograd.grad(y, (x, w), dy)
    wx, ww = reference(x, w, cos, sin, dy, heads, 1e-6, per_head, shift)
    assert_close(dx, wx, 'dx')
    assert_close(dw, ww, 'dw')
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


def test_zero_row_and_other_weight_types():
    """a row of zeros (inv = eps^-1/2), an fp32 weight and half tables, a batch dimension, a transposed dy"""
    from onereel_b200.rope import qk_norm_rope
    heads, dh, rows = 2, 64, 9
    x, w, cos, sin, dy = make(rows, heads, dh, True, seed=3)
    x[4] = 0
    wf = w.float().requires_grad_()
    xb = x[None].clone().requires_grad_()
    y = qk_norm_rope(xb, wf, cos, sin, heads, 1e-4, True, 0)
    g = dy.transpose(0, 1).contiguous().transpose(0, 1)
    dx, dw = torch.autograd.grad(y, (xb, wf), g)
    assert dx.shape == xb.shape and dw.dtype == torch.float32
    wx, ww = reference(x, w, cos, sin, dy, heads, 1e-4, True, 0)
    assert_close(dx[0], wx, 'dx')
    assert_close(dw, ww, 'dw')


def test_gradient_matches_differences():
    from onereel_b200.rope import qk_norm_rope
    heads, dh, rows = 2, 8, 5
    x, w, cos, sin, dy = make(rows, heads, dh, False, seed=6)
    x.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(qk_norm_rope(x, w, cos, sin, heads, 1e-6, False, 0), (x, w), dy)
    wx, ww = reference(x, w, cos, sin, dy, heads, 1e-6, False, 0)

    def loss(X, W):
        n = X * ((X * X).mean(-1, keepdim=True) + 1e-6).rsqrt() * W
        n = n.view(rows, heads, dh // 2, 2)
        c, s = cos.double()[:, None, 0::2], sin.double()[:, None, 0::2]
        y = torch.stack([n[..., 0] * c - n[..., 1] * s, n[..., 0] * s + n[..., 1] * c], -1).view(rows, heads, dh)
        return (y * dy.double()).sum()
    X, W = x.detach().double(), w.detach().double()
    for got, (_, bound), f, base in ((dx, wx, lambda t: loss(t, W), X), (dw, ww, lambda t: loss(X, t), W)):
        v = torch.randn(base.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64).cuda()
        diff = ((f(base + 1e-5 * v) - f(base - 1e-5 * v)) / 2e-5).item()
        assert abs((got.double() * v).sum().item() - diff) <= (bound * v.abs()).sum().item() + 1e-6 * (1 + abs(diff))


def test_refusals():
    from onereel_b200.rope import qk_norm_rope_grad
    x, w, cos, sin, dy = make(6, 2, 64, True)
    with pytest.raises(TypeError):
        qk_norm_rope_grad(x, w, cos, sin, dy.float(), 2, 1e-6, True, 0)
    with pytest.raises(ValueError):
        qk_norm_rope_grad(x, w, cos, sin, dy[:5], 2, 1e-6, True, 0)


@pytest.mark.parametrize('heads,dh,per_head', [(5, 64, True), (1, 128, True), (3, 128, True), (1, 8, True), (4, 64, True),
                                               (5, 24, False), (16, 128, False)])
@pytest.mark.parametrize('eps', [0.0, 1e-2])
def test_gradients_without_and_with_a_large_epsilon(heads, dh, per_head, eps):
    """rows whose elements are not a multiple of a warp's 256 columns: the lanes without elements add nothing, also where
    only eps stands between their sum of squares (0) and a division by it"""
    from onereel_b200.rope import qk_norm_rope
    x, w, cos, sin, dy = make(67, heads, dh, per_head, seed=heads)
    x.requires_grad_()
    w.requires_grad_()
    y = qk_norm_rope(x, w, cos, sin, heads, eps, per_head, 0)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    wx, ww = reference(x, w, cos, sin, dy, heads, eps, per_head, 0)
    assert_close(dx, wx, 'dx')
    assert_close(dw, ww, 'dw')


@pytest.mark.parametrize('per_head', [True, False])
@pytest.mark.parametrize('dtype', [torch.float32, torch.float64])
def test_no_rows(per_head, dtype):
    from onereel_b200.rope import qk_norm_rope
    heads, dh = 3, 64
    x = torch.empty(0, heads * dh, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(dh if per_head else heads * dh, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    table = torch.empty(0, dh, device='cuda', dtype=dtype)
    with torch.no_grad():
        assert qk_norm_rope(x, w, table, table, heads, 1e-6, per_head, 0).shape == (0, heads, dh)
    y = qk_norm_rope(x, w, table, table, heads, 1e-6, per_head, 0)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape and not dw.any()
