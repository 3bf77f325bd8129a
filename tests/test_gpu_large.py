"""Tensors of more than 2^31 elements: the last rows' results and gradients are the bits of the same rows computed alone
(B200 only; up to 50 GB)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module', autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip('needs a B200')
    from onereel_b200.csrc.build import build
    build()
    yield
    torch.cuda.empty_cache()


def generator():
    g = torch.Generator(device='cuda').manual_seed(0)
    return g, lambda *shape: torch.randn(*shape, generator=g, device='cuda', dtype=torch.bfloat16)


def test_linear():
    from onereel_b200 import attention as A
    from onereel_b200.linear import linear
    _, r = generator()
    m, n, k = 270_001, 8192, 64
    leaves = [t.requires_grad_() for t in (r(m, k), r(n, k), r(n), r(n))]
    dy = r(m, n)
    assert dy.numel() > 2 ** 31
    x, w, b, gate = leaves
    y = linear(x, w, b, 'silu', None, gate)
    dx, _, db, _ = torch.autograd.grad(y, leaves, dy)
    tail = slice(m - 300, m)
    xt = x.detach()[tail].contiguous().requires_grad_()
    yt = linear(xt, w, b, 'silu', None, gate)
    (dxt,) = torch.autograd.grad(yt, xt, dy[tail])
    assert torch.equal(y[tail], yt) and torch.equal(dx[tail], dxt)
    want = torch.zeros(n, dtype=torch.float64, device='cuda')
    for i in range(0, m, 30_000):
        z = (x.detach()[i:i + 30_000].float() @ w.detach().float().T + b.detach().float()).double()
        s = torch.sigmoid(z)
        want += (dy[i:i + 30_000].double() * gate.detach().double() * (s * (1 + z * (1 - s)))).sum(0)
    # z was kept as bf16: half a step of it moves the slope of every row, at random; then one rounding of the sum
    assert ((db.double() - want).norm() / want.norm()).item() < 2 * 2.0 ** -8
    torch.cuda.synchronize()
    A.check()


def test_attention():
    from onereel_b200 import attention as A
    _, r = generator()
    H, D, length, n = 16, 128, 4000, 270
    rows = length * n + 77
    q, k, v, dout = (r(rows, H, D) for _ in range(4))
    assert q.numel() > 2 ** 31
    leaves = [t.requires_grad_() for t in (q, k, v)]
    cu = A.cu_seqlens([length] * n + [77])
    out, lse = A.varlen_lse(*leaves, cu, cu, length, length)
    grads = torch.autograd.grad(out, leaves, dout)
    tail = slice(rows - length - 77, rows)
    small = [t.detach()[tail].contiguous().requires_grad_() for t in leaves]
    cu = A.cu_seqlens([length, 77])
    want, want_l = A.varlen_lse(*small, cu, cu, length, length)
    want_g = torch.autograd.grad(want, small, dout[tail].contiguous())
    torch.cuda.synchronize()
    A.check()
    assert torch.equal(out[tail], want) and torch.equal(lse[:, tail], want_l)
    assert all(torch.equal(a[tail], b) for a, b in zip(grads, want_g))


@pytest.mark.parametrize('per_head', [True, False])
def test_norm_rope(per_head):
    from onereel_b200 import attention as A
    from onereel_b200.rope import qk_norm_rope
    g, r = generator()
    H, D, rows = 16, 128, 1_060_003
    x, dy = r(rows, H * D).requires_grad_(), r(rows, H, D)
    assert x.numel() > 2 ** 31
    w = torch.ones(D if per_head else H * D, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    cos, sin = (torch.rand(rows, D, generator=g, device='cuda') for _ in range(2))
    y = qk_norm_rope(x, w, cos, sin, H, 1e-6, per_head, 0)
    dx, _ = torch.autograd.grad(y, (x, w), dy)
    tail = slice(rows - 100, rows)
    xt = x.detach()[tail].contiguous().requires_grad_()
    yt = qk_norm_rope(xt, w, cos[tail].contiguous(), sin[tail].contiguous(), H, 1e-6, per_head, 0)
    (dxt,) = torch.autograd.grad(yt, xt, dy[tail])
    torch.cuda.synchronize()
    A.check()
    assert torch.equal(y[tail], yt) and torch.equal(dx[tail], dxt)


def test_row_sum():
    import numpy as np

    from onereel_b200.pack import RowSum
    _, r = generator()
    n = 1_060_000
    part = r(n, 16, 128)
    assert part.numel() > 2 ** 31
    source = np.concatenate([np.arange(n // 2)] * 2)
    (out,) = RowSum(source, np.arange(n), n // 2, 'cuda').run([part])
    want = (part[n // 2 - 1000:n // 2].float() + part[-1000:].float()).to(torch.bfloat16)
    assert torch.equal(out[-1000:], want)
