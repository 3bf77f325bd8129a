"""The fused linear kernels against float64 with derived elementwise bounds (B200 only).

u = 2^-8: half a bf16 step, once for every value the kernels round (y, z kept for the backward, dz, every gradient);
f = 2^-14 for what is held in fp32 (sums in the tensor cores, the activation's exponential). With |act'| <= 1.13 and
|act''| <= 0.8 for both activations:
  e_z  = f |x| |w|^T                                    e_y  = u |y| + |gate| (1.13 e_z + f |act|)
  e_dz = u |dz| + |gate dy| (0.8 (u |z| + e_z) + f)     e_dx = u |dx| + e_dz |w| + f |dz| |w|   (dw alike)
  e_db = u |db| + sum e_dz                              e_dg = u |dg| + sum |dy| (1.13 (u |z| + e_z) + f |act|)
"""
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


def rand(*shape, seed=0, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(*shape, generator=g) + mean).cuda().to(torch.bfloat16)


def make(m, n, k, bias=True, residual=False, gate=False, seed=0):
    t = dict(x=rand(m, k, seed=seed), weight=rand(n, k, seed=seed + 1, std=k ** -0.5))
    if bias:
        t['bias'] = rand(n, seed=seed + 2, std=0.3)
    if residual:
        t['residual'] = rand(m, n, seed=seed + 3)
    if gate:
        t['gate'] = rand(n, seed=seed + 4, std=0.5, mean=0.3)
    return t


def reference(t, act, dy=None):
    """name -> (float64 value, bound) of y and, given dy, of the gradients"""
    d = {n: x.detach().double() for n, x in t.items()}
    x, w = d['x'], d['weight']
    z = (x @ w.T + d.get('bias', 0)).requires_grad_()
    h = {None: lambda v: v, 'silu': torch.nn.functional.silu,
         'gelu_tanh': lambda v: torch.nn.functional.gelu(v, approximate='tanh')}[act](z)
    (slope,) = torch.autograd.grad(h.sum(), z)
    z, h = z.detach(), h.detach()
    gate = d.get('gate', torch.ones(w.shape[0], dtype=torch.float64, device=x.device))
    y = h * gate + d.get('residual', 0)
    ez = F * (x.abs() @ w.abs().T + z.abs())
    r = {'y': (y, U * y.abs() + gate.abs() * (1.13 * ez + F * h.abs()) + F * y.abs())}
    if dy is not None:
        g = dy.double()
        dz = g * gate * slope
        kept = act is not None or 'gate' in d
        e = (U * dz.abs() + (g * gate).abs() * (0.8 * (U * z.abs() + ez) * (act is not None) + F)) * kept
        r['x'] = (dz @ w, U * (dz @ w).abs() + e @ w.abs() + F * dz.abs() @ w.abs())
        r['weight'] = (dz.T @ x, U * (dz.T @ x).abs() + e.T @ x.abs() + F * dz.abs().T @ x.abs())
        r['bias'] = (dz.sum(0), U * dz.sum(0).abs() + e.sum(0) + F * dz.abs().sum(0))
        dg = (g * h).sum(0)
        r['gate'] = (dg, U * dg.abs() + (g.abs() * (1.13 * (U * z.abs() + ez) + F * h.abs())).sum(0))
        r['residual'] = (g, torch.full_like(g, 1e-30))
    return {n: (v, 1.1 * b + 1e-30) for n, (v, b) in r.items()}


SIZES = [(1, 8, 8), (1, 96, 2048), (2, 264, 72), (4, 64, 136), (5, 8, 8), (77, 512, 320), (130, 200, 1000),
         (256, 256, 64), (300, 136, 72), (1000, 1032, 264)]


@pytest.mark.parametrize('m,n,k', SIZES)
@pytest.mark.parametrize('act,residual,gate', [(None, False, False), ('gelu_tanh', False, False), ('silu', True, True)])
def test_forward_and_gradients(m, n, k, act, residual, gate):
    from onereel_b200 import attention as A
    from onereel_b200.linear import linear
    t = make(m, n, k, residual=residual, gate=gate, seed=m)
    with torch.no_grad():
        plain = linear(t['x'], t['weight'], t['bias'], act, t.get('residual'), t.get('gate'))
    for x in t.values():
        x.requires_grad_()
    y = linear(t['x'], t['weight'], t['bias'], act, t.get('residual'), t.get('gate'))
    assert torch.equal(y, plain)
    dy = rand(m, n, seed=m + 9)
    grads = dict(zip(t, torch.autograd.grad(y, list(t.values()), dy, retain_graph=True)))
    again = torch.autograd.grad(y, list(t.values()), dy)
    torch.cuda.synchronize()
    A.check()
    want = reference(t, act, dy)
    assert_close(y, want['y'], 'y')
    for i, name in enumerate(t):
        assert_close(grads[name], want[name], name)
        assert torch.equal(grads[name], again[i]), name


def test_large_tiles():
    """enough 256 x 256 tiles for the two-CTA kernel in every direction, with ragged ends"""
    from onereel_b200 import attention as A
    from onereel_b200.linear import linear
    t = make(2100, 2056, 2312, residual=True, gate=True, seed=1)
    for x in t.values():
        x.requires_grad_()
    dy = rand(2100, 2056, seed=8)
    y = linear(**t, activation='gelu_tanh')
    grads = dict(zip(t, torch.autograd.grad(y, list(t.values()), dy)))
    torch.cuda.synchronize()
    A.check()
    want = reference(t, 'gelu_tanh', dy)
    assert_close(y, want['y'], 'y')
    for name in t:
        assert_close(grads[name], want[name], name)


@pytest.mark.parametrize('m', [3, 200])
def test_views_and_layouts(m):
    """row-strided and misaligned views, a transposed weight, leading dimensions, an expanded incoming gradient"""
    from onereel_b200.linear import linear
    n, k = 64, 128
    big = rand(m, 3 * k + 8, seed=1)
    t = dict(x=big[:, k:2 * k], weight=rand(k, n, seed=2, std=0.1).t(), bias=rand(n + 1, seed=3)[1:],
             residual=rand(m, 2 * n, seed=4)[:, n:], gate=rand(n, 2, seed=5)[:, 0])
    want = reference(t, 'silu')['y']
    assert_close(linear(**t, activation='silu'), want, 'strided')
    odd = big[:, 3:3 + k]                                     # rows 6 bytes off a 16-byte boundary
    assert_close(linear(odd, t['weight']), reference(dict(x=odd, weight=t['weight']), None)['y'], 'misaligned')
    x3 = rand(2, m, k, seed=6).requires_grad_()
    gate = rand(n, seed=7).requires_grad_()
    y = linear(x3, t['weight'].contiguous(), gate=gate[None, None])
    assert y.shape == (2, m, n)
    dx, dg = torch.autograd.grad(y.sum(), (x3, gate))
    flat = dict(x=x3.reshape(-1, k), weight=t['weight'], gate=gate)
    want = reference(flat, None, torch.ones(2 * m, n, device='cuda'))
    assert_close(dx.reshape(-1, k), want['x'], 'dx')
    assert_close(dg, want['gate'], 'dgate')
    e = linear(x3[:, :0], t['weight'])
    assert e.shape == (2, 0, n)
    z = x3[:, :0].detach().requires_grad_()
    w = t['weight'].contiguous().requires_grad_()
    dz, dw = torch.autograd.grad(linear(z, w).sum(), (z, w))
    assert dz.shape == z.shape and not dw.any()


def test_activation_extremes():
    """large arguments of both signs: no NaN, the limits of the function and its slope"""
    from onereel_b200.linear import linear
    k = 8
    vals = [0.0, -0.0, 1e-4, -1e-4, 5.0, -5.0, 60.0, -60.0, 1e4, -1e4, 1e30, -1e30]
    x = torch.zeros(len(vals), k).index_put((torch.arange(len(vals)), torch.zeros(len(vals), dtype=torch.long)),
                                            torch.tensor(vals)).cuda().bfloat16().requires_grad_()
    w = torch.eye(k).cuda().bfloat16()
    for act in ('gelu_tanh', 'silu'):
        y = linear(x, w, activation=act)
        (dx,) = torch.autograd.grad(y.sum(), x)
        v = x.detach().double()[:, 0].clamp(-1e9, 1e9).requires_grad_()     # float64 z^3 stays finite
        ref = {'silu': torch.nn.functional.silu, 'gelu_tanh': lambda a: torch.nn.functional.gelu(a, approximate='tanh')}
        r = ref[act](v)
        (s,) = torch.autograd.grad(r.sum(), v)
        assert torch.isfinite(y).all() and torch.isfinite(dx).all()
        fin = x.detach()[:, 0].abs() <= 1e4
        assert ((y[:, 0].double() - r)[fin].abs() <= (U + F) * r[fin].abs() + 1e-30).all()
        assert ((dx[:, 0].double() - s)[fin].abs() <= (U + F) * s[fin].abs() + 2 * U).all()
        assert y[-2, 0] == x[-2, 0] and y[-1, 0] == 0 and dx[-2, 0] == 1 and dx[-1, 0] == 0


def test_gradient_matches_differences():
    from onereel_b200.linear import linear
    t = make(20, 16, 24, residual=True, gate=True, seed=3)
    for x in t.values():
        x.requires_grad_()
    dy = rand(20, 16, seed=4)
    grads = dict(zip(t, torch.autograd.grad(linear(**t, activation='gelu_tanh'), list(t.values()), dy)))
    want = reference(t, 'gelu_tanh', dy)
    base = {n: x.detach().double() for n, x in t.items()}

    def loss(d):
        h = torch.nn.functional.gelu(d['x'] @ d['weight'].T + d['bias'], approximate='tanh')
        return ((h * d['gate'] + d['residual']) * dy.double()).sum()
    for i, n in enumerate(t):
        v = torch.randn(base[n].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()
        diff = ((loss({**base, n: base[n] + 1e-5 * v}) - loss({**base, n: base[n] - 1e-5 * v})) / 2e-5).item()
        tol = (want[n][1] * v.abs()).sum().item() + 1e-6 * abs(diff) + 1e-6
        assert abs((grads[n].double() * v).sum().item() - diff) <= tol, n


def test_capture_and_streams():
    """a training step captured into a graph and replayed on new inputs; the same step on another stream"""
    from onereel_b200.linear import linear
    t = make(300, 128, 256, residual=True, gate=True, seed=5)
    leaves = [x.requires_grad_() for x in t.values()]
    dy = rand(300, 128, seed=6)

    def step():
        y = linear(**t, activation='silu')
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    eager = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    with torch.no_grad():
        t['x'].copy_(rand(300, 256, seed=77))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(res, step()))


def test_refusals():
    from onereel_b200.linear import linear
    t = make(4, 16, 24)
    x, w, b = t['x'], t['weight'], t['bias']
    with pytest.raises(TypeError):
        linear(x.float(), w)
    with pytest.raises(TypeError):
        linear(x, w.cpu())
    with pytest.raises(TypeError):
        linear(x, w, b.half())
    with pytest.raises(ValueError):
        linear(x, w[:, :16])
    with pytest.raises(ValueError):
        linear(x[:, :20], w[:, :20].contiguous())
    with pytest.raises(ValueError):
        linear(x, w, b[:8])
    with pytest.raises(ValueError):
        linear(x, w, activation='relu')
    with pytest.raises(ValueError):
        linear(x, w, residual=x)
    with pytest.raises(ValueError):
        linear(x, w, gate=x[:1, :8])


@pytest.mark.parametrize('act', [None, 'silu'])
def test_gradient_of_the_residual_alone_and_of_no_rows(act):
    from onereel_b200.linear import linear
    g = torch.Generator().manual_seed(5)
    w = torch.randn(64, 128, generator=g).cuda().bfloat16()
    x = torch.randn(5, 128, generator=g).cuda().bfloat16()
    gate = torch.randn(64, generator=g).cuda().bfloat16()
    residual = torch.randn(5, 64, generator=g).cuda().bfloat16().requires_grad_()
    dy = torch.randn(5, 64, generator=g).cuda().bfloat16()
    (dr,) = torch.autograd.grad(linear(x, w, None, act, residual, gate), residual, dy)
    assert torch.equal(dr, dy)
    none = torch.empty(0, 128, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    leaf, b, gt = w.clone().requires_grad_(), gate.clone().requires_grad_(), gate.clone().requires_grad_()
    y = linear(none, leaf, b, act, None, gt)
    grads = torch.autograd.grad(y, (none, leaf, b, gt), torch.empty_like(y))
    assert [t.shape for t in grads] == [none.shape, leaf.shape, b.shape, gt.shape] and not any(t.any() for t in grads)


def test_infinite_gate_reaches_only_its_own_column():
    """a row strip's missing second row adds nothing, not 0 * inf, to the column sums"""
    from onereel_b200.linear import linear
    g = torch.Generator().manual_seed(6)
    x, w = (torch.randn(*s, generator=g).cuda().bfloat16() for s in ((9, 64), (64, 64)))
    b = torch.zeros(64, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    gate = torch.ones(64, device='cuda', dtype=torch.bfloat16)
    gate[3] = float('inf')
    (db,) = torch.autograd.grad(linear(x, w, b, None, None, gate), b, torch.ones(9, 64, device='cuda', dtype=torch.bfloat16))
    want = torch.full_like(db, 9.0)
    want[3] = float('inf')
    assert torch.equal(db, want)


@pytest.mark.parametrize('m', [3, 150])
@pytest.mark.parametrize('act,with_gate', [(None, False), (None, True), ('gelu_tanh', False), ('silu', True)])
def test_frozen_inputs_keep_only_what_the_others_gradients_need(m, act, with_gate):
    """every set of inputs that want gradients: the bits of the call where all do, and no tensor kept without a use"""
    from itertools import combinations

    from onereel_b200.linear import linear
    n, k = 72, 136
    t = make(m, n, k, residual=True, gate=with_gate, seed=m)
    dy = rand(m, n, seed=9)

    def grads(names):
        kept = []
        d = {a: x.detach().requires_grad_(a in names) for a, x in t.items()}
        with torch.autograd.graph.saved_tensors_hooks(lambda x: kept.append(tuple(x.shape)) or x, lambda x: x):
            y = linear(**d, activation=act)
        return dict(zip(names, torch.autograd.grad(y, [d[a] for a in names], dy))), sorted(kept)
    full = grads(tuple(t))[0]
    for size in range(1, len(t) + 1):
        for names in combinations(t, size):
            got, kept = grads(names)
            assert all(torch.equal(got[a], full[a]) for a in names), names
            slope = any(a in names for a in ('x', 'weight', 'bias'))
            want = [(m, k)] * ('weight' in names) + [(n, k)] * ('x' in names) + [(n,)] * (with_gate and slope)
            want += [(m, n)] * ('gate' in names or (act is not None and slope))
            assert kept == sorted(want), names


@pytest.mark.parametrize('act,residual,gate', [(None, False, False), ('silu', True, True), ('gelu_tanh', True, False)])
@pytest.mark.parametrize('m,n,k', [(1801, 1504, 1000), (1000, 2056, 1024)])
def test_middle_tiles(m, n, k, act, residual, gate):
    """sizes between the one-CTA tiles and 256 x 256: the pair's 256 x 128 tile, in every direction's operand layout at the
    first size (y: 96 tiles, dx: 64, dw: 48) and with ragged ends"""
    from onereel_b200 import attention as A
    from onereel_b200.linear import linear
    t = make(m, n, k, residual=residual, gate=gate, seed=m)
    for x in t.values():
        x.requires_grad_()
    dy = rand(m, n, seed=8)
    y = linear(t['x'], t['weight'], t['bias'], act, t.get('residual'), t.get('gate'))
    grads = dict(zip(t, torch.autograd.grad(y, list(t.values()), dy)))
    torch.cuda.synchronize()
    A.check()
    want = reference(t, act, dy)
    assert_close(y, want['y'], 'y')
    for name in t:
        assert_close(grads[name], want[name], name)


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('m,n,k', [(3, 72, 136), (77, 200, 1000), (1801, 1504, 1000), (2100, 2056, 520)])
def test_values_that_are_not_finite_stay_where_they_belong(m, n, k, bad):
    """a bad element of x or dy reaches its row of y and dx, one of the weight its column, one of the residual itself; what lies
    around strided operands (here all of it bad) reaches nothing"""
    from onereel_b200.linear import linear
    t = make(m, n, k, residual=True, gate=True, seed=m)
    dy = rand(m, n, seed=9)

    def inside(v):
        big = torch.full((v.shape[0] + 2, v.shape[1] + 16), bad, dtype=v.dtype, device='cuda')
        big[1:-1, 8:-8] = v
        return big[1:-1, 8:-8]

    def grads(d, g):
        leaves = {a: x.detach().requires_grad_() for a, x in d.items()}
        y = linear(**leaves, activation='silu')
        return (y.detach(), *torch.autograd.grad(y, [leaves['x'], leaves['weight'], leaves['bias']], g))
    clean = grads(t, dy)
    assert all(torch.isfinite(x).all() for x in clean)
    wrapped = {a: inside(v) if v.dim() == 2 else v for a, v in t.items()}
    assert all(torch.equal(a, b) for a, b in zip(grads(wrapped, inside(dy)), clean))
    row, col = m // 2, n // 3

    def put(name, at):
        v = t[name].clone()
        v[at] = bad
        return {**t, name: v}
    y, dx, *_ = grads(put('x', (row, 5)), dy)
    keep = torch.arange(m, device='cuda') != row
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert not torch.isfinite(y[row]).all()
    y = grads(put('weight', (col, 5)), dy)[0]
    cols = torch.arange(n, device='cuda') != col
    assert torch.equal(y[:, cols], clean[0][:, cols]) and not torch.isfinite(y[:, col]).all()
    y, dx, dw, db = grads(put('residual', (row, col)), dy)
    want = clean[0].clone()
    want[row, col] = bad
    assert torch.equal(y.nan_to_num(nan=123.0), want.nan_to_num(nan=123.0))
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), clean[1:]))
    g = dy.clone()
    g[row, col] = bad
    y, dx, dw, db = grads(t, g)
    rows = torch.arange(n, device='cuda') != col
    assert torch.equal(y, clean[0]) and torch.equal(dx[keep], clean[1][keep]) and not torch.isfinite(dx[row]).any()
    assert torch.equal(dw[rows], clean[2][rows]) and torch.equal(db[rows], clean[3][rows]) and not torch.isfinite(db[col])
