"""Training through the framework's own paths on one GPU: the processors' scene attention, the gradient of the pack, and a
fused DiT block end to end (linear layers, q/k norm + rotary embedding, scene attention, their gradients) against the same
model in float64 (B200 only)."""
import copy

import pytest
import torch
import torch.nn.functional as F

from oracle import layout_oracle as LO
from tests.grad_ref import F as FP32, U, assert_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module', autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip('needs a B200')
    from onereel_b200.csrc.build import build
    build()


def rand(*shape, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(*shape, generator=g)).cuda().to(torch.bfloat16)


def rel(x, y):
    return ((x.double() - y.double()).norm() / y.double().norm()).item()


def scene_attention(lay, T, counts, q, k, v, eq, ek, ev, rotate=None):
    """the oracle's segments in the inputs' precision, differentiable; rotate(scene, keys) -> keys"""
    olay = LO.Layout(lay.lengths, lay.halo, lay.sides, lay.extra)
    L = lay.n_frames * T
    segs = LO.hunyuan_segments(olay, T, counts, LO.scene_pieces(olay, T, (0, L))[0], set(range(olay.n_scenes)))
    Q, K, V = (torch.cat([x, e]) for x, e in ((q, eq), (k, ek), (v, ev)))
    idx = lambda rows: torch.tensor([L + r[1] if isinstance(r, tuple) else r for r in rows], device=q.device)
    rows, outs = [], []
    for kind, j, qr, kr in segs:
        if not len(qr):
            continue
        kk = K[idx(kr)]
        if rotate is not None and kind == 'v':
            kk = rotate(j, kk)
        s = torch.einsum('qhd,khd->hqk', Q[idx(qr)], kk) * q.shape[-1] ** -0.5
        outs.append(torch.einsum('hqk,khd->qhd', torch.softmax(s, -1), V[idx(kr)]))
        rows.append(idx(qr))
    out = torch.cat(outs)[torch.argsort(torch.cat(rows))]
    return out[:L], out[L:]


@pytest.mark.parametrize('shared_pos', ['source', 'adjacent'])
@pytest.mark.parametrize('D', [64, 128])
def test_scene_processor_gradients(D, shared_pos):
    """Processor.scene with shared frames (rows packed for several scenes) and text: values bit-equal to the call without
    gradients, gradients of all six inputs within two roundings in the 2-norm (dS or P, the packed rows, their sum)"""
    from onereel_b200 import attention as A, hunyuan15 as HY, standin
    from onereel_b200.layout import SceneLayout
    lay = SceneLayout([3, 2, 4], halo=1, extra={0: [7], 2: [0]})
    T, H, counts = 48, 2, [7, 9, 5]
    L = lay.n_frames * T
    ctx = HY.Context(lay, T=T, counts={True: counts}, fwd=1, own=[(0, L)], shared_pos=shared_pos)
    cos, sin = (t.cuda() for t in standin.rope_3d(lay.n_frames, 6, 8, D, axes=(16, 56, 56) if D == 128 else (8, 28, 28)))
    ctx._rot_full = (cos, sin)
    x = [rand(n, H, D, seed=i) for i, n in enumerate((L, L, L, *[sum(counts)] * 3))]
    gv, gt = rand(L, H, D, seed=10), rand(sum(counts), H, D, seed=11)
    with torch.no_grad():
        want_v, want_t = HY.Processor(ctx, 0).scene(*x)
    leaves = [t.requires_grad_() for t in x]
    ov, ot = HY.Processor(ctx, 0).scene(*leaves)
    assert torch.equal(ov, want_v) and torch.equal(ot, want_t)
    got = torch.autograd.grad((ov, ot), leaves, (gv, gt))
    torch.cuda.synchronize()
    A.check()

    def rotate(j, kk):
        shared = lay.shared_frames(j)
        if not shared:
            return kk
        n = len(lay.frames[j]) * T
        ar, br = (r.cuda() for r in HY._shift_rows(ctx, j))
        ca, sa, cb, sb = (t.double()[:, None] for t in (cos[ar], sin[ar], cos[br], sin[br]))
        c, s = cb * ca + sb * sa, sb * ca - cb * sa
        part = kk[n:n + len(shared) * T]
        xr, xi = part.unflatten(-1, (-1, 2)).unbind(-1)
        turned = part * c + torch.stack([-xi, xr], -1).flatten(-2) * s
        return torch.cat([kk[:n], turned, kk[n + len(shared) * T:]])
    wide = [t.detach().double().requires_grad_() for t in x]
    rv, rt = scene_attention(lay, T, counts, *wide, rotate=rotate if shared_pos == 'adjacent' else None)
    want = torch.autograd.grad((rv, rt), wide, (gv.double(), gt.double()))
    for n, a, b in zip(('q', 'k', 'v', 'eq', 'ek', 'ev'), got, want):
        assert rel(a, b) < 2 * U, (n, rel(a, b))


def test_wan_ranges_gradients():
    """scenes with extra frames (packed) and without (key ranges read in place)"""
    from onereel_b200 import attention as A, wan
    from onereel_b200.layout import SceneLayout
    T, H, D = 32, 2, 64
    for extra in ({}, {0: [5], 2: [0, 4]}):
        lay = SceneLayout([3, 2, 4], halo=1, extra=extra)
        L = lay.n_frames * T
        ctx = wan.Context(lay, T=T, own=[(0, L)])
        x = [rand(L, H, D, seed=i) for i in range(3)]
        g = rand(L, H, D, seed=5)
        with torch.no_grad():
            want_o = wan.Processor(ctx, 'self', None, 0).ranges(*x)
        leaves = [t.requires_grad_() for t in x]
        o = wan.Processor(ctx, 'self', None, 0).ranges(*leaves)
        assert torch.equal(o, want_o)
        got = torch.autograd.grad(o, leaves, g)
        A.check()
        wide = [t.detach().double().requires_grad_() for t in x]
        outs = []
        for j, (lo, hi) in enumerate(lay.ranges):
            rows = torch.cat([torch.arange(f * T, (f + 1) * T) for f in lay.key_frames(j)]).cuda()
            s = torch.einsum('qhd,khd->hqk', wide[0][lo * T:hi * T], wide[1][rows]) * D ** -0.5
            outs.append(torch.einsum('hqk,khd->qhd', torch.softmax(s, -1), wide[2][rows]))
        want = torch.autograd.grad(torch.cat(outs), wide, g.double())
        for n, a, b in zip('qkv', got, want):
            assert rel(a, b) < 2 * U, (n, rel(a, b))


@pytest.mark.parametrize('rows,H,D,n', [(50, 2, 64, 200), (3, 1, 8, 7), (40, 16, 128, 11), (5, 3, 64, 0)])
def test_row_sum(rows, H, D, n):
    """sums of copies, rows without any, many copies of one row; bf16 sums in fp32: one rounding"""
    from onereel_b200.pack import RowSum
    g = torch.Generator().manual_seed(n)
    src = torch.randint(0, rows, (n,), generator=g)
    src[:n // 3] = rows - 1
    parts = [rand(max(n, 1), H, D, seed=s) for s in (1, 2)]
    got = RowSum(src.numpy(), torch.arange(n).numpy(), rows, 'cuda').run(parts)
    for p, x in zip(parts, got):
        want = torch.zeros(rows, H, D, dtype=torch.float64, device='cuda').index_add_(0, src.cuda(), p[:n].double())
        size = torch.zeros_like(want).index_add_(0, src.cuda(), p[:n].double().abs())
        assert_close(x, (want, U * want.abs() + FP32 * size + 1e-30), 'row sum')


class _PlainProcessor:
    """the attention layer in torch operations of the model's precision (wide: float64, else bf16 with fp32 inside)"""

    def __init__(self, ctx):
        self.ctx = ctx

    def __call__(self, attn, hs, ehs, mask, rot):
        ctx = self.ctx
        inner = torch.float64 if hs.dtype == torch.float64 else torch.float32

        def norm(x, m):
            return F.rms_norm(x.to(inner), (x.shape[-1],), m.weight.to(inner), m.eps)

        def prep(x, m):
            x = norm(x.unflatten(2, (attn.heads, -1))[0], m)
            xr, xi = x.unflatten(-1, (-1, 2)).unbind(-1)
            c, s = (t.to(inner)[:, None] for t in rot)
            return (x * c + torch.stack([-xi, xr], -1).flatten(-2) * s).to(hs.dtype)
        q, k = prep(attn.to_q(hs), attn.norm_q), prep(attn.to_k(hs), attn.norm_k)
        v = attn.to_v(hs).unflatten(2, (attn.heads, -1))[0]
        eq, ek, ev = (f(ehs).unflatten(2, (attn.heads, -1))[0] for f in (attn.add_q_proj, attn.add_k_proj, attn.add_v_proj))
        eq, ek = norm(eq, attn.norm_added_q).to(hs.dtype), norm(ek, attn.norm_added_k).to(hs.dtype)
        ov, ot = scene_attention(ctx.layout, ctx.T, ctx.counts[True], *(t.to(inner) for t in (q, k, v, eq, ek, ev)))
        return (attn.to_out[0](ov.to(hs.dtype).flatten(1, 2)[None]), attn.to_add_out(ot.to(hs.dtype).flatten(1, 2)[None]))


def test_fused_block_trains():
    """two blocks, forward and backward: every parameter's gradient is at most twice as far from float64 as the same
    model's in bf16 torch operations (which rounds the same stored tensors; the kernels round P and dS besides) or within
    four roundings, and the values likewise"""
    from onereel_b200 import attention as A, hunyuan15 as HY, standin
    from onereel_b200.layout import SceneLayout
    lay = SceneLayout([3, 2, 4], halo=1, extra={0: [5], 2: [0]})
    T, counts = 48, [7, 9, 5]
    L = lay.n_frames * T
    ctx = HY.Context(lay, T=T, counts={True: counts, False: counts}, own=[(0, L)], fwd=1)
    fused = standin.build(ctx, 'cuda', dim=256, heads=2, blocks=2, seed=3, fused=True)
    plain = standin.build(ctx, 'cuda', dim=256, heads=2, blocks=2, seed=3)
    for blk in plain.transformer_blocks:
        blk.attn.processor = _PlainProcessor(ctx)
    with torch.no_grad():                                  # gates and biases that are not zero
        for i, (a, b) in enumerate(zip(fused.parameters(), plain.parameters())):
            assert torch.equal(a, b)
            if a.dim() == 1:
                a.add_(rand(*a.shape, seed=100 + i, std=0.3))
                b.copy_(a)
    wide = copy.deepcopy(plain).double()
    hs, ehs, temb = rand(1, L, 256, seed=1), rand(1, sum(counts), 256, seed=2), rand(1, 256, seed=3)
    cos, sin = (t.cuda() for t in standin.rope_3d(lay.n_frames, 6, 8, 128))
    gv, gt = rand(1, L, 256, seed=4), rand(1, sum(counts), 256, seed=5)

    def step(model, dtype):
        x = [t.to(dtype).requires_grad_() for t in (hs, ehs, temb)]
        out = model(*x, (cos, sin))
        params = list(model.parameters())
        grads = torch.autograd.grad(out, x + params, (gv.to(dtype), gt.to(dtype)))
        return [o.detach() for o in out] + list(grads)
    a, b, c = step(fused, torch.bfloat16), step(plain, torch.bfloat16), step(wide, torch.float64)
    torch.cuda.synchronize()
    A.check()
    names = ['video', 'text', 'd video', 'd text', 'd temb'] + [n for n, _ in fused.named_parameters()]
    assert len(names) == len(a) == len(b) == len(c)
    for n, x, y, z in zip(names, a, b, c):
        if z.norm() == 0:
            assert not x.any(), n
            continue
        assert rel(x, z) <= max(2 * rel(y, z), 4 * U), (n, rel(x, z), rel(y, z))
    again = step(fused, torch.bfloat16)
    assert all(torch.equal(x, y) for x, y in zip(a, again))


def test_backward_captures_while_an_eager_graph_lives():
    """a training step captured into a graph with an eager graph of the same tensors alive, then replayed on new inputs.
    The step takes fresh leaves of its tensors: with the eager graph's own leaves, torch's engine waits for the stream
    that built them, which invalidates a capture whatever the operators are (F.linear alone does it too)."""
    from onereel_b200 import attention as A
    from onereel_b200.linear import linear
    H, D, n = 2, 64, 96
    x = rand(n, H * D, seed=1).requires_grad_()
    w = rand(3 * H * D, H * D, seed=2, std=0.1).requires_grad_()
    g = rand(n, H, D, seed=3)
    cu = A.cu_seqlens([40, 56])

    def out(x, w):
        q, k, v = (t.contiguous().view(n, H, D) for t in linear(x, w).chunk(3, -1))
        return A.varlen(q, k, v, cu, cu, 56, 56)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w)]
        return torch.autograd.grad(out(*leaves), leaves, g)
    step()
    alive = out(x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    with torch.no_grad():
        x.copy_(rand(n, H * D, seed=9))
    graph.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(res, want))
    del alive
    A.check()


def test_forward_mode_tangents_are_refused():
    """every differentiable entry point, with and without an input that requires a gradient"""
    from torch.autograd import forward_ad

    from onereel_b200 import attention as A
    from onereel_b200.linear import linear
    from onereel_b200.rope import qk_norm_rope
    H, D, n = 2, 64, 10
    x, w = rand(n, H, D, seed=1), rand(H * D, H * D, seed=2)
    cos, sin = torch.ones(n, D, device='cuda'), torch.zeros(n, D, device='cuda')
    cu = A.cu_seqlens([n])
    calls = [lambda t: A.varlen(t, x, x, cu, cu, n, n), lambda t: A.varlen_lse(x, t, x, cu, cu, n, n),
             lambda t: A.varlen(x, x, t, [0, n], [0, n], n, n), lambda t: A.packed([(t, x, x)]),
             lambda t: A.packed_lse([(x, t, x)]), lambda t: A.overlapping_ranges(x, x, t, [(0, n)], [(0, n)]),
             lambda t: A.dense(t[None], x[None], x[None]), lambda t: linear(t.view(n, -1), w),
             lambda t: linear(t.view(n, -1), w.requires_grad_()),
             lambda t: qk_norm_rope(t.view(n, -1), w[0, :D].detach(), cos, sin, H, 1e-6, True, 0)]
    for call in calls:
        call(x)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(NotImplementedError):
                call(dual)
    A.check()


def test_paths_without_gradients_raise_in_the_backward_pass():
    """bounded memory, Ulysses and the ring, for both models: the same bits as without autograd, and an error where a
    training step would leave the attention out of its gradients"""
    from onereel_b200 import hunyuan15 as HY, ring as R, wan
    from onereel_b200.layout import SceneLayout
    lay = SceneLayout([3, 2, 4], halo=0)
    T, H, D, counts = 16, 2, 64, [7, 9, 5]
    L = lay.n_frames * T
    x = [rand(n, H, D, seed=i) for i, n in enumerate((L, L, L, *[sum(counts)] * 3))]
    scale = torch.ones(D, device='cuda', dtype=torch.bfloat16, requires_grad=True)

    def hunyuan(**kw):
        return HY.Processor(HY.Context(lay, T=T, counts={True: counts}, fwd=1, own=[(0, L)], **kw), 0)

    def wan_(**kw):
        return wan.Processor(wan.Context(lay, T=T, own=[(0, L)], fwd=1, **kw), 'self', None, 0)
    calls = [lambda *t: hunyuan(memory=8).memory(*t), lambda *t: hunyuan().ulysses(*t),
             lambda *t: wan_(memory=8).memory(*t[:3]), lambda *t: wan_().scene(*t[:3]),
             lambda *t: R.attention(R.RingPlan(lay, 1, T), *t, [(0, 7), (7, 16), (16, 21)], 0)]
    for call in calls:
        with torch.no_grad():
            want = call(*x)
        got = call(*(t * scale for t in x))
        pairs = list(zip(got, want)) if isinstance(got, tuple) else [(got, want)]
        for a, b in pairs:
            assert torch.equal(a, b)
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(a.float().sum() + scale.float().sum(), scale)


def test_in_place_kernels_raise_in_the_backward_pass():
    """merging two key parts' results, accumulating one, rotating rows, norm + rope into a buffer: the bits of a call without
    autograd, and an error in the backward pass where a gradient would come out wrong"""
    from onereel_b200 import attention as A
    from onereel_b200.rope import qk_norm_rope, rotate_rows
    H, D, n, m = 2, 64, 40, 90
    x = [rand(r, H, D, seed=i) for i, r in enumerate((n, m, m))]
    cut = lambda t, lo, hi: t[lo:hi].contiguous()
    cos, sin = torch.full((n, D), 0.6, device='cuda'), torch.full((n, D), 0.8, device='cuda')
    rows = torch.arange(0, n, 2, dtype=torch.int32, device='cuda')

    def parts(q, k, v):
        return [A.varlen_lse(q, cut(k, lo, hi), cut(v, lo, hi), [0, n], [0, hi - lo], n, hi - lo)
                for lo, hi in ((0, 30), (30, m))]

    def merge(q, k, v):
        (o, l), (o2, l2) = parts(q, k, v)
        return A.lse_merge(o, l, o2, l2)

    def merge_second_only(q, k, v):
        with torch.no_grad():
            o, l = parts(q, k, v)[0]
        return A.lse_merge(o, l, *parts(q, k, v)[1])

    def accumulate(q, k, v):
        acc, l = torch.zeros(n, H, D, device='cuda'), torch.full((H, n), -float('inf'), device='cuda')
        for o2, l2 in parts(q, k, v):
            A.lse_merge_acc(acc, l, o2, l2)
        return acc, l
    calls = [merge, merge_second_only, accumulate, lambda q, k, v: (rotate_rows(q.clone(), rows, cos, sin),),
             lambda q, k, v: (qk_norm_rope(q.reshape(n, -1), torch.ones(D, device='cuda'), cos, sin, H, 1e-6, True, 0,
                                           out=torch.empty_like(q)),)]
    leaves = [t.clone().requires_grad_() for t in x]
    for call in calls:
        with torch.no_grad():
            want = call(*x)
        got = call(*leaves)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for t in got:
            with pytest.raises((NotImplementedError, RuntimeError), match='carries no gradients'):
                torch.autograd.grad(t.float().sum() + sum(y.float().sum() for y in leaves), leaves, retain_graph=True)
    # the first part's own backward pass does not run on the merged values
    (o, l), second = parts(*leaves)
    head = o[:5] * 2
    A.lse_merge(o, l, *second)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(head.float().sum(), leaves)
    A.check()


def test_phase_marks_with_and_without_gradients(monkeypatch):
    """the scene path marks the same phases in the same order whether or not it records a backward pass"""
    from onereel_b200 import hunyuan15 as HY
    from onereel_b200.layout import SceneLayout
    lay = SceneLayout([2, 3], halo=1)
    T, H, D, counts = 16, 2, 64, [3, 4]
    L = lay.n_frames * T
    proc = HY.Processor(HY.Context(lay, T=T, counts={True: counts}, fwd=1, own=[(0, L)]), 0)
    x = [rand(n, H, D, seed=i) for i, n in enumerate((L, L, L, 7, 7, 7))]
    seen = []
    for grad in (False, True):
        monkeypatch.setattr(HY, 'PHASES', [])
        proc.scene(*(t.clone().requires_grad_(grad) for t in x))
        seen.append([name for name, _ in HY.PHASES])
    assert seen[0] == seen[1] and seen[0][0] == 'start' and 'near' in seen[0]


@pytest.mark.parametrize('shared_pos', ['source', 'adjacent'])
def test_captured_scene_step(shared_pos):
    """a training step of Processor.scene captured after a first one, replayed on new values when the work-list caches have
    been emptied of its layout since"""
    from onereel_b200 import attention as A, hunyuan15 as HY, standin
    from onereel_b200.layout import SceneLayout
    lay = SceneLayout([3, 2, 4], halo=1, extra={0: [7], 2: [0]})
    T, H, D, counts = 48, 2, 64, [7, 0, 5]
    L = lay.n_frames * T
    ctx = HY.Context(lay, T=T, counts={True: counts}, fwd=1, own=[(0, L)], shared_pos=shared_pos)
    ctx._rot_full = tuple(t.cuda() for t in standin.rope_3d(lay.n_frames, 6, 8, D, axes=(8, 28, 28)))
    proc = HY.Processor(ctx, 0)
    x = [rand(n, H, D, seed=i) for i, n in enumerate((L, L, L, *[sum(counts)] * 3))]
    gv, gt = rand(L, H, D, seed=10), rand(sum(counts), H, D, seed=11)

    def step():
        leaves = [t.detach().requires_grad_() for t in x]
        out = proc.scene(*leaves)
        return (*(t.detach() for t in out), *torch.autograd.grad(out, leaves, (gv, gt)))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for n in range(1, 700):
        A.plan([0], [n], [0], [n], H, x[0].device)
        A._plan_bwd([0], [n], [0], [n], H, n, n, x[0].device)
    x[0].copy_(rand(L, H, D, seed=50))
    x[4].copy_(rand(sum(counts), H, D, seed=51))
    graph.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(res, want))
    A.check()


def test_scene_step_without_text_rows():
    """sentences of no tokens: the text side is empty, the video side is the layer's without text"""
    from onereel_b200 import attention as A, hunyuan15 as HY, wan
    from onereel_b200.layout import SceneLayout
    lay = SceneLayout([2, 3], halo=1, extra={0: [4]})
    T, H, D = 16, 2, 64
    L = lay.n_frames * T
    x = [rand(n, H, D, seed=i).requires_grad_() for i, n in enumerate((L, L, L, 0, 0, 0))]
    g = rand(L, H, D, seed=9)
    proc = HY.Processor(HY.Context(lay, T=T, counts={True: [0, 0]}, fwd=1, own=[(0, L)]), 0)
    with torch.no_grad():
        want_v, want_t = proc.scene(*x)
    ov, ot = proc.scene(*x)
    assert torch.equal(ov, want_v) and ot.shape == want_t.shape == (0, H, D)
    got = torch.autograd.grad((ov, ot), x, (g, torch.empty_like(ot)))
    o = wan.Processor(wan.Context(lay, T=T, own=[(0, L)]), 'self', None, 0).ranges(*x[:3])
    assert torch.equal(o, ov)
    want = torch.autograd.grad(o, x[:3], g)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(t.shape == (0, H, D) for t in got[3:])
    A.check()
