"""The attention backward kernel against float64 gradients with derived error bounds (B200 only)."""
import numpy as np
import pytest
import torch

from tests.grad_ref import assert_close, attention_grads

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


def inputs(nq, nk, H, D, seed=0):
    q, k, v = rand(nq, H, D, seed=seed), rand(nk, H, D, seed=seed + 1), rand(nk, H, D, seed=seed + 2)
    dlse = rand(H, nq, seed=seed + 4).float()
    return q, k, v, rand(nq, H, D, seed=seed + 3), dlse


def starts(lengths):
    return np.cumsum([0] + list(lengths))[:-1].tolist()


def check_all(got, want):
    from onereel_b200 import attention as A
    torch.cuda.synchronize()
    A.check()
    for n, t in got.items():
        if n == 'lse':
            fin = torch.isfinite(want['lse'][0])
            assert torch.equal(fin, torch.isfinite(t))
            assert (t.double() - want['lse'][0])[fin].abs().max().item() < 1e-4
        else:
            assert_close(t, want[n], n)


CASES = [
    [(1, 2)],
    [(128, 128)],
    [(127, 129), (128, 128), (129, 127)],
    [(256, 300), (257, 5), (300, 1100)],
    [(16, 336), (256, 336), (1, 2050), (600, 77)],
    [(1000, 513), (3, 1000), (130, 1)],
    [(5, 0), (64, 64), (0, 70), (200, 130)],
]


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('H', [1, 3])
@pytest.mark.parametrize('ci', range(len(CASES)))
def test_grads_match_float64(ci, H, D):
    """segments from one row and one key to several tiles, an empty key side, an empty query side; out and lse grads"""
    from onereel_b200 import attention as A
    lq, lk = [a for a, _ in CASES[ci]], [b for _, b in CASES[ci]]
    q, k, v, dout, dlse = inputs(sum(lq), sum(lk), H, D, seed=10 * ci)
    segs = (starts(lq), lq, starts(lk), lk)
    out, lse = A.attend(q, k, v, *segs, lse=True)
    dlse = torch.where(torch.isfinite(lse), dlse, torch.zeros_like(dlse))
    dq, dk, dv = A.attend_grad(q, k, v, out, lse, dout, *segs, dlse=dlse)
    check_all(dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv), attention_grads(q, k, v, dout, *segs, dlse=dlse))
    # without a gradient of the log-sum-exp, and the same bits again
    a = A.attend_grad(q, k, v, out, lse, dout, *segs)
    b = A.attend_grad(q, k, v, out, lse, dout, *segs)
    check_all(dict(zip(('dq', 'dk', 'dv'), a)), attention_grads(q, k, v, dout, *segs))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('D', [64, 128])
def test_varlen_autograd_device_plan_equals_host_plan(D):
    """autograd through varlen / varlen_lse with device cu_seqlens: the host-planned results, bit for bit"""
    from onereel_b200 import attention as A
    lq, lk = [16, 256, 1, 600, 0], [336, 336, 900, 77, 30]
    H = 4
    q, k, v, dout, dlse = inputs(sum(lq), sum(lk), H, D, seed=3)
    for x in (q, k, v):
        x.requires_grad_()
    segs = (starts(lq), lq, starts(lk), lk)
    cq, ck = A.cu_seqlens(lq), A.cu_seqlens(lk)
    out, lse = A.varlen_lse(q, k, v, cq, ck, max(lq), max(lk))
    got = torch.autograd.grad((out, lse), (q, k, v), (dout, dlse))
    host = A.attend_grad(q.detach(), k.detach(), v.detach(), out.detach(), lse.detach(), dout, *segs, dlse=dlse)
    assert all(torch.equal(a, b) for a, b in zip(got, host))
    want = attention_grads(q, k, v, dout, *segs, dlse=dlse)
    check_all(dict(zip(('dq', 'dk', 'dv'), got), out=out.detach(), lse=lse.detach()), want)
    o2 = A.varlen(q, k, v, cq, ck, max(lq), max(lk))
    assert torch.equal(o2, out)
    g2 = torch.autograd.grad(o2, (q, k, v), dout)
    o3 = A.varlen(q, k, v, cq.tolist(), ck.tolist(), max(lq), max(lk))
    g3 = torch.autograd.grad(o3, (q, k, v), dout)
    assert all(torch.equal(a, b) for a, b in zip(g2, g3))
    # the log-sum-exp alone
    _, l4 = A.varlen_lse(q, k, v, cq, ck, max(lq), max(lk))
    g4 = torch.autograd.grad(l4, (q, k, v), dlse)
    want4 = attention_grads(q, k, v, torch.zeros_like(dout), *segs, dlse=dlse)
    check_all(dict(dq=g4[0], dk=g4[1]), want4)
    assert not g4[2].any()


def test_rows_outside_the_segments():
    """cu_seqlens that leave rows before and after the segments: their gradients are zero, and NaN in the keys and
    queries there reaches nothing"""
    from onereel_b200 import attention as A
    H, D = 2, 128
    lq, lk = [70, 130], [200, 300]
    q, k, v, dout, _ = inputs(sum(lq) + 150, sum(lk) + 150, H, D, seed=8)
    segs = ([40, 110], lq, [30, 230], lk)
    nan = float('nan')
    for x, lo, hi in ((q, 40, 240), (dout, 40, 240), (k, 30, 530)):
        x[:lo] = nan
        x[hi:] = nan
    for x in (q, k, v):
        x.requires_grad_()
    cq, ck = (torch.tensor(c, dtype=torch.int32, device='cuda') for c in ([40, 110, 240], [30, 230, 530]))
    out = A.varlen(q, k, v, cq, ck, 130, 300)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    assert not dq[:40].any() and not dq[240:].any()
    for x in (dk, dv):
        assert not x[:30].any() and not x[530:].any()
    want = attention_grads(*(x.detach().nan_to_num() for x in (q, k, v, dout)), *segs)
    check_all(dict(dq=dq, dk=dk, dv=dv), want)


def test_overlapping_key_ranges_sum_their_readers():
    from onereel_b200 import attention as A
    H, D = 2, 128
    qr = [(0, 96), (96, 256), (256, 384)]
    kr = [(0, 160), (64, 300), (10, 384)]
    q, k, v, dout, _ = inputs(384, 390, H, D, seed=5)
    for x in (q, k, v):
        x.requires_grad_()
    out = A.overlapping_ranges(q, k, v, qr, kr)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    segs = tuple(zip(*[(a, b - a, c, d - c) for (a, b), (c, d) in zip(qr, kr)]))
    check_all(dict(dq=dq, dk=dk, dv=dv), attention_grads(q, k, v, dout, *segs))
    assert not dk[384:].any() and not dv[384:].any()


def test_packed_and_dense_autograd():
    """segments that share a tensor get the sum of its gradients; dense with strided inputs; a non-contiguous dout"""
    from onereel_b200 import attention as A
    H, D = 2, 64
    q1, q2, k, v = (rand(n, H, D, seed=s).requires_grad_() for s, n in enumerate((40, 200, 150, 150)))
    g1, g2 = rand(40, H, D, seed=7), rand(200, H, D, seed=8)
    (o1, l1), (o2, l2) = A.packed_lse([(q1, k, v), (q2, k, v)])
    p1, p2 = A.packed([(q1, k, v), (q2, k, v)])
    assert torch.equal(p1, o1) and torch.equal(p2, o2)
    grads = torch.autograd.grad((p1, p2), (q1, q2, k, v), (g1, g2))
    want = attention_grads(torch.cat([q1, q2]), k, v, torch.cat([g1, g2]), [0, 40], [40, 200], [0, 0], [150, 150])
    # k and v are summed over two calls' bf16 results by autograd: one more rounding of each and of the sum
    extra = lambda w: (w[0], 3 * w[1])
    check_all(dict(dq=torch.cat(grads[:2])), want)
    for got, n in zip(grads[2:], ('dk', 'dv')):
        d = (got.double() - want[n][0]).abs()
        assert (d <= extra(want[n])[1]).all()
    B, S = 2, 130
    base = [rand(S, B, H, D, seed=20 + i).requires_grad_() for i in range(3)]
    o = A.dense(*(x.transpose(0, 1) for x in base))
    dout = rand(S, B, H, D, seed=30).transpose(0, 1)
    got = torch.autograd.grad(o, base, dout)
    flat = [x.detach().transpose(0, 1).reshape(B * S, H, D) for x in base]
    want = attention_grads(*flat, dout.reshape(B * S, H, D), [0, S], [S, S], [0, S], [S, S])
    check_all({n: g.transpose(0, 1).reshape(B * S, H, D) for n, g in zip(('dq', 'dk', 'dv'), got)}, want)


def test_gradient_matches_differences():
    """the loss along random directions: central differences of the float64 loss, whose inputs the kernel shares"""
    from onereel_b200 import attention as A
    H, D = 1, 64
    q, k, v, dout, _ = inputs(50, 90, H, D, seed=40)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(A.varlen(q, k, v, [0, 50], [0, 90], 50, 90), leaves, dout)

    def loss(x):
        s = torch.einsum('qhd,khd->hqk', x[0], x[1]) * D ** -0.5
        return (torch.einsum('hqk,khd->qhd', torch.softmax(s, -1), x[2]) * dout.double()).sum()
    base = [x.detach().double() for x in leaves]
    want = attention_grads(q, k, v, dout, [0], [50], [0], [90])
    for i, n in enumerate(('dq', 'dk', 'dv')):
        t = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()
        move = lambda e: [x + e * t if j == i else x for j, x in enumerate(base)]
        diff = ((loss(move(1e-4)) - loss(move(-1e-4))) / 2e-4).item()
        tol = (want[n][1] * t.abs()).sum().item() + 1e-6 * abs(diff)
        assert abs((grads[i].double() * t).sum().item() - diff) <= tol


def test_captured_backward_and_side_stream():
    """forward and backward captured into a graph and replayed on new values; the same call on another stream"""
    from onereel_b200 import attention as A
    H, D, lq, lk = 2, 64, [100, 30], [64, 200]
    q, k, v, dout, _ = inputs(130, 264, H, D, seed=50)
    cq, ck = A.cu_seqlens(lq), A.cu_seqlens(lk)
    leaves = [x.requires_grad_() for x in (q, k, v)]

    def step():
        return torch.autograd.grad(A.varlen(q, k, v, cq, ck, 100, 200), leaves, dout)
    eager = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    with torch.no_grad():
        v.copy_(rand(264, H, D, seed=99))
    # both graphs in flight at once, on two streams
    side.wait_stream(torch.cuda.current_stream())
    graphs[0][0].replay()
    with torch.cuda.stream(side):
        graphs[1][0].replay()
    torch.cuda.current_stream().wait_stream(side)
    want = step()
    for _, res in graphs:
        assert all(torch.equal(a, b) for a, b in zip(res, want))
    A.check()


def test_refusals():
    from onereel_b200 import _lib as L
    from onereel_b200 import attention as A
    H, D = 2, 64
    q, k, v, dout, dlse = inputs(32, 48, H, D)
    out, lse = A.attend(q, k, v, [0], [32], [0], [48], lse=True)
    seg = ([0], [32], [0], [48])
    with pytest.raises(TypeError):
        A.attend_grad(q, k, v, out, lse, dout.float(), *seg)
    with pytest.raises(TypeError):
        A.attend_grad(q.float(), k, v, out, lse, dout, *seg)
    with pytest.raises(ValueError):
        A.attend_grad(q, k, v, out, lse, dout[:31], *seg)
    with pytest.raises(ValueError):
        A.attend_grad(q, k, v, out, lse, dout, *seg, dlse=dlse[:, :30])
    with pytest.raises(L.OrlError):
        A.attend_grad(q, k, v, out, lse, dout, [0, 16], [32, 16], [0, 0], [48, 48])     # a query row twice
    with pytest.raises(L.OrlError):
        A.attend_grad(q, k, v, out, lse, dout, [0], [32], [1], [48])                    # keys past the end
    with pytest.raises(RuntimeError):                                                    # first derivatives only
        x = q.clone().requires_grad_()
        (g,) = torch.autograd.grad(A.varlen(x, k, v, [0, 32], [0, 48], 32, 48).sum(), x, create_graph=True)
        torch.autograd.grad(g.sum(), x)
    # cu_seqlens the device planner rejects: reported through the error word, as in the forward
    bad = torch.tensor([0, 40, 32], dtype=torch.int32, device='cuda')
    ck = torch.tensor([0, 20, 48], dtype=torch.int32, device='cuda')
    A._attend_cu_grad(q, k, v, out, lse, dout, None, bad, ck)
    with pytest.raises(L.OrlError):
        A.check()
    A.check()


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('lk', [2, 3, 7, 31, 64, 65, 129])
def test_few_keys_keep_their_precision(lk, D):
    """with few keys dS is a small difference of large terms: the gradients stay within the two roundings that remain
    (dS or P, and the result), whatever the rounding of out. A rounding's relative error in the 2-norm is
    u sqrt(E[1 / m^2] / 3) = 0.425 u for a significand m spread evenly in its logarithm; a quarter more for the data."""
    from onereel_b200 import attention as A
    H, lq = 3, [300, 40]
    q, k, v, dout, dlse = inputs(sum(lq), 2 * lk, H, D, seed=lk)
    segs = (starts(lq), lq, [0, lk], [lk, lk])
    out, lse = A.attend(q, k, v, *segs, lse=True)
    got = A.attend_grad(q, k, v, out, lse, dout, *segs, dlse=dlse)
    want = attention_grads(q, k, v, dout, *segs, dlse=dlse)
    tol = 1.25 * 2 ** 0.5 * 0.425 * 2.0 ** -8
    for t, n in zip(got, ('dq', 'dk', 'dv')):
        rel = ((t.double() - want[n][0]).norm() / want[n][0].norm()).item()
        assert rel < tol, (n, rel)


@pytest.mark.parametrize('D', [64, 128])
def test_calls_on_two_streams_at_once(D):
    """backward passes that share the GPU (each one's key blocks wait for its own query blocks) give the bits of one alone"""
    from onereel_b200 import attention as A
    H, n = 6, 2500
    q, k, v, dout, _ = inputs(n, n, H, D, seed=21)
    seg = ([0, 900], [900, n - 900], [0, 700], [1500, n - 700])
    out, lse = A.attend(q, k, v, *seg, lse=True)
    want = A.attend_grad(q, k, v, out, lse, dout, *seg)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(A.attend_grad(q, k, v, out, lse, dout, *seg))
    torch.cuda.synchronize()
    A.check()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_one_tensor_in_every_place_and_gradients_of_some():
    """q, k and v one leaf: its gradient is the three roles' sum; gradients asked of v alone; a broadcast dout"""
    from onereel_b200 import attention as A
    H, n, D = 2, 200, 64
    x = rand(n, H, D, seed=30)
    cu = A.cu_seqlens([n])
    leaves = [x.clone().requires_grad_() for _ in range(3)]
    parts = torch.autograd.grad(A.varlen(*leaves, cu, cu, n, n).sum(), leaves)
    one = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(A.varlen(one, one, one, cu, cu, n, n).sum(), one)
    # autograd adds the three in some order and rounds each sum
    total = sum(p.double() for p in parts)
    assert (g.double() - total).abs().max().item() <= 2.0 ** -7 * sum(p.double().abs() for p in parts).max().item()
    v = x.clone().requires_grad_()
    (gv,) = torch.autograd.grad(A.varlen(x, x, v, cu, cu, n, n).sum(), v)
    assert torch.equal(gv, parts[2])
    # Elementwise bounds, not the norm's two roundings: here s_ii = |x_i|^2 / 8 is about 8 where the others are about 1, so
    # P_ii is near 1 and dS_ii = P_ii (dP_ii - delta_i) a difference of sums over 64 elements of size 1 that nearly
    # cancel: out's rounding alone moves delta_i by u |sum_d o_id| / sqrt(3), some 0.02, against dS of a few tenths.
    want = attention_grads(x, x, x, torch.ones_like(x), [0], [n], [0], [n])
    for p, name in zip(parts, ('dq', 'dk', 'dv')):
        assert ((p.double() - want[name][0]).abs() <= want[name][1]).all(), name


def test_captured_host_planned_calls_outlive_the_plan_cache(monkeypatch):
    """forward and backward of overlapping ranges captured after a first call, replayed when the caches have dropped
    hundreds of layouts since and their memory has been given out again: the replay's own work lists are still there"""
    from onereel_b200 import attention as A
    H, D = 2, 64
    qr, kr = [(0, 90), (90, 250)], [(0, 150), (40, 260)]
    q, k, v, dout, _ = inputs(250, 260, H, D, seed=60)

    def step():
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        return torch.autograd.grad(A.overlapping_ranges(*leaves, qr, kr), leaves, dout)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for n in range(1, 700):
        A.plan([0], [n], [0], [n], H, q.device)
        A._plan_bwd([0], [n], [0], [n], H, n, n, q.device)
    key = next(iter(A._BWD_PLANS.held))
    assert key not in A._BWD_PLANS.entries and len(A._BWD_PLANS.entries) <= A._BWD_PLANS.limit
    junk = [torch.full((4096,), 7, dtype=torch.int32, device='cuda') for _ in range(600)]
    with torch.no_grad():
        q.copy_(rand(250, H, D, seed=70))
    graph.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(res, want))
    A.check()
    del junk


def test_first_use_of_a_layout_in_a_capture_is_refused():
    """host-planned calls and packs say so instead of ending the capture; the same calls work afterwards"""
    from onereel_b200 import attention as A
    H, D = 1, 64
    q, k, v, dout, _ = inputs(37, 41, H, D, seed=80)
    leaf = q.clone().requires_grad_()
    torch.cuda.synchronize()
    for call in (lambda: A.overlapping_ranges(q, k, v, [(0, 37)], [(3, 41)]), lambda: A.packed([(q, k, v)]),
                 lambda: A.dense(q[None, :31], k[None, :29], v[None, :29])):
        with pytest.raises(RuntimeError, match='once before capturing'):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        call()
    (want,) = torch.autograd.grad(A.overlapping_ranges(leaf, k, v, [(0, 37)], [(3, 41)]), leaf, dout)
    torch.cuda.synchronize()
    A.check()
    assert want.shape == q.shape


@pytest.mark.parametrize('H,D', [(40, 128), (24, 64), (7, 128)])
def test_many_heads(H, D):
    from onereel_b200 import attention as A
    lq, lk = [33, 200], [150, 65]
    q, k, v, dout, dlse = inputs(sum(lq), sum(lk), H, D, seed=H)
    segs = (starts(lq), lq, starts(lk), lk)
    out, lse = A.attend(q, k, v, *segs, lse=True)
    dq, dk, dv = A.attend_grad(q, k, v, out, lse, dout, *segs, dlse=dlse)
    check_all(dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv), attention_grads(q, k, v, dout, *segs, dlse=dlse))


@pytest.mark.parametrize('n', [1000, 4096])
def test_many_segments_on_the_device_plan(n):
    """thousands of short segments, empty ones among them: the device-planned passes give the host-planned bits, which match
    float64; one segment more than the device plan takes is refused by both passes"""
    from onereel_b200 import _lib as L, attention as A
    H, D = 2, 64
    g = torch.Generator().manual_seed(n)
    lq = torch.randint(0, 6, (n,), generator=g).tolist()
    lk = (2 + torch.randint(0, 9, (n,), generator=g)).tolist()
    lq[3], lk[5], lk[7], lq[n // 2], lk[n // 2] = 0, 0, 300, 260, 200
    q, k, v, dout, _ = inputs(sum(lq), sum(lk), H, D, seed=n)
    segs = (starts(lq), lq, starts(lk), lk)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    cq, ck = A.cu_seqlens(lq), A.cu_seqlens(lk)
    out, lse = A.varlen_lse(*leaves, cq, ck, max(lq), max(lk))
    got = torch.autograd.grad(out, leaves, dout)
    plain = [x.detach() for x in leaves]
    want_o, want_l = A.attend(*plain, *segs, lse=True)
    host = A.attend_grad(*plain, want_o, want_l, dout, *segs)
    assert torch.equal(out, want_o) and torch.equal(lse, want_l) and all(torch.equal(a, b) for a, b in zip(got, host))
    want = attention_grads(*plain, dout, *segs)
    torch.cuda.synchronize()
    A.check()
    for name, t in dict(out=out.detach(), dq=got[0], dk=got[1], dv=got[2]).items():
        assert ((t.double() - want[name][0]).abs() <= want[name][1]).all(), name
    if n == 4096:
        more = torch.zeros(n + 2, dtype=torch.int32, device='cuda')
        for call in (lambda: A.varlen(q, k, v, more, more, 1, 1),
                     lambda: A._attend_cu_grad(*plain, want_o, want_l, dout, None, more, more)):
            with pytest.raises(L.OrlError):
                call()


def test_long_segment():
    """thousands of rows on both sides: tens of tiles per item in either kind, rows past the last whole tile"""
    from onereel_b200 import attention as A
    H, D, lq, lk = 1, 128, [4001, 900], [7003, 12001]
    q, k, v, dout, dlse = inputs(sum(lq), sum(lk), H, D, seed=90)
    segs = (starts(lq), lq, starts(lk), lk)
    out, lse = A.attend(q, k, v, *segs, lse=True)
    dq, dk, dv = A.attend_grad(q, k, v, out, lse, dout, *segs, dlse=dlse)
    check_all(dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv), attention_grads(q, k, v, dout, *segs, dlse=dlse))


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('lq,lk', [([0, 0], [40, 7]), ([33, 150], [0, 0]), ([0], [0]), ([], [])])
def test_no_queries_and_no_keys(lq, lk, D):
    """tensors without rows on either side, through every entry point: zeros (log-sum-exp -inf) and zero gradients"""
    from onereel_b200 import attention as A
    H = 2
    q, k, v, dout, _ = inputs(sum(lq), sum(lk), H, D, seed=1)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    cq, ck = A.cu_seqlens(lq), A.cu_seqlens(lk)
    calls = [lambda *t: A.varlen_lse(*t, cq, ck, 200, 40), lambda *t: A.varlen_lse(*t, cq.tolist(), ck.tolist(), 200, 40)]
    if len(lq) == 2:
        ranges = [(0, lq[0]), (lq[0], sum(lq))], [(0, lk[0]), (lk[0], sum(lk))]
        calls.append(lambda *t: (A.overlapping_ranges(*t, *ranges), None))
    for call in calls:
        with torch.no_grad():
            plain = call(q, k, v)
        out, lse = call(*leaves)
        assert out.shape == q.shape and not out.any() and torch.equal(out, plain[0])
        assert lse is None or (lse == -float('inf')).all()
        grads = torch.autograd.grad(out, leaves, dout)
        assert all(g.shape == x.shape and not g.any() for g, x in zip(grads, leaves))
    torch.cuda.synchronize()
    A.check()


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('lq,lk', [([70, 300], [130, 200]), ([1, 129], [5, 64]), ([200, 57], [65, 400]), ([256, 128], [63, 1])])
def test_a_segment_beside_a_bad_one(lq, lk, D):
    """the next segment's q, k, v and dout all NaN: the first segment's gradients keep their bits, planned on either side"""
    from onereel_b200 import attention as A
    H = 2
    data = inputs(sum(lq), sum(lk), H, D, seed=lq[0])[:4]
    cq, ck = A.cu_seqlens(lq), A.cu_seqlens(lk)
    for plan in (lambda c: c, lambda c: c.tolist()):
        res = []
        for bad in (False, True):
            x = [t.clone() for t in data]
            if bad:
                for t, n in zip(x, (lq[0], lk[0], lk[0], lq[0])):
                    t[n:] = float('nan')
            leaves = [t.requires_grad_() for t in x[:3]]
            out = A.varlen(*leaves, plan(cq), plan(ck), max(lq), max(lk))
            dq, dk, dv = torch.autograd.grad(out, leaves, x[3])
            res.append((out.detach()[:lq[0]], dq[:lq[0]], dk[:lk[0]], dv[:lk[0]]))
        for a, b in zip(*res):
            assert torch.isfinite(a).all() and torch.equal(a, b)
    torch.cuda.synchronize()
    A.check()
