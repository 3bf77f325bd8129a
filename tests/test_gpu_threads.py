"""Calls from threads that have made no CUDA call yet (a server's worker, autograd's own thread): the kernels' tensor maps are
encoded by a driver call, which needs the device's context on the calling thread (B200 only)."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope='module', autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip('needs a B200')
    from onereel_b200.csrc.build import build
    build()


def in_a_thread(call):
    res = []

    def run():
        try:
            res.append(call())
        except Exception as e:                            # noqa: BLE001 (raised below)
            res.append(e)
    t = threading.Thread(target=run)
    t.start()
    t.join()
    if isinstance(res[0], Exception):
        raise res[0]
    return res[0]


def test_forward_calls_from_a_new_thread():
    from onereel_b200 import attention as A
    from onereel_b200.linear import linear
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, 4, 64, generator=g).cuda().bfloat16() for n in (100, 300, 300))
    w = torch.randn(512, 256, generator=g).cuda().bfloat16()
    cq, ck = A.cu_seqlens([100]), A.cu_seqlens([300])
    calls = [lambda: A.varlen(q, k, v, cq, ck, 100, 300), lambda: A.varlen(q, k, v, [0, 100], [0, 300], 100, 300),
             lambda: linear(q.view(100, 256), w), lambda: linear(q.view(100, 256)[:2], w)]
    for call in calls:
        want = call()
        torch.cuda.synchronize()
        got = in_a_thread(call)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    A.check()


@pytest.mark.parametrize('op', ['linear', 'varlen', 'overlapping_ranges', 'rope'])
def test_a_processs_first_backward_pass(op):
    """in a new process the pass is the first thing that autograd's thread does"""
    code = f'''
import torch
from onereel_b200 import attention as A
from onereel_b200.linear import linear
from onereel_b200.rope import qk_norm_rope
g = torch.Generator().manual_seed(0)
x, k, v, dy = (torch.randn(n, 4, 64, generator=g).cuda().bfloat16() for n in (100, 300, 300, 100))
w = torch.randn(256, 256, generator=g).cuda().bfloat16()
one, c = torch.ones(64, device='cuda').bfloat16(), torch.ones(100, 64, device='cuda')
cq, ck = A.cu_seqlens([100]), A.cu_seqlens([300])
calls = dict(linear=lambda t: linear(t.view(100, 256), w).view(100, 4, 64),
             varlen=lambda t: A.varlen(t, k, v, cq, ck, 100, 300),
             overlapping_ranges=lambda t: A.overlapping_ranges(t, k, v, [(0, 100)], [(0, 300)]),
             rope=lambda t: qk_norm_rope(t.view(100, 256), one, c, c, 4, 1e-6, True, 0))
warm = torch.empty(64 << 20, dtype=torch.uint8, device='cuda')        # what the pass allocates comes from the allocator's cache
del warm
leaf = x.requires_grad_()
(d,) = torch.autograd.grad(calls[{op!r}](leaf), leaf, dy)
torch.cuda.synchronize()
A.check()
assert torch.isfinite(d).all() and d.any()
'''
    r = subprocess.run([sys.executable, '-c', code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_threads_on_their_own_streams_share_the_plan_caches(monkeypatch):
    """three threads, each with a stream of its own, run layouts that keep pushing one another's work lists out of a cache of
    four: every result has the bits of the same call alone"""
    from onereel_b200 import attention as A
    H, D = 2, 64
    g = torch.Generator().manual_seed(5)
    q, k, v, dout = (torch.randn(400, H, D, generator=g).cuda().bfloat16() for _ in range(4))
    layouts = [([(0, n), (n, 400)], [(0, 400 - n // 2), (n // 3, 400)]) for n in range(20, 380, 23)]

    def step(qr, kr):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = A.overlapping_ranges(*leaves, qr, kr)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))
    want = [step(*x) for x in layouts]
    torch.cuda.synchronize()
    monkeypatch.setattr(A, '_PLANS', A._Plans(limit=4))
    monkeypatch.setattr(A, '_BWD_PLANS', A._Plans(limit=4))
    errors = []

    def run(first):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(60):
                    j = (first + i) % len(layouts)
                    if not all(torch.equal(a, b) for a, b in zip(step(*layouts[j]), want[j])):
                        errors.append(f'layout {j} differs')
        except Exception as e:                            # noqa: BLE001 (reported below)
            errors.append(repr(e))
    threads = [threading.Thread(target=run, args=(5 * t,)) for t in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    A.check()
    assert not errors, errors[:3]
    assert len(A._PLANS.entries) <= 4 and len(A._BWD_PLANS.entries) <= 4
