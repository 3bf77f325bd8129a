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
calls = dict(linear=lambda t: linear(t.view(100, 256), w).view(100, 4, 64), varlen=lambda t: A.varlen(t, k, v, cq, ck, 100, 300),
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
