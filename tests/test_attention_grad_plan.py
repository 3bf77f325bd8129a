"""The backward work list (orl_attn_bwd_plan, host only): every row of q, k is covered once per head, every key row's
ranges are the query rows of the segments that read it."""
import ctypes

import numpy as np
import pytest


@pytest.fixture(scope='module')
def lib():
    from onereel_b200.csrc.build import build
    build()
    from onereel_b200 import _lib
    return _lib


def plan(lib, segs, heads, nq, nk):
    a = [np.ascontiguousarray([s[i] for s in segs], np.int32) for i in range(4)]
    args = [lib.i32p(x) for x in a] + [len(segs), heads, nq, nk]
    m = ctypes.c_int(0)
    f = lib.lib().orl_attn_bwd_plan
    n = f(*args, None, 0, None, 0, m)
    if n > -1000:
        return n, None, None
    work = np.zeros(-n - 1000, lib.BWD_WORK_DTYPE)
    ranges = np.zeros((max(m.value, 1), 2), np.int32)
    assert f(*args, work.ctypes.data, len(work), ranges.ctypes.data, m.value, m) == len(work)
    return len(work), work, ranges[:m.value]


CASES = [
    ([(0, 300, 0, 10), (300, 257, 10, 4990)], 600, 5001),
    ([(10, 20, 5, 0), (40, 129, 5, 128)], 200, 140),
    ([(0, 96, 0, 160), (96, 160, 64, 236), (256, 128, 10, 374)], 384, 390),
    ([(0, 5, 0, 5), (5, 0, 0, 5), (5, 7, 0, 5)], 12, 5),
    ([], 3, 130),
    ([(0, 1, 0, 1)], 1, 1),
]


@pytest.mark.parametrize('ci', range(len(CASES)))
@pytest.mark.parametrize('heads', [1, 3])
def test_plan_covers_every_row_once(lib, ci, heads):
    segs, nq, nk = CASES[ci]
    n, work, ranges = plan(lib, segs, heads, nq, nk)
    seen = np.zeros((2, heads, max(nq, nk)), int)
    cost = []
    for w in work:
        assert 1 <= w['rows'] <= 128
        rows = np.arange(w['row0'], w['row0'] + w['rows'])
        seen[w['kind'], w['head'], rows] += 1
        got = [tuple(r) for r in ranges[w['range0']:w['range0'] + w['n_ranges']]]
        for r in rows:
            if w['kind'] == 0:
                want = [(q0, lq) for q0, lq, k0, lk in segs if lq > 0 and k0 <= r < k0 + lk]
            else:
                want = [(k0, lk) for q0, lq, k0, lk in segs if q0 <= r < q0 + lq]
            assert got == want
        tile = 128 if w['kind'] == 0 else 64
        assert w['n_tiles'] == sum((x + tile - 1) // tile for _, x in got)
        assert w['whole'] == (w['kind'] == 1 and bool(got) and 0 < got[0][1] <= 64)     # one tile holds all its keys
        cost.append((w['kind'], w['n_tiles']))                          # queries first, longest first
    assert (seen[0, :, :nk] == 1).all() and (seen[1, :, :nq] == 1).all()
    assert cost == sorted(cost, reverse=True)


def test_plan_refuses(lib):
    assert plan(lib, [(0, 10, 0, 5), (9, 3, 0, 5)], 1, 20, 5)[0] == -1       # a query row in two segments
    assert plan(lib, [(0, 10, 0, 6)], 1, 20, 5)[0] == -1                     # keys past the end
    assert plan(lib, [(0, 21, 0, 5)], 1, 20, 5)[0] == -1
    assert plan(lib, [(0, -1, 0, 5)], 1, 20, 5)[0] == -1
    assert plan(lib, [(0, 1, 0, 1)], 0, 1, 1)[0] == -1
    assert plan(lib, [], 1, 0, 0)[0] == 0


def test_backward_refuses_bad_arguments_without_a_gpu(lib):
    h = lib.lib()
    p = 4096                                                                 # never dereferenced: refused before
    ok = [p] * 6 + [None] + [p] * 3 + [8, 8, 2, 64, 0.125]
    tail = [p, 1, p, p, p, None]
    bad = lambda i, x: h.orl_attn_bwd(*(ok[:i] + [x] + ok[i + 1:]), *tail)
    assert bad(0, None) == -1 and bad(7, None) == -1 and bad(14, 0.0) == -1 and bad(12, 0) == -1 and bad(10, -1) == -1
    assert bad(13, 96) == -3
    assert bad(4, p + 8) == -2 and bad(9, p + 2) == -2
    assert h.orl_attn_bwd_cu_scratch(-1, 0, 0, 1) == -1
    need = h.orl_attn_bwd_cu_scratch(300, 200, 2, 3)
    assert need == 32 * (1 + 3 * (3 + 2 + 8)) + 32
    cu = [p, p, 2, p, need - 1, p, p, None]
    assert h.orl_attn_bwd_cu(*ok[:10], 300, 200, 3, 64, 0.125, *cu) == -7
    cu[2] = 5000
    assert h.orl_attn_bwd_cu(*ok[:10], 300, 200, 3, 64, 0.125, *cu) == -7
