"""The C entry points of the linear layers and of the norm + rope gradients refuse bad arguments before touching a GPU;
the Python layer refuses CPU tensors."""
import pytest
import torch


@pytest.fixture(scope='module')
def h():
    from onereel_b200.csrc.build import build
    build()
    from onereel_b200 import _lib
    return _lib.lib()


P = 4096                                      # an address that is never dereferenced: the calls refuse before


def with_(args, **at):
    return [at.get(f'a{i}', a) for i, a in enumerate(args)]


def test_linear_refuses(h):
    ok = [P, 64, P, 64, P, P, P, 32, P, None, 5, 32, 64, 0, P, None]
    call = lambda **at: h.orl_linear(*with_(ok, **at))
    assert call(a0=None) == -1 and call(a2=None) == -1 and call(a8=None) == -1 and call(a14=None) == -1
    assert call(a10=-1) == -1 and call(a11=0) == -1 and call(a13=3) == -1 and call(a13=-1) == -1
    assert call(a1=56) == -1 and call(a3=56) == -1 and call(a7=24) == -1
    assert call(a11=36) == -2 and call(a12=60) == -2 and call(a1=68) == -2 and call(a4=P + 2) == -2
    assert call(a10=0) == 0                                              # no rows: nothing to do


def test_linear_gradients_refuse(h):
    ok = [P, 32, P, 64, P, 64, P, P, 1, P, P, P, P, P, P, 5, 32, 64, P, None]
    call = lambda **at: h.orl_linear_bwd(*with_(ok, **at))
    assert call(a0=None) == -1 and call(a2=None) == -1 and call(a4=None) == -1 and call(a18=None) == -1
    assert call(a6=None) == -1 and call(a9=None) == -1 and call(a14=None) == -1 and call(a8=7) == -1
    assert call(a1=24) == -1 and call(a3=56) == -1 and call(a5=56) == -1 and call(a15=-1) == -1 and call(a16=0) == -1
    assert call(a1=36) == -2 and call(a3=68) == -2 and call(a5=68) == -2 and call(a16=30) == -2 and call(a17=60) == -2
    assert call(a10=P + 8) == -2 and call(a6=P + 4) == -2
    assert h.orl_linear_bwd_scratch(-1, 8, 8) == -1 and h.orl_linear_bwd_scratch(5, 12, 8) == -1
    # one partial row per strip of eight rows or more, for each of the two sums
    assert h.orl_linear_bwd_scratch(5, 32, 64) == 2 * 32 and h.orl_linear_bwd_scratch(1000, 32, 64) == 2 * 125 * 32
    # few rows: a partial dx per strip of 64 rows of the weight or more
    assert h.orl_linear_bwd_scratch(3, 640, 512) == 10 * 3 * 512


def test_norm_rope_gradient_refuses(h):
    ok = [P] * 8 + [10, 2, 64, 1, 1e-6, 0, 64, P, None]
    call = lambda **at: h.orl_qk_norm_rope_bwd(*with_(ok, **at))
    assert all(call(**{f'a{i}': None}) == -1 for i in (*range(8), 15))
    assert call(a8=-1) == -1 and call(a9=0) == -1 and call(a10=60) == -1 and call(a13=2) == -1 and call(a14=32) == -1
    assert call(a9=200) == -3 and call(a10=96, a14=96) == -3 and call(a14=66) == -2 and call(a1=P + 4) == -2
    assert h.orl_qk_norm_rope_bwd_scratch(10, 2, 64, 1) == 10 * 64      # a partial row of the weight per block
    assert h.orl_qk_norm_rope_bwd_scratch(10, 200, 64, 1) == -1


def test_python_refuses_cpu_tensors():
    from onereel_b200.linear import linear
    from onereel_b200.rope import qk_norm_rope
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        linear(x, x)
    with pytest.raises(TypeError):
        qk_norm_rope(x, x[0], x, x, 1, 1e-6, True, 0)


def test_row_sum_refuses_and_plans(h):
    import ctypes

    import numpy as np

    from onereel_b200 import _lib as L
    from onereel_b200.pack import RowSum
    arr = L.c_vp * 2
    src, dst, odd = arr(P, P), arr(P, P), arr(P, P + 8)
    call = lambda s, d, planes, off, rows, n, rb: h.orl_row_sum(s, d, planes, off, rows, n, rb, None)
    assert call(src, dst, 4, P, P, 5, 64) == -1 and call(src, dst, 0, P, P, 5, 64) == -1
    assert call(src, dst, 2, None, P, 5, 64) == -1 and call(src, dst, 2, P, P, -1, 64) == -1
    assert call(src, dst, 2, P, P, 5, 0) == -1 and call(arr(P, None), dst, 2, P, P, 5, 64) == -1
    assert call(src, dst, 2, P, P, 5, 24) == -2 and call(src, odd, 2, P, P, 5, 64) == -2
    assert call(src, dst, 2, P, P, 0, 64) == 0
    s = RowSum([3, 0, 3, 1], [0, 1, 2, 3], 5, 'cpu')
    assert s.offsets.tolist() == [0, 1, 2, 2, 4, 4] and s.rows.tolist() == [1, 3, 0, 2] and s.n_packed == 4
    with pytest.raises(ValueError):
        RowSum([5], [0], 5, 'cpu')
    with pytest.raises(ValueError):
        RowSum([-1], [0], 5, 'cpu')
    with pytest.raises(ValueError):
        s.run([torch.zeros(3, 1, 8, dtype=torch.bfloat16)])


def test_plan_row_sums_cover_every_copy():
    """the copies that a scene plan's pack makes: every packed row is counted once, for its own source row"""
    import numpy as np

    from onereel_b200 import scene as S
    from onereel_b200.layout import SceneLayout
    lay = SceneLayout([3, 2, 4], halo=1, extra={0: [5], 2: [0]})
    T, counts = 5, [2, 0, 3]
    L = lay.n_frames * T
    scenes = [(j, (lo * T, hi * T)) for j, (lo, hi) in enumerate(lay.ranges)]
    segs = S.scene_segments(lay, T, counts, scenes, {0, 1, 2}, (0, L))
    plan = S.ScenePlan(segs, 64, 1, 'cpu')
    video, text = plan.row_sums(S.VIDEO, L), plan.row_sums(S.TEXT, sum(counts))
    packed = [(src, r) for s in segs for src, lo, hi in s.kv for r in range(lo, hi)]
    for rs, source, n in ((video, S.VIDEO, L), (text, S.TEXT, sum(counts))):
        off, rows = rs.offsets.tolist(), rs.rows.tolist()
        assert len(off) == n + 1
        for i in range(n):
            assert rows[off[i]:off[i + 1]] == [p for p, x in enumerate(packed) if x == (source, i)]
    assert len(video.rows) + len(text.rows) == plan.n_keys


def test_linear_gradients_without_the_product(h):
    """z may be left out where no gradient needs it: with a gate and no activation; not for the gate's own gradient"""
    ok = [P, 32, None, 64, P, 64, None, P, 0, P, P, None, P, None, P, 5, 32, 64, P, None]
    call = lambda **at: h.orl_linear_bwd(*with_(ok, **at))
    assert call(a13=P) == -1 and call(a8=1) == -1 and call(a9=None) == -1    # dgate, an activation, no room for dz
    assert call(a10=P + 8) == -2                                             # past those checks: dx misaligned


def test_linear_refuses_sizes_past_its_counters(h):
    """4 rows of 2^30 columns and rows up to the last strip's step would wrap 32-bit counters"""
    fwd = [P, 64, P, 64, P, P, P, 32, P, None, 5, 32, 64, 0, P, None]
    bwd = [P, 32, P, 64, P, 64, P, P, 1, P, P, P, P, P, P, 5, 32, 64, P, None]
    big = 2 ** 28 + 8
    assert h.orl_linear(*with_(fwd, a12=big, a1=big, a3=big)) == -1 and h.orl_linear(*with_(fwd, a11=big, a7=big)) == -1
    assert h.orl_linear(*with_(fwd, a10=0x7fff0001)) == -1
    assert h.orl_linear_bwd(*with_(bwd, a15=4, a17=big, a3=big, a5=big)) == -1
    assert h.orl_linear_bwd_scratch(4, 64, big) == -1 and h.orl_linear_bwd_scratch(0x7fff0001, 64, 64) == -1
    assert h.orl_linear_bwd_scratch(4, 64, 2 ** 28) == 4 * 2 ** 28      # one strip
