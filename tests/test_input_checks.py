"""What the entry points refuse before they hand an address to a kernel (no GPU: tensors without storage stand for CUDA
ones)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def fake():
    from onereel_b200.csrc.build import build
    build()
    with FakeTensorMode(allow_non_fake_inputs=True):
        yield


def cuda(*shape, dtype=BF16, index=0):
    return torch.empty(*shape, dtype=dtype, device=f'cuda:{index}')


def test_attention_refuses_tensors_of_two_devices():
    from onereel_b200 import attention as A
    q, k, v = cuda(5, 2, 64), cuda(7, 2, 64), cuda(7, 2, 64)
    A._check_inputs(q, k, v)
    for bad in ((cuda(5, 2, 64, index=1), k, v), (q, cuda(7, 2, 64, index=1), v), (q, k, cuda(7, 2, 64, index=1))):
        with pytest.raises(ValueError, match='cuda:1'):
            A._check_inputs(*bad)
        with pytest.raises(ValueError, match='cuda:1'):
            A.varlen(*bad, [0, 5], [0, 7], 5, 7)


def test_norm_rope_refuses_shapes_that_do_not_fit():
    """a weight, tables or an output of other sizes than x's, a batch, half a head: refused by the call and its gradient"""
    from onereel_b200.rope import qk_norm_rope, qk_norm_rope_grad
    f32 = torch.float32
    x, w, c = cuda(6, 128), cuda(64), cuda(6, 64, dtype=f32)
    args = lambda **kw: {**dict(x=x, weight=w, cos=c, sin=c, heads=2, eps=1e-6, per_head=True, sin_shift=0), **kw}
    bad = [dict(weight=cuda(128)), dict(per_head=False), dict(heads=3), dict(cos=cuda(5, 64, dtype=f32)),
           dict(sin=cuda(6, 32, dtype=f32)), dict(cos=cuda(6, 32, dtype=f32), sin=cuda(6, 32, dtype=f32))]
    for kw in bad:
        with pytest.raises((ValueError, RuntimeError)):
            qk_norm_rope(**args(**kw))
        with pytest.raises(ValueError):
            qk_norm_rope_grad(**args(**kw), dy=cuda(6, 2, 64))
    for kw in (dict(x=cuda(2, 6, 128)), dict(out=cuda(5, 2, 64)), dict(out=cuda(6, 2, 64, dtype=f32)),
               dict(out=cuda(6, 64, 2).transpose(1, 2)), dict(row_map=cuda(5, dtype=torch.int32))):
        with pytest.raises(ValueError):
            qk_norm_rope(**args(**kw))
    for kw in (dict(x=cuda(6, 256)[:, :128]), dict(weight=cuda(64, dtype=f32)), dict(cos=cuda(6, 64)),
               dict(sin=cuda(6, 64, dtype=f32, index=1))):
        with pytest.raises(TypeError):
            qk_norm_rope_grad(**args(**kw), dy=cuda(6, 2, 64))


def test_scene_plan_refuses_tensors_that_do_not_fit():
    """fewer rows than the plan reads, strided or missing tensors, other heads; parts of a pack's gradient that differ"""
    from onereel_b200 import scene as S
    from onereel_b200.layout import SceneLayout
    from onereel_b200.pack import RowSum
    lay, T, counts, H = SceneLayout([2, 3], halo=1), 8, [3, 4], 2
    L, E = lay.n_frames * T, sum(counts)
    scenes = [(j, (lo * T, hi * T)) for j, (lo, hi) in enumerate(lay.ranges)]
    plan = S.ScenePlan(S.scene_segments(lay, T, counts, scenes, {0, 1}, (0, L)), H * 128, H, 'cpu')
    assert plan.rows_needed(S.VIDEO) == L and plan.rows_needed(S.TEXT) == E and plan.rows_needed(S.REMOTE) == 0
    good = [cuda(n, H, 64) for n in (L, L, L, E, E, E)]
    for i, t in ((0, cuda(L - 1, H, 64)), (1, cuda(L - 1, H, 64)), (2, cuda(L, 64, H).transpose(1, 2)), (3, cuda(E - 1, H, 64)),
                 (4, cuda(E, H, 128)), (3, None), (5, None)):
        with pytest.raises(ValueError):
            S.attend_plan(plan, *(t if i == j else x for j, x in enumerate(good)))
    with pytest.raises(ValueError):
        S.attend_plan(plan, *(cuda(x.shape[0] - 1, H, 64) if i in (1, 2) else x for i, x in enumerate(good)))
    with pytest.raises(ValueError):
        S.attend_plan(plan, *good[:3])
    with pytest.raises(ValueError):
        S.attend_plan(plan, *(cuda(x.shape[0], 2 * H, 64) for x in good))
    with pytest.raises(TypeError):
        S.attend_plan(plan, *(x.float() for x in good))


def test_row_sum_refuses_parts_that_differ():
    from onereel_b200.pack import RowSum
    with torch._subclasses.fake_tensor.unset_fake_temporarily():
        s = RowSum([0, 1, 1], [0, 1, 2], 2, 'cpu')
        part = lambda *shape, dtype=BF16: torch.zeros(*shape, dtype=dtype)
        for parts in ([part(3, 1, 16), part(3, 1, 8)], [part(3, 1, 8), part(2, 1, 8)],
                      [part(3, 1, 8), part(3, 1, 8, dtype=torch.half)]):
            with pytest.raises(ValueError, match='alike'):
                s.run(parts)
