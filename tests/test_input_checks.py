"""What the entry points refuse before they hand an address to a kernel (no GPU: tensors without storage stand for CUDA ones)."""
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
