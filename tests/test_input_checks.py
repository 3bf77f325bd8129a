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
