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
    assert h.orl_linear_bwd_scratch(-1, 8) == -1 and h.orl_linear_bwd_scratch(5, 12) == -1
    # one partial row per strip of eight rows or more, for each of the two sums
    assert h.orl_linear_bwd_scratch(5, 32) == 2 * 32 and h.orl_linear_bwd_scratch(1000, 32) == 2 * 125 * 32


def test_norm_rope_gradient_refuses(h):
    ok = [P] * 8 + [10, 2, 64, 1, 1e-6, 0, 64, None]
    call = lambda **at: h.orl_qk_norm_rope_bwd(*with_(ok, **at))
    assert all(call(**{f'a{i}': None}) == -1 for i in range(8))
    assert call(a8=-1) == -1 and call(a9=0) == -1 and call(a10=60) == -1 and call(a13=2) == -1 and call(a14=32) == -1
    assert call(a9=200) == -3 and call(a10=96, a14=96) == -3 and call(a14=66) == -2 and call(a1=P + 4) == -2
    assert h.orl_qk_norm_rope_bwd_scratch(10, 2, 64, 1) == 2 * 64       # 8 rows of 32 threads share a block
    assert h.orl_qk_norm_rope_bwd_scratch(10, 200, 64, 1) == -1


def test_python_refuses_cpu_tensors():
    from onereel_b200.linear import linear
    from onereel_b200.rope import qk_norm_rope
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        linear(x, x)
    with pytest.raises(TypeError):
        qk_norm_rope(x, x[0], x, x, 1, 1e-6, True, 0)
