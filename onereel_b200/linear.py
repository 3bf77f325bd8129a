"""Linear layers with their epilogue on the B200 matrix kernels (onereel_b200/csrc/linear.cu): the projections and
feed-forward layers around the scene attention, with bias, activation, gate and residual in the kernel that computes the
product, and their gradients.

There is no CPU or library fallback: bf16 CUDA tensors, feature sizes that are multiples of 8. A wait of a kernel that
gave up is reported by onereel_b200.attention.check().
"""
from __future__ import annotations

import torch

from onereel_b200 import _lib as L
from onereel_b200.attention import _Device, _err_word, _first_order, _scratch_size, _stream, _wants_grad

ACTIVATIONS = {None: 0, 'gelu_tanh': 1, 'silu': 2}


def _check(name, t, shape, device):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.bfloat16):
        raise TypeError(f'{name} must be a bf16 CUDA tensor (the B200 path has no fallback), got '
                        f'{getattr(t, "dtype", type(t))} on {getattr(t, "device", "?")}')
    if t.device != device:
        raise ValueError(f'{name} is on {t.device}, x on {device}')
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name} must have shape {tuple(shape)}, got {tuple(t.shape)}')


def _rows(t):
    """t as the kernels read it: unit column stride, row stride a multiple of 8 and at least the row, 16-byte base (a
    copy where a view does not have them)"""
    ok = t.stride(1) == 1 and t.data_ptr() % 16 == 0 and \
        (t.shape[0] <= 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1]))
    return t if ok else t.contiguous().clone() if t.is_contiguous() else t.contiguous()


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _vector(t):
    t = t.reshape(-1)
    return t if t.stride(0) == 1 and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _ptr(t):
    return None if t is None else t.data_ptr()


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
           residual: torch.Tensor | None = None, gate: torch.Tensor | None = None) -> torch.Tensor:
    """residual + gate * activation(x weight^T + bias), accumulated and finished in fp32, rounded once.

    x [..., K], weight [N, K], bias [N], gate of N elements (one factor per output feature, e.g. [1, 1, N]), residual
    and the result [..., N]; activation None, 'gelu_tanh' or 'silu'; bf16 CUDA tensors, K and N multiples of 8. Views
    whose rows are strided by multiples of 8 elements are read in place, others are copied. Differentiable in every
    tensor (first derivatives in reverse mode; deterministic). Kept for the backward pass is what the wanted gradients need:
    x for the weight's, the weight for x's, and the product x weight^T + bias (m x n) for the gate's and, under an
    activation, for all but the residual's."""
    if activation not in ACTIVATIONS:
        raise ValueError(f'unknown activation {activation!r}: one of {sorted(map(str, ACTIVATIONS))}')
    _check('x', x, None, getattr(x, 'device', None))
    dev = x.device
    _check('weight', weight, None, dev)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f'shape mismatch x {tuple(x.shape)} weight {tuple(weight.shape)}')
    N, K = weight.shape
    if N % 8 or K % 8 or N == 0 or K == 0:
        raise ValueError(f'feature sizes must be positive multiples of 8, got {K} -> {N}')
    shape = (*x.shape[:-1], N)
    if bias is not None:
        _check('bias', bias, (N,), dev)
    if residual is not None:
        _check('residual', residual, shape, dev)
    if gate is not None:
        _check('gate', gate, None, dev)
        if gate.numel() != N:
            raise ValueError(f'gate must have {N} elements, got {tuple(gate.shape)}')
    # reshaped only where need be: with gradients each view is one more node of the graph
    flat = x.dim() == 2
    args = (x if flat else x.reshape(-1, K), weight, bias,
            gate if gate is None or gate.dim() == 1 else gate.reshape(-1),
            residual if residual is None or flat else residual.reshape(-1, N))
    act = ACTIVATIONS[activation]
    if _wants_grad(*args):
        y = _Linear.apply(*args, act)
    else:
        y = _forward(*args, act, keep=False)[0]
    return y if flat else y.view(shape)


def _forward(x, w, b, gate, residual, act, keep):
    """(y, z or None): the kernel call; keep: also store z = x w^T + bias"""
    M, N, K, dev = x.shape[0], w.shape[0], x.shape[1], x.device
    with _Device(dev):
        x, w = _rows(x), _rows(w)
        b, gate = (None if t is None else _vector(t) for t in (b, gate))
        residual = None if residual is None else _rows(residual)
        y = torch.empty(M, N, dtype=torch.bfloat16, device=dev)
        z = torch.empty_like(y) if keep else None
        L.check(L.lib().orl_linear(x.data_ptr(), _ld(x), w.data_ptr(), _ld(w), _ptr(b), _ptr(gate), _ptr(residual),
                                   0 if residual is None else _ld(residual), y.data_ptr(), _ptr(z), M, N, K, act,
                                   _err_word(dev).data_ptr(), _stream(dev)),
                'orl_linear')
    return y, z


class _Linear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w, b, gate, residual, act):
        # Kept is what the wanted gradients are made of: z for act' and for the gate's gradient (without either, dz is dy or
        # gate dy), x for dw, w for dx.
        need_x, need_w, need_b, need_gate, _, _ = ctx.needs_input_grad
        slope = need_x or need_w or need_b
        y, z = _forward(x, w, b, gate, residual, act, keep=need_gate or (slope and act != 0))
        ctx.save_for_backward(x if need_w else None, w if need_x else None, gate if slope else None, z)
        ctx.act, ctx.sizes = act if z is not None else 0, (x.shape[0], *w.shape)
        return y

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, w, gate, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        if not any(need[:4]):
            return None, None, None, None, dy, None
        (M, N, K), dev = ctx.sizes, dy.device
        with _Device(dev):
            d, xr, wr = _rows(dy), x if x is None else _rows(x), w if w is None else _rows(w)
            new = lambda *shape: torch.empty(*shape, dtype=torch.bfloat16, device=dev)
            dx = new(M, K) if need[0] else None
            dw = new(N, K) if need[1] else None
            db = new(N) if need[2] else None
            dgate = new(N) if need[3] else None
            # scratch: partial sums, then dz where it is not dy itself
            own_dz = z is not None or gate is not None
            sums = 4 * _scratch_size('orl_linear_bwd_scratch', M, N, K)
            scratch = torch.empty(sums + (2 * M * N if own_dz else 0), dtype=torch.uint8, device=dev)
            at = scratch.data_ptr()
            L.check(L.lib().orl_linear_bwd(d.data_ptr(), _ld(d), _ptr(xr), K if x is None else _ld(xr), _ptr(wr),
                                           K if w is None else _ld(wr), _ptr(z),
                                           None if gate is None else _vector(gate).data_ptr(), ctx.act,
                                           at + sums if own_dz else None, _ptr(dx), _ptr(dw), _ptr(db), _ptr(dgate),
                                           at, M, N, K, _err_word(dev).data_ptr(), _stream(dev)), 'orl_linear_bwd')
        return dx, dw, db, dgate, dy if need[4] else None, None
