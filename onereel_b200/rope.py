"""q/k RMSNorm + rotary embedding on the fused CUDA kernel (orl_qk_norm_rope) — the q/k preparation of the
reference processors (src/onereel/models/hunyuan15.py:187-190: per-head RMSNorm then diffusers' apply_rotary_emb;
src/onereel/models/wan.py:64-74 `_qk`: hidden-dimension RMSNorm then Wan's interleaved RoPE, compiled by the reference
into a Triton kernel)."""
from __future__ import annotations

import torch

from onereel_b200 import _lib as L
from onereel_b200.attention import (_Device, _err_word, _first_order, _scratch_size, _stream, _wants_grad, overwrites,
                                    without_gradient)


def qk_norm_rope(x: torch.Tensor, weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, heads: int,
                 eps: float, per_head: bool, sin_shift: int, out: torch.Tensor | None = None,
                 row_map: torch.Tensor | None = None) -> torch.Tensor:
    """x [rows, heads * D] (or [1, rows, heads * D]) bf16 -> [rows, heads, D] bf16, normalised and rotated; cos / sin
    [rows, D] (any float dtype; converted to fp32 contiguous). out / row_map: write row i to out[row_map[i]].
    Differentiable in x and weight (first derivatives; the tables get none); with out or row_map a backward pass through
    the returned tensor raises."""
    if x.dim() == 3:
        if x.shape[0] != 1:
            raise ValueError(f'qk_norm_rope: x must be [rows, heads * D] or [1, rows, heads * D], got {tuple(x.shape)}')
        x = x[0]
    if not (x.is_cuda and x.dtype == torch.bfloat16):
        raise TypeError('qk_norm_rope: x must be a bf16 CUDA tensor (no fallback)')
    x = x.contiguous()
    rows = x.shape[0]
    w = weight.to(device=x.device, dtype=torch.bfloat16).contiguous()
    c, s = _table(cos, rows, x.device), _table(sin, rows, x.device)
    _check_shapes(x, w, c, s, heads, per_head)
    if out is not None and not (out.dtype == x.dtype and out.device == x.device and out.is_contiguous() and
                                (row_map is not None or out.numel() >= x.numel())):
        raise ValueError(f'qk_norm_rope: out must be contiguous, with {tuple(x.shape)} bf16 elements on {x.device}')
    if row_map is not None and row_map.numel() != rows:
        raise ValueError(f'qk_norm_rope: row_map must have {rows} entries, got {row_map.numel()}')
    if _wants_grad(x, w) and out is None and row_map is None:
        return _QkNormRope.apply(x, w, c, s, heads, float(eps), int(per_head), int(sin_shift))
    y = _forward(x, w, c, s, heads, eps, per_head, sin_shift, out, row_map)
    return y if out is None and row_map is None else without_gradient('qk_norm_rope with out or row_map', y, x, w)


def _check_shapes(x, w, c, s, heads: int, per_head):
    """that the kernels, which get addresses and the sizes of x, stay inside the weight and the tables"""
    hidden = x.shape[-1]
    if x.dim() != 2 or heads <= 0 or hidden % heads:
        raise ValueError(f'qk_norm_rope: x must have rows of {heads} equal heads, got {tuple(x.shape)}')
    dh = hidden // heads
    if w.numel() != (dh if per_head else hidden):
        raise ValueError(f'qk_norm_rope: weight must have {dh if per_head else hidden} elements, got {tuple(w.shape)}')
    if c.shape != s.shape or c.dim() != 2 or c.shape[0] != x.shape[0] or c.shape[1] < dh:
        raise ValueError(f'qk_norm_rope: cos and sin must be tables [{x.shape[0]}, {dh}], got {tuple(c.shape)} and '
                         f'{tuple(s.shape)}')


def _table(t, rows: int, device):
    """a rotary table as the kernels read it: fp32 [rows, D], contiguous"""
    if t.dtype is torch.float32 and t.device == device and t.dim() == 2 and t.shape[0] == rows and t.is_contiguous():
        return t
    t = t.to(device=device, dtype=torch.float32)
    return t.reshape(rows, -1 if rows else t.shape[-1]).contiguous()


def _forward(x, w, c, s, heads, eps, per_head, sin_shift, out=None, row_map=None):
    rows, Dh = x.shape[0], x.shape[1] // heads
    if out is None:
        out = torch.empty(rows, heads, Dh, dtype=torch.bfloat16, device=x.device)
    rm = None if row_map is None else row_map.to(device=x.device, dtype=torch.int32).contiguous()
    L.check(L.lib().orl_qk_norm_rope(x.data_ptr(), out.data_ptr(), w.data_ptr(), c.data_ptr(), s.data_ptr(), rows,
                                     heads, Dh, int(per_head), float(eps), int(sin_shift), c.shape[1],
                                     None if rm is None else rm.data_ptr(),
                                     _stream(x.device)), 'orl_qk_norm_rope')
    return out


class _QkNormRope(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w, c, s, heads, eps, per_head, sin_shift):
        ctx.save_for_backward(x, w, c, s)
        ctx.args = heads, eps, per_head, sin_shift
        with _Device(x.device):
            return _forward(x, w, c, s, heads, eps, per_head, sin_shift)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, w, c, s = ctx.saved_tensors
        dx, dw = _grad(x, w, c, s, dy, *ctx.args)
        return dx, dw, None, None, None, None, None, None


def qk_norm_rope_grad(x, weight, cos, sin, dy, heads: int, eps: float, per_head: bool, sin_shift: int):
    """(dx, dweight) of qk_norm_rope (orl_qk_norm_rope_bwd): x [rows, heads * D] and weight bf16, cos / sin fp32
    [rows, D], all contiguous as the forward used them; dy [rows, heads, D] bf16"""
    for name, t, dtype in (('x', x, torch.bfloat16), ('weight', weight, torch.bfloat16), ('cos', cos, torch.float32),
                           ('sin', sin, torch.float32)):
        if t.dtype != dtype or not t.is_cuda or t.device != x.device or not t.is_contiguous():
            raise TypeError(f'qk_norm_rope: {name} must be a contiguous {dtype} tensor on {x.device}')
    _check_shapes(x, weight, cos, sin, heads, per_head)
    rows, hidden = x.shape
    if dy.dtype != torch.bfloat16 or dy.device != x.device:
        raise TypeError(f'qk_norm_rope: dy must be bf16 on {x.device}')
    if dy.shape != (rows, heads, hidden // heads):
        raise ValueError(f'qk_norm_rope: dy must have shape {(rows, heads, hidden // heads)}, got {tuple(dy.shape)}')
    return _grad(x, weight, cos, sin, dy, heads, eps, per_head, sin_shift)


def _grad(x, weight, cos, sin, dy, heads, eps, per_head, sin_shift):
    rows, hidden = x.shape
    dy = dy.contiguous()
    dy = dy if dy.data_ptr() % 16 == 0 else dy.clone()
    with _Device(x.device):
        n = _scratch_size('orl_qk_norm_rope_bwd_scratch', rows, heads, hidden // heads, int(per_head))
        scratch = torch.empty(n, dtype=torch.float32, device=x.device)
        dx, dw = torch.empty_like(x), torch.empty_like(weight)
        L.check(L.lib().orl_qk_norm_rope_bwd(x.data_ptr(), dy.data_ptr(), weight.data_ptr(), cos.data_ptr(),
                                             sin.data_ptr(), dx.data_ptr(), dw.data_ptr(), scratch.data_ptr(), rows,
                                             heads, hidden // heads, int(per_head), float(eps), int(sin_shift),
                                             cos.shape[1], _err_word(x.device).data_ptr(), _stream(x.device)),
                'orl_qk_norm_rope_bwd')
    return dx, dw


def rotate_rows(x: torch.Tensor, rows: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, sin_shift: int = 0):
    """in place: rows `rows` (int32 CUDA tensor) of x [N, H, D] bf16 rotated by the table rows cos / sin
    [len(rows), D] fp32 (orl_rope_rows). A backward pass through the rotated values raises."""
    Nr = rows.numel()
    if Nr == 0:
        return x
    overwrites('rotate_rows', (x,))
    H, Dh = x.shape[1:]
    L.check(L.lib().orl_rope_rows(x.data_ptr(), rows.data_ptr(), Nr, H, Dh, cos.data_ptr(), sin.data_ptr(),
                                  cos.shape[1], int(sin_shift), _stream(x.device)),
            'orl_rope_rows')
    return x
