"""Varlen attention on the B200 kernel (onereel_b200/csrc/attn_fwd.cu) — the drop-in for src/onereel/attention.py.

Same functions, arguments and return values as the reference module (attention.py:13-84): `cu_seqlens`, `dense`,
`varlen`, `varlen_lse`, `packed`, `packed_lse`, `overlapping_ranges`, and the module global `BACKEND`. The reference
selects FlashAttention-2/-3 by BACKEND; here every value runs the sm_100a kernel ('b200'; the reference's 'fa2', 'fa3'
and 'auto' are accepted so existing callers keep working). There is no CPU or library fallback: inputs must be bf16
CUDA tensors with head_dim 64 or 128.

Gradients: like the reference's FlashAttention calls, `varlen`, `varlen_lse`, `packed`, `packed_lse`,
`overlapping_ranges` and `dense` are differentiable in q, k and v (also through the log-sum-exp) when autograd is on
and an input requires a gradient; the backward pass (onereel_b200/csrc/attn_bwd.cu) recomputes the probabilities and is
deterministic. `attend_grad` is the same computation as a plain call. First derivatives in reverse mode only.

Kernel failures: the kernel never hangs; a bounded wait that gives up sets a per-device error word. `check()`
synchronises and raises if it is set (tests and benchmarks call it; it costs a device sync).
"""
from __future__ import annotations

import functools
import threading
from collections import OrderedDict

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from onereel_b200 import _lib as L
from onereel_b200.pack import capturing, pack_rows, upload

BACKEND = 'b200'         # 'b200' (also accepted: the reference's 'fa2' | 'fa3' | 'auto', all served by this kernel)
_BACKENDS = ('b200', 'fa2', 'fa3', 'auto')


def backend() -> str:
    if BACKEND not in _BACKENDS:
        raise ImportError(f'unknown attention backend {BACKEND!r}')
    return 'b200'


def cu_seqlens(lengths, device='cuda') -> torch.Tensor:
    """attention.py:28-29: int32 [0, cumsum(lengths)]"""
    return torch.tensor([0] + np.cumsum(lengths).tolist(), dtype=torch.int32, device=device)


# ------------------------------------------------------------------------------------------------ plans and errors

class _Plans:
    """Device tables by layout (layouts repeat every layer and step), shared by the calling and autograd's threads. Kernels
    read the tables by address, so an entry's memory outlives its readers: what a captured graph was given stays for good
    (a replay reads it again), and the others leave half the cache at a time, least recently used first, after their
    devices have been waited for (no kernel on any stream still reads them)."""

    def __init__(self, limit: int = 512):
        self.limit = limit
        self.entries: OrderedDict = OrderedDict()
        self.held: dict = {}                     # entries given to a captured graph
        self.lock = threading.Lock()

    def get(self, key, device, build):
        """the entry of key (on `device`), made by build() where there is none"""
        taken = capturing(device)
        with self.lock:
            hit = self.held.get(key)
            if hit is None:
                hit = self.entries.get(key)
                if hit is not None:
                    self.entries.move_to_end(key)
                    if taken:
                        self.held[key] = hit
            if hit is not None:
                return hit
        entry = build()                          # refused in a capture
        gone = []
        with self.lock:
            entry = self.entries.setdefault(key, entry)
            if len(self.entries) > self.limit:
                gone = [self.entries.popitem(last=False) for _ in range(len(self.entries) - self.limit // 2)]
        for dev in {t.device for _, e in gone for t in e if isinstance(t, torch.Tensor) and t.is_cuda}:
            torch.cuda.synchronize(dev)
        return entry


_PLANS = _Plans()
_ERR: dict = {}


def _err_word(device: torch.device) -> torch.Tensor:
    key = device.index if device.index is not None else torch.cuda.current_device()
    if key not in _ERR:
        _ERR[key] = torch.zeros(1, dtype=torch.int32, device=device)
    return _ERR[key]


def _stream(dev: torch.device) -> int:
    """the current stream of dev as the C ABI takes it (without building a torch.cuda.Stream: the small calls' host
    time is of the order of their kernels')"""
    return torch._C._cuda_getCurrentRawStream(dev.index)


class _Device:
    """`with _Device(dev)`: dev current, as torch.cuda.device, for free where it already is"""
    __slots__ = ('index', 'back')

    def __init__(self, dev: torch.device):
        self.index = dev.index

    def __enter__(self):
        self.back = torch._C._cuda_getDevice()
        if self.back != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.back != self.index:
            torch.cuda.set_device(self.back)


def _first_order(backward):
    """once_differentiable, whose own cost (it enters no_grad and looks every gradient over) is only paid where a second
    derivative could be asked for: without create_graph the backward pass runs with autograd off"""
    guarded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


@functools.lru_cache(maxsize=1024)
def _scratch_size(name: str, *sizes) -> int:
    """what the C ABI's size query `name` answers for these sizes"""
    return L.check(getattr(L.lib(), name)(*sizes), name)


def check(device=None) -> None:
    """synchronise and raise if a kernel on `device` (default: every device used) set a bit in its error word (a
    bounded wait that ran out, or cu_seqlens the device planner rejected)"""
    for key, w in list(_ERR.items()):
        if device is not None and torch.device(device).index not in (None, key):
            continue
        bits = int(w.item())
        if bits:
            w.zero_()
            raise L.OrlError(f'kernel on cuda:{key} reported: {L.describe_error_bits(bits)}')


def plan(q_start, q_len, k_start, k_len, heads: int, device) -> tuple[torch.Tensor, int, int, int]:
    """for segments given as (start, length) rows: device work list, its item count, and the rows of q and of k / v that the
    tensors must have for it (cached)"""
    key = (tuple(q_start), tuple(q_len), tuple(k_start), tuple(k_len), heads, str(device))
    return _PLANS.get(key, device, lambda: _make_plan(*key[:4], heads, device))


def _make_plan(q_start, q_len, k_start, k_len, heads, device):
    arrs = [np.ascontiguousarray(x, dtype=np.int32) for x in (q_start, q_len, k_start, k_len)]
    n_seg = len(arrs[0])
    need = L.lib().orl_attn_plan_ranges(*(L.i32p(a) for a in arrs), n_seg, heads, None, 0)
    if need >= 0:                                   # nothing to do
        need_n = 0
    else:
        L.check(need if need > -1000 else 0, 'orl_attn_plan_ranges')
        need_n = -need - 1000
    work = np.zeros(max(need_n, 1), dtype=L.WORK_DTYPE)
    n = L.check(L.lib().orl_attn_plan_ranges(*(L.i32p(a) for a in arrs), n_seg, heads, work.ctypes.data, len(work)),
                'orl_attn_plan_ranges')
    ends = lambda start, length: max((a + b for a, b, c in zip(start, length, q_len) if b > 0 and c > 0), default=0)
    return upload(work.view(np.uint8), device), n, ends(q_start, q_len), ends(k_start, k_len)


def _host_list(x) -> list[int]:
    return x.tolist() if isinstance(x, torch.Tensor) else [int(v) for v in x]


def _check_inputs(q, k, v):
    good = torch.bfloat16
    if (q.__class__ is k.__class__ is v.__class__ is torch.Tensor and q.dtype is k.dtype is v.dtype is good and
            q.is_cuda and q.dim() == 3 and q.is_contiguous() and k.is_contiguous() and v.is_contiguous() and
            k.device == v.device == q.device and k.shape == v.shape and k.dim() == 3 and
            q.shape[1:] == k.shape[1:] and q.shape[2] in (64, 128)):
        return
    for name, x in (('q', q), ('k', k), ('v', v)):
        if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype == torch.bfloat16):
            raise TypeError(f'{name} must be a bf16 CUDA tensor (the B200 path has no fallback), got '
                            f'{getattr(x, "dtype", type(x))} on {getattr(x, "device", "?")}')
        if x.dim() != 3 or x.stride(-1) != 1 or x.stride(1) != x.shape[2] or x.stride(0) != x.shape[1] * x.shape[2]:
            raise ValueError(f'{name} must be a contiguous [rows, heads, head_dim] tensor, got {tuple(x.shape)} '
                             f'strides {x.stride()}')
        if x.device != q.device:
            raise ValueError(f'{name} is on {x.device}, q on {q.device}')
    if q.shape[1:] != k.shape[1:] or k.shape != v.shape:
        raise ValueError(f'shape mismatch q {tuple(q.shape)} k {tuple(k.shape)} v {tuple(v.shape)}')
    if q.shape[2] not in (64, 128):
        raise ValueError(f'head_dim {q.shape[2]} not supported (64 or 128)')


# Key split of coarse launches (split_keys=True): a launch of fewer than SPLIT_WAVES waves of work items whose longest
# segment has at least SPLIT_MIN_KEYS keys runs as two launches over the two halves of every segment's keys, on two
# streams so the second fills the first's tail, merged by log-sum-exp. Exact attention, but another rounding than
# one pass: callers that promise bit-exact results across partitions (K/V gathering) never ask for it.
SPLIT_WAVES = 4
SPLIT_MIN_KEYS = 2048
LAUNCHES = 0          # attention launches issued by this process (benchmark launch accounting)
SPLITS = 0            # launches that took the key split
_SIDE = {}
_SMS = {}


def _sm_count(dev) -> int:
    key = dev.index if dev.index is not None else torch.cuda.current_device()
    if key not in _SMS:
        _SMS[key] = torch.cuda.get_device_properties(key).multi_processor_count
    return _SMS[key]


def _attend_split(q, k, v, q_start, q_len, k_start, k_len, out, lse, scale):
    """the two key halves (at a 128-key boundary) on the current and a side stream, then orl_lse_merge"""
    global SPLITS
    SPLITS += 1
    dev = q.device
    H, Nq = q.shape[1], q.shape[0]
    half = [128 * ((x + 255) // 256) if x >= 256 else x for x in k_len]
    cur = torch.cuda.current_stream(dev)
    key = dev.index if dev.index is not None else torch.cuda.current_device()
    side = _SIDE.get(key)
    if side is None:
        side = _SIDE[key] = torch.cuda.Stream(dev)
    out = torch.empty_like(q) if out is None else out
    lse_a = torch.empty(H, Nq, dtype=torch.float32, device=dev) if not isinstance(lse, torch.Tensor) else lse
    out_b = torch.empty_like(q)
    lse_b = torch.empty(H, Nq, dtype=torch.float32, device=dev)
    side.wait_stream(cur)
    attend(q, k, v, q_start, q_len, k_start, half, out=out, lse=lse_a, scale=scale)
    with torch.cuda.stream(side):
        attend(q, k, v, q_start, q_len, [a + h for a, h in zip(k_start, half)], [x - h for x, h in zip(k_len, half)],
               out=out_b, lse=lse_b, scale=scale, stream=side.cuda_stream)
    out_b.record_stream(side)
    lse_b.record_stream(side)
    cur.wait_stream(side)
    lse_merge(out, lse_a, out_b, lse_b)
    return out, (lse_a if lse is not None else None)


def attend(q, k, v, q_start, q_len, k_start, k_len, out=None, lse=None, scale=None, stream=None, split_keys=False):
    """the kernel call, without a backward pass: segment i = q rows q_start[i] + [0, q_len[i]) attending to k / v rows
    k_start[i] + [0, k_len[i]). out [Nq, H, D] bf16 (allocated if None); lse None, True (allocate [H, Nq] fp32) or a tensor.
    split_keys: allow the key split of coarse launches (see SPLIT_WAVES)."""
    _check_inputs(q, k, v)
    Nq, H, Dh = q.shape
    dev = q.device
    work, n, need_q, need_k = plan(q_start, q_len, k_start, k_len, H, dev)
    if need_q > Nq or need_k > k.shape[0]:
        raise ValueError(f'segments reach to row {need_q} of q and {need_k} of k / v, which have {Nq} and {k.shape[0]}')
    if (split_keys and stream is None and n and n < SPLIT_WAVES * _sm_count(dev) and
            max(k_len) >= SPLIT_MIN_KEYS):
        if lse is True:
            lse = torch.empty(H, Nq, dtype=torch.float32, device=dev)
        return _attend_split(q, k, v, q_start, q_len, k_start, k_len, out, lse, scale)
    if out is None:
        out = torch.empty_like(q)
    if lse is True:
        lse = torch.empty(H, Nq, dtype=torch.float32, device=dev)
    scale = Dh ** -0.5 if scale is None else float(scale)
    s = stream if stream is not None else _stream(dev)
    global LAUNCHES
    LAUNCHES += 1
    L.check(L.lib().orl_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                 None if lse is None else lse.data_ptr(), Nq, k.shape[0], H, Dh, scale,
                                 work.data_ptr(), n, _err_word(dev).data_ptr(), s), 'orl_attn_fwd')
    return out, lse


def attend_work(q, k, v, work, n_items: int, out, lse=None, scale=None, stream=None):
    """the kernel call, without a backward pass, with a caller-held device work list (orl_attn_plan_ranges items, possibly
    edited on the device since: the bounded memory sets each item's key count per head from its selection)"""
    _check_inputs(q, k, v)
    Nq, H, Dh = q.shape
    dev = q.device
    scale = Dh ** -0.5 if scale is None else float(scale)
    s = stream if stream is not None else torch.cuda.current_stream(dev).cuda_stream
    L.check(L.lib().orl_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                 None if lse is None else lse.data_ptr(), Nq, k.shape[0], H, Dh, scale,
                                 work.data_ptr(), n_items, _err_word(dev).data_ptr(), s), 'orl_attn_fwd')
    return out


def _cu_to_ranges(cu_q, cu_k):
    cq, ck = _host_list(cu_q), _host_list(cu_k)
    if len(cq) != len(ck):
        raise ValueError('cu_seqlens_q and cu_seqlens_k differ in length')
    qs, ks = cq[:-1], ck[:-1]
    ql = [b - a for a, b in zip(cq[:-1], cq[1:])]
    kl = [b - a for a, b in zip(ck[:-1], ck[1:])]
    if any(x < 0 for x in ql + kl):
        raise ValueError('cu_seqlens must be non-decreasing')
    return qs, ql, ks, kl


_CU_WORK = {}    # (device, stream) -> work-list scratch of orl_attn_fwd_cu (uint8), grown as needed


def _check_cu(q, cu_q, cu_k):
    for name, c in (('cu_seqlens_q', cu_q), ('cu_seqlens_k', cu_k)):
        if c.dtype != torch.int32 or c.dim() != 1 or c.device != q.device or not c.is_contiguous():
            raise TypeError(f'{name} must be a contiguous int32 tensor on {q.device}')
    if cu_q.numel() != cu_k.numel() or cu_q.numel() < 1:
        raise ValueError('cu_seqlens_q and cu_seqlens_k differ in length')


def _attend_cu(q, k, v, cu_q, cu_k, lse, own_scratch=False):
    """cu_seqlens on the device: orl_attn_fwd_cu plans the work list on the GPU, no host synchronisation. The
    scratch is per (device, stream), so calls on one stream reuse it in order; own_scratch, and any call that is being
    captured: scratch of this call alone (graphs may replay side by side, and after a larger call replaced the stream's
    scratch)."""
    _check_inputs(q, k, v)
    _check_cu(q, cu_q, cu_k)
    Nq, H, Dh = q.shape
    dev = q.device
    own_scratch = own_scratch or capturing(dev)
    n_seg = cu_q.numel() - 1
    need = _scratch_size('orl_attn_fwd_cu_capacity', Nq, n_seg, H)
    stream = _stream(dev)
    key = (dev.index, stream)
    work = None if own_scratch else _CU_WORK.get(key)
    if own_scratch:
        work = torch.empty(need * L.WORK_DTYPE.itemsize, dtype=torch.uint8, device=dev)
    elif work is None or work.numel() < need * L.WORK_DTYPE.itemsize:
        work = _CU_WORK[key] = torch.empty(need * L.WORK_DTYPE.itemsize, dtype=torch.uint8, device=dev)
    out = torch.empty_like(q)
    lse_t = torch.empty(H, Nq, dtype=torch.float32, device=dev) if lse else None
    L.check(L.lib().orl_attn_fwd_cu(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                    None if lse_t is None else lse_t.data_ptr(), Nq, k.shape[0], H, Dh, Dh ** -0.5,
                                    cu_q.data_ptr(), cu_k.data_ptr(), n_seg, work.data_ptr(),
                                    work.numel() // L.WORK_DTYPE.itemsize, _err_word(dev).data_ptr(),
                                    stream), 'orl_attn_fwd_cu')
    return out, lse_t


# ------------------------------------------------------------------------------------------------ gradients

_BWD_PLANS = _Plans()


def _plan_bwd(q_start, q_len, k_start, k_len, heads: int, nq: int, nk: int, device):
    """device work list and ranges of the backward pass for segments given as (start, length) rows (cached like
    `plan`): (items uint8 [32 n], ranges int32 [m, 2], n)"""
    key = (tuple(q_start), tuple(q_len), tuple(k_start), tuple(k_len), heads, nq, nk, str(device))
    return _BWD_PLANS.get(key, device, lambda: _make_bwd_plan(*key[:4], heads, nq, nk, device))


def _make_bwd_plan(q_start, q_len, k_start, k_len, heads, nq, nk, device):
    arrs = [np.ascontiguousarray(x, dtype=np.int32) for x in (q_start, q_len, k_start, k_len)]
    args = [L.i32p(a) for a in arrs] + [len(arrs[0]), heads, nq, nk]
    n_ranges = L.c_int(0)
    n = L.lib().orl_attn_bwd_plan(*args, None, 0, None, 0, n_ranges)
    if n <= -1000:
        work = np.zeros(-n - 1000, dtype=L.BWD_WORK_DTYPE)
        ranges = np.zeros((max(n_ranges.value, 1), 2), dtype=np.int32)
        n = L.lib().orl_attn_bwd_plan(*args, work.ctypes.data, len(work), ranges.ctypes.data, n_ranges.value, n_ranges)
    else:
        work, ranges = np.zeros(1, dtype=L.BWD_WORK_DTYPE), np.zeros((1, 2), dtype=np.int32)
    L.check(n, 'orl_attn_bwd_plan')
    return upload(work.view(np.uint8), device), upload(ranges, device), n


def _aligned(x):
    """x contiguous and 16-byte aligned (an incoming gradient may be any view)"""
    x = x if x.is_contiguous() else x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _check_grad_inputs(q, out, lse, dout, dlse):
    Nq, H, Dh = q.shape
    for name, x, shape, dtype in (('out', out, q.shape, torch.bfloat16), ('dout', dout, q.shape, torch.bfloat16),
                                  ('lse', lse, (H, Nq), torch.float32), ('dlse', dlse, (H, Nq), torch.float32)):
        if x is None and name == 'dlse':
            continue
        if not (isinstance(x, torch.Tensor) and x.device == q.device and x.dtype == dtype):
            raise TypeError(f'{name} must be a {dtype} tensor on {q.device}')
        if tuple(x.shape) != tuple(shape):
            raise ValueError(f'{name} must have shape {tuple(shape)}, got {tuple(x.shape)}')


def _bwd_args(q, k, v, out, lse, dout, dlse, extra: int = 0):
    """((dq, dk, dv), the C call's tensor arguments and sizes, addresses of the statistics scratch and of `extra` bytes
    more, what keeps them alive)"""
    out, dout, lse = _aligned(out), _aligned(dout), _aligned(lse)
    dlse = None if dlse is None else _aligned(dlse)
    Nq, H, Dh = q.shape
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    stats = (12 * H * Nq + 31) // 16 * 16
    scratch = torch.empty(stats + extra, dtype=torch.uint8, device=q.device)
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse.data_ptr(),
            None if dlse is None else dlse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), Nq, k.shape[0], H, Dh)
    at = scratch.data_ptr()
    return (dq, dk, dv), args, at, at + stats, (out, dout, lse, dlse, scratch)


def attend_grad(q, k, v, out, lse, dout, q_start, q_len, k_start, k_len, dlse=None, scale=None):
    """(dq, dk, dv) of `attend` on the same segments from its out and lse, the gradient dout of out and (optional) dlse
    of lse. Query ranges must not overlap; key ranges may, and a shared key row's gradient is the sum over its readers.
    Rows of no segment get zeros."""
    _check_inputs(q, k, v)
    _check_grad_inputs(q, out, lse, dout, dlse)
    return _attend_grad(q, k, v, out, lse, dout, q_start, q_len, k_start, k_len, dlse, scale)


def _attend_grad(q, k, v, out, lse, dout, q_start, q_len, k_start, k_len, dlse, scale=None):
    dev = q.device
    with _Device(dev):
        grads, args, stats, _, keep = _bwd_args(q, k, v, out, lse, dout, dlse)
        work, ranges, n = _plan_bwd(q_start, q_len, k_start, k_len, q.shape[1], q.shape[0], k.shape[0], dev)
        L.check(L.lib().orl_attn_bwd(*args, q.shape[2] ** -0.5 if scale is None else float(scale), work.data_ptr(), n,
                                     ranges.data_ptr(), stats, _err_word(dev).data_ptr(), _stream(dev)), 'orl_attn_bwd')
    return grads


def _attend_cu_grad(q, k, v, out, lse, dout, dlse, cu_q, cu_k):
    """attend_grad for cu_seqlens on the device, planned there (orl_attn_bwd_cu)"""
    dev, n_seg = q.device, cu_q.numel() - 1
    with _Device(dev):
        need = _scratch_size('orl_attn_bwd_cu_scratch', q.shape[0], k.shape[0], n_seg, q.shape[1])
        grads, args, stats, scratch, keep = _bwd_args(q, k, v, out, lse, dout, dlse, need)
        L.check(L.lib().orl_attn_bwd_cu(*args, q.shape[2] ** -0.5, cu_q.data_ptr(), cu_k.data_ptr(), n_seg, scratch,
                                        need, stats, _err_word(dev).data_ptr(), _stream(dev)), 'orl_attn_bwd_cu')
    return grads


class _Ranges(torch.autograd.Function):
    """attend on (start, length) segments, differentiable in q, k, v"""

    @staticmethod
    def forward(ctx, q, k, v, segments):
        with _Device(q.device):
            out, lse = attend(q, k, v, *segments, lse=True)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.segments = segments
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @_first_order
    def backward(ctx, dout, dlse):
        if dout is None and dlse is None:
            return None, None, None, None
        q, k, v, out, lse = ctx.saved_tensors
        dout = torch.zeros_like(out) if dout is None else dout
        return *_attend_grad(q, k, v, out, lse, dout, *ctx.segments, dlse), None


class _Varlen(torch.autograd.Function):
    """attention on device cu_seqlens, differentiable in q, k, v; neither pass synchronises with the host"""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k):
        with _Device(q.device):
            out, lse = _attend_cu(q, k, v, cu_q, cu_k, lse=True, own_scratch=True)
        ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @_first_order
    def backward(ctx, dout, dlse):
        if dout is None and dlse is None:
            return None, None, None, None, None
        q, k, v, out, lse, cu_q, cu_k = ctx.saved_tensors
        dout = torch.zeros_like(out) if dout is None else dout
        return *_attend_cu_grad(q, k, v, out, lse, dout, dlse, cu_q, cu_k), None, None


class _PackRows(torch.autograd.Function):
    """row tensors packed back to back (pack_rows); every part's gradient is its rows of the packed gradient"""

    @staticmethod
    def forward(ctx, *parts):
        ctx.lengths = [p.shape[0] for p in parts]
        return pack_rows(parts, parts[0].new_empty(sum(ctx.lengths), *parts[0].shape[1:]))

    @staticmethod
    @_first_order
    def backward(ctx, g):
        return g.split(ctx.lengths)


def _wants_grad(*tensors) -> bool:
    """whether a call on these tensors (None: not there) has to record a backward pass; refuses tangents of forward-mode
    differentiation, which a kernel that writes into a fresh tensor would drop"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise NotImplementedError('the B200 kernels have no forward-mode derivative (reverse mode only)')
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


class _NoGradient(torch.autograd.Function):
    """a value computed outside autograd, handed on; a backward pass that reaches it raises instead of leaving its share out"""

    @staticmethod
    def forward(ctx, what, value, *inputs):
        ctx.what = what
        return value

    @staticmethod
    def backward(ctx, g):
        raise NotImplementedError(f'{ctx.what} carries no gradients on the B200 path')


def without_gradient(what: str, values, *inputs):
    """values (a tensor, or a tuple of tensors and None) that a path without a backward pass computed from inputs: as they
    are, except that a backward pass through them raises where an input asks for a gradient"""
    if not _wants_grad(*inputs):
        return values
    inputs = [x for x in inputs if x is not None]
    tie = lambda v: v if v is None or v.requires_grad else _NoGradient.apply(what, v, *inputs)
    return tuple(tie(v) for v in values) if isinstance(values, tuple) else tie(values)


class _Overwritten(torch.autograd.Function):
    """a tensor that a kernel overwrites: what its old values were saved for refuses them, and a backward pass through the new
    ones raises"""

    @staticmethod
    def forward(ctx, what, target, *inputs):
        ctx.what = what
        ctx.mark_dirty(target)
        return target

    @staticmethod
    def backward(ctx, g):
        raise NotImplementedError(f'{ctx.what} carries no gradients on the B200 path')


def overwrites(what: str, targets, *inputs):
    """to be called before a kernel overwrites `targets` from inputs: autograd learns of it as of any in-place operation (and
    refuses the same: leaves, outputs of split)"""
    if _wants_grad(*targets, *inputs):
        for t in targets:                        # each tied to all that the kernel reads, one output per node (views need it)
            _Overwritten.apply(what, t, *(x for x in (*targets, *inputs) if x is not t))


def no_gradients(what: str):
    """decorator of a method on tensors whose results go through without_gradient (those that carry a graph already pass)"""
    def wrap(method):
        @functools.wraps(method)
        def run(self, *tensors, **named):
            return without_gradient(what, method(self, *tensors, **named), *tensors, *named.values())
        return run
    return wrap


def _attend_ranges(q, k, v, q_start, q_len, k_start, k_len, lse=False):
    """(out, lse or None) of host-planned segments, differentiable where an input asks for it"""
    if _wants_grad(q, k, v):
        _check_inputs(q, k, v)
        return _Ranges.apply(q, k, v, (q_start, q_len, k_start, k_len))
    return attend(q, k, v, q_start, q_len, k_start, k_len, lse=True if lse else None)


def varlen(q, k, v, cu_q, cu_k, max_q, max_k):
    """attention.py:39-43: packed q [Nq, H, D], k / v [Nk, H, D] -> out [Nq, H, D]. cu_seqlens as device int32
    tensors (as the reference passes them) are planned on the GPU without a host sync; host lists are planned on
    the host."""
    if isinstance(cu_q, torch.Tensor) and cu_q.is_cuda:
        if _wants_grad(q, k, v):
            return _Varlen.apply(q, k, v, cu_q, cu_k)[0]
        return _attend_cu(q, k, v, cu_q, cu_k, lse=False)[0]
    return _attend_ranges(q, k, v, *_cu_to_ranges(cu_q, cu_k))[0]


def varlen_lse(q, k, v, cu_q, cu_k, max_q, max_k):
    """attention.py:46-53: (out [Nq, H, D], lse [H, Nq] fp32, natural log)"""
    if isinstance(cu_q, torch.Tensor) and cu_q.is_cuda:
        if _wants_grad(q, k, v):
            return _Varlen.apply(q, k, v, cu_q, cu_k)
        return _attend_cu(q, k, v, cu_q, cu_k, lse=True)
    return _attend_ranges(q, k, v, *_cu_to_ranges(cu_q, cu_k), lse=True)


def _pack_segments(segments):
    lq = [s[0].shape[0] for s in segments]
    lk = [s[1].shape[0] for s in segments]
    q0 = segments[0][0]
    H, Dh = q0.shape[1:]
    c = lambda x: x if x.is_contiguous() else x.contiguous()
    if _wants_grad(*(x for s in segments for x in s)):
        qp, kp, vp = (_PackRows.apply(*(c(s[i]) for s in segments)) for i in range(3))
    else:
        qp = q0.new_empty(sum(lq), H, Dh)
        kp = q0.new_empty(sum(lk), H, Dh)
        vp = q0.new_empty(sum(lk), H, Dh)
        pack_rows([c(s[0]) for s in segments], qp)
        pack_rows([c(s[1]) for s in segments], kp)
        pack_rows([c(s[2]) for s in segments], vp)
    cq, ck = np.cumsum([0] + lq), np.cumsum([0] + lk)
    return qp, kp, vp, lq, list(cq[:-1]), lk, list(ck[:-1])


def packed_lse(segments):
    """attention.py:56-62: list of (out, lse [H, n]) per segment, one kernel call"""
    qp, kp, vp, lq, qs, lk, ks = _pack_segments(segments)
    o, lse = _attend_ranges(qp, kp, vp, qs, lq, ks, lk, lse=True)
    return list(zip(o.split(lq), lse.split(lq, dim=1)))


def packed(segments):
    """attention.py:65-71: segments = list of (q, k, v) -> list of outputs, one gather/pack launch per tensor and one
    attention launch"""
    qp, kp, vp, lq, qs, lk, ks = _pack_segments(segments)
    return _attend_ranges(qp, kp, vp, qs, lq, ks, lk)[0].split(lq)


def overlapping_ranges(q, k, v, q_ranges, k_ranges):
    """attention.py:74-84: q rows q_ranges[j] attend to k / v rows k_ranges[j], read in place (no copy); q_ranges
    tile q in order"""
    qs = [a for a, _ in q_ranges]
    ql = [b - a for a, b in q_ranges]
    if qs and (qs[0] != 0 or any(qs[i] + ql[i] != qs[i + 1] for i in range(len(qs) - 1)) or qs[-1] + ql[-1] != q.shape[0]):
        raise ValueError('q_ranges must tile q in order')
    return _attend_ranges(q, k, v, qs, ql, [a for a, _ in k_ranges], [b - a for a, b in k_ranges])[0]


def dense(q, k, v):
    """attention.py:32-36: q, k, v [B, S, H, D] -> [B, S, H, D], full attention per batch entry"""
    B, S, H, Dh = q.shape
    Sk = k.shape[1]
    c = lambda x: x.reshape(B * x.shape[1], H, Dh).contiguous()
    o = _attend_ranges(c(q), c(k), c(v), [b * S for b in range(B)], [S] * B, [b * Sk for b in range(B)], [Sk] * B)[0]
    return o.view(B, S, H, Dh)


def lse_merge(o1, lse1, o2, lse2):
    """in place: (o1, lse1) <- the merge of two partial results over disjoint keys (hunyuan15.py:274-276,
    ring.py:63-70). o [n, H, D] bf16 contiguous, lse [H, >= n] fp32 (row stride = its second dimension). A backward pass
    through the merged values raises."""
    overwrites('the log-sum-exp merge', (o1, lse1), o2, lse2)
    n, H, Dh = o1.shape
    s = torch.cuda.current_stream(o1.device).cuda_stream
    L.check(L.lib().orl_lse_merge(o1.data_ptr(), lse1.data_ptr(), o2.data_ptr(), lse2.data_ptr(), n, lse1.stride(0),
                                  lse2.stride(0), H, Dh, s), 'orl_lse_merge')
    return o1, lse1


def lse_merge_acc(acc, lse_acc, part, lse_part):
    """in place: fp32 (acc, lse_acc) <- merged with a bf16 partial result (part, lse_part) over disjoint keys
    (ring.py:63-70). acc [n, H, D] fp32 / part [n, H, D] bf16 contiguous rows, lse [H, >= n] fp32. A backward pass
    through the merged values raises."""
    overwrites('the log-sum-exp merge', (acc, lse_acc), part, lse_part)
    n, H, Dh = acc.shape
    s = torch.cuda.current_stream(acc.device).cuda_stream
    L.check(L.lib().orl_lse_merge_acc(acc.data_ptr(), lse_acc.data_ptr(), part.data_ptr(), lse_part.data_ptr(), n,
                                      lse_acc.stride(0), lse_part.stride(0), H, Dh, s), 'orl_lse_merge_acc')
    return acc, lse_acc
