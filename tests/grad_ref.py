"""Float64 gradients of packed attention with elementwise error bounds, for the backward kernel's tests (CPU or GPU
tensors; not a product path).

The bounds count the kernel's roundings to bf16 (u = 2^-8 each, half a step) and give everything held in fp32 (tensor
core sums, exponentials, the log-sum-exp) a relative 2^-14. With the kernel's P~, o~ (bf16) and delta~ = sum dO o~ - dL:
  |dv~ - dv|   <= u |dv| + (u + f) sum_i P |dO|
  |delta~ - delta| <= (2 u + f) sum_d |dO| sum_j P |v|  =: e_i          (o~: P rounded, then o rounded)
  |dS~ - dS|   <= (u + f) |dS| + P (1 + u) (e_i + f sum_d |dO| |v| + f |dL|)  =: E
  |dq~ - dq|   <= u |dq| + scale sum_j E |k|,     |dk~ - dk| <= u |dk| + scale sum_i E |q|
(first order; a factor 1.1 covers the products of the small terms).
"""
import torch

U, F = 2.0 ** -8, 2.0 ** -14


def attention_grads(q, k, v, dout, q_start, q_len, k_start, k_len, dlse=None):
    """dict name -> (float64 value, elementwise bound) for out, dq, dk, dv; lse -> (value, None)"""
    H, D = q.shape[1:]
    scale = D ** -0.5
    Q, K, V, G = (x.detach().double().transpose(0, 1) for x in (q, k, v, dout))
    val = {n: torch.zeros_like(x) for n, x in (('out', Q), ('dq', Q), ('dk', K), ('dv', K))}
    bnd = {n: torch.zeros_like(x) for n, x in val.items()}
    lse = torch.full(Q.shape[:2], -float('inf'), dtype=torch.float64, device=q.device)
    for qs, ql, ks, kl in zip(q_start, q_len, k_start, k_len):
        if ql == 0 or kl == 0:
            continue
        a, b = slice(qs, qs + ql), slice(ks, ks + kl)
        for h in range(H):
            qq, kk, vv, gg = Q[h, a], K[h, b], V[h, b], G[h, a]
            dl = torch.zeros(ql, dtype=torch.float64, device=q.device) if dlse is None else dlse[h, a].double()
            s = qq @ kk.T * scale
            lse[h, a] = torch.logsumexp(s, -1)
            p = torch.softmax(s, -1)
            o = p @ vv
            dp = gg @ vv.T
            ds = p * (dp - (gg * o).sum(-1, keepdim=True) + dl[:, None])
            val['out'][h, a] = o
            bnd['out'][h, a] = (U + F) * (p @ vv.abs())
            val['dv'][h, b] += p.T @ gg
            bnd['dv'][h, b] += (U + F) * (p.T @ gg.abs())
            val['dq'][h, a] = scale * ds @ kk
            val['dk'][h, b] += scale * ds.T @ qq
            e = (2 * U + F) * (gg.abs() * (p @ vv.abs())).sum(-1, keepdim=True) + F * dl.abs()[:, None]
            err = (U + F) * ds.abs() + p * (1 + U) * (e + F * (gg.abs() @ vv.abs().T))
            bnd['dq'][h, a] = scale * err @ kk.abs()
            bnd['dk'][h, b] += scale * err.T @ qq.abs()
    res = {n: (val[n].transpose(0, 1), (1.1 * (bnd[n] + U * val[n].abs()) + 1e-30).transpose(0, 1)) for n in val}
    res['lse'] = (lse, None)
    return res


def assert_close(got, want, what):
    """elementwise inside the bound and, over the whole tensor, within two roundings (independent roundings of random
    data: at most four, each u / sqrt(3) of the result's norm)"""
    val, bound = want
    d = (got.double() - val).abs()
    worst = (d / bound).max().item() if d.numel() else 0.0
    assert worst <= 1.0, f'{what}: {worst:.2f} times its error bound'
    norm = val.norm().item()
    if norm > 0:
        rel = d.norm().item() / norm
        assert rel < 2 * U, f'{what}: relative error {rel:.2e}'
