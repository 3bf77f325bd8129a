"""Cases and plain forms of the operators that make the scene-attention layer trainable and of its fused linear layers.

attention   packed attention over segments with its gradients (onereel_b200.attention)
linear      y = residual + gate * act(x w^T + bias), with its gradients in training (onereel_b200.linear)
norm_rope   q/k RMSNorm + rotary embedding with its gradients (onereel_b200.rope)

`run` with own = False computes them with elementary torch operations in 32 bits; with own = True it makes the calls a
program makes of the framework. `exact` is the definition in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-6
SQRT_2_OVER_PI = math.sqrt(2.0 / math.pi)


def listed():
    return [
        # one short sentence reading two small frames: launch latency of a forward and a backward
        dict(name='attention-small', op='attention', via='varlen', heads=4, dim=64, q='5 64', k='7 200', lse=False),
        # sentences and scenes of a short clip, ragged lengths, with the log-sum-exp a merge of partial results needs
        dict(name='attention-ragged-lse', op='attention', via='varlen', heads=16, dim=128, q='16 256 600 1000 1',
             k='336 336 77 513 4096', lse=True),
        # a batch of equal sequences with 64-wide heads
        dict(name='attention-batch-64', op='attention', via='varlen', heads=16, dim=64, q='2048 2048 2048',
             k='2048 2048 2048', lse=False),
        # scenes of [3, 5, 4] frames of 880 tokens, keys read in place with one halo frame on each side: shared keys
        dict(name='attention-ranges', op='attention', via='ranges', heads=12, dim=128, q='2640 4400 3520',
             k='0-3520 1760-7920 6160-10560', lse=False),
        # two scenes of 8 and 6 frames of 1590 tokens with frame memory and 128 text tokens: a layer's training pass
        dict(name='attention-scenes', op='attention', via='varlen', heads=16, dim=128, q='12720 9540 128 128',
             k='14438 11258 12848 9668', lse=False),
        # the modulation vector of a block: one row through a 2048 -> 12 x 2048 layer
        dict(name='linear-one-row', op='linear', m=1, k=2048, n=24576, bias=True, act='', residual=False, gate=False,
             train=False),
        # text tokens of one scene through the first feed-forward layer
        dict(name='linear-text', op='linear', m=77, k=2048, n=8192, bias=True, act='gelu_tanh', residual=False,
             gate=False, train=False),
        # the second feed-forward layer of all video rows with its gated residual, in sampling
        dict(name='linear-down', op='linear', m=22260, k=8192, n=2048, bias=True, act='', residual=True, gate=True,
             train=False),
        # the first feed-forward layer of one scene, training
        dict(name='linear-up-train', op='linear', m=9540, k=2048, n=8192, bias=True, act='gelu_tanh', residual=False,
             gate=False, train=True),
        # an output projection with its gated residual on a ragged number of rows, training
        dict(name='linear-out-train', op='linear', m=1001, k=2048, n=2048, bias=True, act='', residual=True, gate=True,
             train=True),
        # q or k of the text rows, per-head norm
        dict(name='norm-rope-small', op='norm_rope', rows=77, heads=16, dim=128, per_head=True),
        # q or k of two scenes' video rows, norm over the whole row
        dict(name='norm-rope-large', op='norm_rope', rows=22260, heads=16, dim=128, per_head=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['attention', 'attention', 'linear', 'linear', 'norm_rope'])
    if op == 'attention':
        heads, dim = rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([64, 128])
        n = rng.randint(1, 6)
        # two keys at least: with one key a row's gradients of q and k are zero but for rounding
        lens = [(_log_int(rng, 1, 12000), _log_int(rng, 2, 14000)) for _ in range(n)]
        while heads > 1 and heads * dim * sum(a * (b + 1400) for a, b in lens) > 5e11:
            heads -= 1
        if rng.random() < 0.3:
            # scenes in order, each reading its own rows and up to 700 of its neighbours'
            starts = [sum(a for a, _ in lens[:i]) for i in range(n + 1)]
            ks = [(max(0, starts[i] - rng.randint(1, 700)), min(starts[n] + 1, starts[i + 1] + rng.randint(1, 700)))
                  for i in range(n)]
            return dict(op=op, via='ranges', heads=heads, dim=dim, q=' '.join(str(a) for a, _ in lens),
                        k=' '.join('%d-%d' % r for r in ks), lse=False)
        return dict(op=op, via='varlen', heads=heads, dim=dim, q=' '.join(str(a) for a, _ in lens),
                    k=' '.join(str(b) for _, b in lens), lse=rng.random() < 0.3)
    if op == 'linear':
        m = _log_int(rng, 1, 16000)
        residual = rng.random() < 0.5
        return dict(op=op, m=m, k=8 * _log_int(rng, 8, 1024), n=8 * _log_int(rng, 8, 1024), bias=rng.random() < 0.8,
                    act=rng.choice(['', 'gelu_tanh', 'silu']), residual=residual, gate=residual and rng.random() < 0.5,
                    train=rng.random() < 0.5)
    return dict(op=op, rows=_log_int(rng, 1, 22000), heads=rng.choice([1, 2, 5, 8, 12, 16]),
                dim=rng.choice([64, 128]), per_head=rng.random() < 0.5)


def _segments(case):
    """[(first query row, query rows, first key row, key rows)], rows of q, rows of k"""
    ql = [int(x) for x in case['q'].split()]
    qs = [sum(ql[:i]) for i in range(len(ql))]
    if case['via'] == 'ranges':
        ks = [tuple(int(x) for x in r.split('-')) for r in case['k'].split()]
        return [(a, n, lo, hi - lo) for a, n, (lo, hi) in zip(qs, ql, ks)], sum(ql), max(hi for _, hi in ks)
    kl = [int(x) for x in case['k'].split()]
    return [(a, n, sum(kl[:i]), kl[i]) for i, (a, n) in enumerate(zip(qs, ql))], sum(ql), sum(kl)


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def randn(*shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device='cuda').mul_(std).add_(mean).to(dtype)

    s = {'case': case}
    if case['op'] == 'attention':
        segs, nq, nk = _segments(case)
        H, D = case['heads'], case['dim']
        s['segments'] = segs
        # q and k as they leave an RMS norm, the incoming gradient of a later layer's scale
        s['q'], s['k'], s['v'] = (randn(n, H, D).requires_grad_() for n in (nq, nk, nk))
        s['dout'] = randn(nq, H, D, std=0.5)
        if case['lse']:
            s['dlse'] = randn(H, nq, std=0.5, dtype=torch.float32)
        if case['via'] == 'varlen':
            s['cu_q'], s['cu_k'] = (torch.tensor([x[i] for x in segs] + [n], dtype=torch.int32, device='cuda')
                                    for i, n in ((0, nq), (2, nk)))
        else:
            s['q_ranges'] = [(a, a + n) for a, n, _, _ in segs]
            s['k_ranges'] = [(a, a + n) for _, _, a, n in segs]
        s['max_q'], s['max_k'] = max(x[1] for x in segs), max(x[3] for x in segs)
    elif case['op'] == 'linear':
        m, k, n, train = case['m'], case['k'], case['n'], case['train']
        s['x'] = randn(m, k).requires_grad_(train)
        s['w'] = randn(n, k, std=k ** -0.5).requires_grad_(train)
        s['b'] = randn(n, std=0.1).requires_grad_(train) if case['bias'] else None
        s['residual'] = randn(m, n) if case['residual'] else None
        s['gate'] = randn(n, std=0.3, mean=0.5).requires_grad_(train) if case['gate'] else None
        s['dy'] = randn(m, n) if train else None
    else:
        rows, H, D = case['rows'], case['heads'], case['dim']
        s['x'] = randn(rows, H * D, std=2.0).requires_grad_()
        s['w'] = randn(D if case['per_head'] else H * D, std=0.1, mean=1.0).requires_grad_()
        angle = torch.rand(rows, D // 2, generator=g, device='cuda') * 60
        # both tables hold each angle twice, as the rotary embeddings of the video models do
        s['cos'], s['sin'] = angle.cos().repeat_interleave(2, -1), angle.sin().repeat_interleave(2, -1)
        s['dy'] = randn(rows, H, D)
    return s


def run(s):
    case = s['case']
    if own:
        if case['op'] == 'attention':
            return _own_attention(s)
        if case['op'] == 'linear':
            return _own_linear(s)
        return _own_norm_rope(s)
    with torch.no_grad():
        if case['op'] == 'attention':
            return _plain_attention(s)
        if case['op'] == 'linear':
            return _plain_linear(s)
        return _plain_norm_rope(s)


# ------------------------------------------------------------------------------------------ the framework's calls

def _own_attention(s):
    from onereel_b200 import attention as A
    q, k, v = s['q'], s['k'], s['v']
    if s['case']['via'] == 'ranges':
        out = A.overlapping_ranges(q, k, v, s['q_ranges'], s['k_ranges'])
    elif s['case']['lse']:
        out, lse = A.varlen_lse(q, k, v, s['cu_q'], s['cu_k'], s['max_q'], s['max_k'])
        dq, dk, dv = torch.autograd.grad((out, lse), (q, k, v), (s['dout'], s['dlse']))
        return {'out': out.detach(), 'lse': lse.detach(), 'dq': dq, 'dk': dk, 'dv': dv}
    else:
        out = A.varlen(q, k, v, s['cu_q'], s['cu_k'], s['max_q'], s['max_k'])
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), s['dout'])
    return {'out': out.detach(), 'dq': dq, 'dk': dk, 'dv': dv}


def _own_linear(s):
    from onereel_b200.linear import linear
    case = s['case']
    y = linear(s['x'], s['w'], s['b'], activation=case['act'] or None, residual=s['residual'], gate=s['gate'])
    if not case['train']:
        return {'y': y}
    names = [n for n in ('x', 'w', 'b', 'gate') if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s['dy'])
    return {'y': y.detach(), **{'d' + n: t for n, t in zip(names, grads)}}


def _own_norm_rope(s):
    from onereel_b200.rope import qk_norm_rope
    case = s['case']
    y = qk_norm_rope(s['x'], s['w'], s['cos'], s['sin'], case['heads'], EPS, per_head=case['per_head'], sin_shift=0)
    dx, dw = torch.autograd.grad(y, (s['x'], s['w']), s['dy'])
    return {'y': y.detach(), 'dx': dx, 'dw': dw}


# ------------------------------------------------------------------------------------------ plain forms, 32 bits

def _plain_attention(s):
    case = s['case']
    H, D = case['heads'], case['dim']
    scale = D ** -0.5
    q, k, v, do = (s[n].float().transpose(0, 1).contiguous() for n in ('q', 'k', 'v', 'dout'))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(k)
    lse = torch.full(q.shape[:2], -math.inf, device=q.device)
    for q0, lq, k0, lk in s['segments']:
        step = max(1, (1 << 29) // max(1, lq * lk))          # heads at a time: four arrays of 2 GiB at most
        for h in range(0, H, step):
            a, b, c = slice(h, h + step), slice(q0, q0 + lq), slice(k0, k0 + lk)
            p = torch.matmul(q[a, b], k[a, c].transpose(1, 2)).mul_(scale)
            top = p.amax(-1, keepdim=True)
            p = p.sub_(top).exp_()
            total = p.sum(-1, keepdim=True)
            p = p.div_(total)
            o = torch.matmul(p, v[a, c])
            out[a, b], lse[a, b] = o, (top + total.log())[..., 0]
            delta = (do[a, b] * o).sum(-1, keepdim=True)
            if case['lse']:
                delta = delta - s['dlse'][a, b, None]
            dv[a, c] += torch.matmul(p.transpose(1, 2), do[a, b])
            ds = torch.matmul(do[a, b], v[a, c].transpose(1, 2)).sub_(delta).mul_(p).mul_(scale)
            dq[a, b] = torch.matmul(ds, k[a, c])
            dk[a, c] += torch.matmul(ds.transpose(1, 2), q[a, b])
    r = {n: t.transpose(0, 1).to(torch.bfloat16).contiguous() for n, t in
         (('out', out), ('dq', dq), ('dk', dk), ('dv', dv))}
    return {**r, 'lse': lse} if case['lse'] else r


def _plain_linear(s):
    case = s['case']
    x, w = s['x'].float(), s['w'].float()
    z = torch.matmul(x, w.t())
    if s['b'] is not None:
        z = z + s['b'].float()
    if case['act'] == 'gelu_tanh':
        t = torch.tanh(SQRT_2_OVER_PI * (z + 0.044715 * z * z * z))
        h, slope = 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * SQRT_2_OVER_PI * (1 + 3 * 0.044715 * z * z)
    elif case['act'] == 'silu':
        t = 1 / (1 + torch.exp(-z))
        h, slope = z * t, t * (1 + z * (1 - t))
    else:
        h, slope = z, None
    y = h if s['gate'] is None else h * s['gate'].float()
    if s['residual'] is not None:
        y = y + s['residual'].float()
    r = {'y': y.to(torch.bfloat16)}
    if case['train']:
        dy = s['dy'].float()
        dz = dy if s['gate'] is None else dy * s['gate'].float()
        dz = dz if slope is None else dz * slope
        r['dx'] = torch.matmul(dz, w).to(torch.bfloat16)
        r['dw'] = torch.matmul(dz.t(), x).to(torch.bfloat16)
        if s['b'] is not None:
            r['db'] = dz.sum(0).to(torch.bfloat16)
        if s['gate'] is not None:
            r['dgate'] = (dy * h).sum(0).to(torch.bfloat16)
    return r


def _plain_norm_rope(s):
    case = s['case']
    rows, H, D = case['rows'], case['heads'], case['dim']
    shape = (rows, H, D) if case['per_head'] else (rows, H * D)
    x, w, dy = s['x'].float().view(shape), s['w'].float(), s['dy'].float()
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = (x * inv * w).view(rows, H, D // 2, 2)
    c, sn = s['cos'][:, None, 0::2], s['sin'][:, None, 0::2]
    y = torch.stack([n[..., 0] * c - n[..., 1] * sn, n[..., 0] * sn + n[..., 1] * c], -1).view(rows, H, D)
    dy = dy.view(rows, H, D // 2, 2)
    u = torch.stack([dy[..., 0] * c + dy[..., 1] * sn, dy[..., 1] * c - dy[..., 0] * sn], -1).view(shape)
    dw = (u * x * inv).sum((0, 1) if case['per_head'] else 0)
    wu = w * u
    dx = inv * wu - x * inv * inv * inv * (wu * x).mean(-1, keepdim=True)
    return {'y': y.to(torch.bfloat16), 'dx': dx.reshape(rows, H * D).to(torch.bfloat16), 'dw': dw.to(torch.bfloat16)}


# ------------------------------------------------------------------------------------------ cost and 64-bit values

def work(case):
    """the inputs read once and the outputs written once; the products of the definition"""
    if case['op'] == 'attention':
        segs, nq, nk = _segments(case)
        H, D = case['heads'], case['dim']
        # q, dout read, out, dq written; k, v read, dk, dv written; seven products of lq x lk x D
        return {'bytes': 8 * (nq + nk) * H * D + (8 * nq * H if case['lse'] else 0),
                'flops': 14 * sum(a * b for _, a, _, b in segs) * H * D}
    if case['op'] == 'linear':
        m, k, n = case['m'], case['k'], case['n']
        elems = m * k + n * k + m * n * (2 if case['residual'] else 1)
        if case['train']:
            elems += m * n + m * k + n * k
        return {'bytes': 2 * elems, 'flops': (6 if case['train'] else 2) * m * n * k}
    rows, H, D = case['rows'], case['heads'], case['dim']
    # x, dy read, y, dx written; both tables read
    return {'bytes': 8 * rows * H * D + 8 * rows * D, 'flops': 30 * rows * H * D}


def exact(case, seed):
    s = prepare(case, seed)
    wide = {n: t.detach().double() for n, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
    if case['op'] == 'attention':
        return _exact_attention(case, s['segments'], wide)
    with torch.enable_grad():
        names = [n for n in ('x', 'w', 'b', 'gate') if n in wide]
        leaves = {n: wide[n].requires_grad_() for n in names}
        if case['op'] == 'linear':
            y = torch.nn.functional.linear(leaves['x'], leaves['w'], leaves.get('b'))
            if case['act'] == 'gelu_tanh':
                y = torch.nn.functional.gelu(y, approximate='tanh')
            elif case['act'] == 'silu':
                y = torch.nn.functional.silu(y)
            if 'gate' in leaves:
                y = y * leaves['gate']
            if 'residual' in wide:
                y = y + wide['residual']
            if not case['train']:
                return {'y': y.detach()}
        else:
            # the rotation as a product of complex numbers
            H, D = case['heads'], case['dim']
            x = leaves['x'].view(-1, H, D) if case['per_head'] else leaves['x']
            n = torch.nn.functional.rms_norm(x, x.shape[-1:], leaves['w'], EPS).reshape(-1, H, D // 2, 2)
            turn = torch.complex(wide['cos'][:, None, 0::2].contiguous(), wide['sin'][:, None, 0::2].contiguous())
            y = torch.view_as_real(torch.view_as_complex(n.contiguous()) * turn).reshape(-1, H, D)
        grads = torch.autograd.grad(y, [leaves[n] for n in names], wide['dy'])
    return {'y': y.detach(), **{'d' + n: t for n, t in zip(names, grads)}}


def _exact_attention(case, segments, wide):
    H, D = case['heads'], case['dim']
    out, dq = torch.zeros_like(wide['q']), torch.zeros_like(wide['q'])
    dk, dv = torch.zeros_like(wide['k']), torch.zeros_like(wide['v'])
    lse = torch.full((H, out.shape[0]), -math.inf, dtype=torch.float64, device=out.device)
    for q0, lq, k0, lk in segments:
        for h in range(H):
            with torch.enable_grad():
                leaves = [wide[n][r0:r0 + m, h].clone().requires_grad_() for n, r0, m in
                          (('q', q0, lq), ('k', k0, lk), ('v', k0, lk))]
                scores = leaves[0] @ leaves[1].t() / math.sqrt(D)
                o, total = torch.softmax(scores, -1) @ leaves[2], torch.logsumexp(scores, -1)
                loss = (o * wide['dout'][q0:q0 + lq, h]).sum()
                if case['lse']:
                    loss = loss + (total * wide['dlse'][h, q0:q0 + lq]).sum()
                a, b, c = torch.autograd.grad(loss, leaves)
            out[q0:q0 + lq, h], lse[h, q0:q0 + lq], dq[q0:q0 + lq, h] = o.detach(), total.detach(), a
            dk[k0:k0 + lk, h] += b
            dv[k0:k0 + lk, h] += c
    r = {'out': out, 'dq': dq, 'dk': dk, 'dv': dv}
    return {**r, 'lse': lse} if case['lse'] else r
