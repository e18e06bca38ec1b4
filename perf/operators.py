"""The operators that a language-model training step adds around the model's
body, as cases to time and to compare:

  lce     ops.linear_cross_entropy -- softmax cross entropy of a projection
          onto a large vocabulary, with the gradients of its inputs, its
          table and its bias;
  ns      ops.newton_schulz        -- an update matrix made orthogonal by
          Newton-Schulz products;
  muon    optim.Muon               -- the optimizer step that uses it;
  rotary  ops.apply_rotary         -- rotary positions of queries and keys,
          and their gradients.

``run`` computes an operator in plain torch operations where ``own`` is
false and through the framework where it is true.
"""

import math

import torch

own = False

DEV = 'cuda'
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16,
         'fp32': torch.float32}
NS_COEFFS = (3.4445, -4.7750, 2.0315)
NS_EPS = 1e-7
MUON_LR, MUON_MOMENTUM, MUON_DECAY = 0.02, 0.95, 0.01


def listed():
    return [
        # a toy vocabulary and a handful of tokens: the launches' latency
        dict(name='lce small', op='lce', n=16, v=2000, d=128, dtype='bf16',
             bias=True, smooth=0.0, ignored=0.0, train=True),
        # NMT transformer, tied 32k target table, padded target batch
        dict(name='lce nmt', op='lce', n=2048, v=32000, d=512, dtype='bf16',
             bias=False, smooth=0.1, ignored=0.2, train=True),
        # LM1B: 128 x 20 tokens against the whole 793,470-word table
        dict(name='lce lm1b', op='lce', n=2560, v=793470, d=512,
             dtype='bf16', bias=True, smooth=0.0, ignored=0.0, train=True),
        # LM1B held-out perplexity: 16 x 20 tokens, fp32 table, loss only
        dict(name='lce lm1b eval', op='lce', n=320, v=793470, d=512,
             dtype='fp32', bias=True, smooth=0.0, ignored=0.0, train=False),
        # skip-thoughts decoder, fp32, a ragged batch of odd length
        dict(name='lce skip', op='lce', n=999, v=20000, d=256, dtype='fp32',
             bias=False, smooth=0.0, ignored=0.1, train=True),
        # one attention output projection of the NMT transformer
        dict(name='ns out', op='ns', batch=1, m=512, n=512, dtype='bf16'),
        # the feed-forward weights of its 12 layers, as one batch
        dict(name='ns ffn', op='ns', batch=12, m=2048, n=512, dtype='bf16'),
        # the LM1B LSTM's gate weights, fp32
        dict(name='ns lstm', op='ns', batch=1, m=1024, n=8192,
             dtype='fp32'),
        # two odd matrices: the smallest step of an optimizer
        dict(name='muon pair', op='muon', shapes='150x100,64x200'),
        # the matrices of the NMT transformer's 6 encoder layers
        dict(name='muon nmt', op='muon', shapes=','.join(
            ['1536x512,512x512,2048x512,512x2048'] * 6)),
        # one new token for each of 64 sequences at places of their own
        dict(name='rotary step', op='rotary', b=64, t=1, h=8, hk=8, d=64,
             r=64, interleaved=False, scaled=False, places=4096,
             dtype='bf16', train=False),
        # long sequences, grouped keys, part of the head, scaled angles
        dict(name='rotary long', op='rotary', b=2, t=32768, h=16, hk=4,
             d=128, r=64, interleaved=True, scaled=True, places=65536,
             dtype='bf16', train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['lce', 'lce', 'ns', 'muon', 'rotary'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    if op == 'lce':
        d = _log(rng, 16, 1024)
        if rng.random() < 0.5:
            d = max(64, d // 64 * 64)
        n, v = _log(rng, 1, 4096), _log(rng, 100, 800000)
        most = 2560 * 793470 * 512 // (8 if dtype == 'fp32' else 2)
        v = max(100, min(v, most // (n * d)))
        return dict(op=op, n=n, v=v, d=d, dtype=dtype,
                    bias=rng.random() < 0.5,
                    smooth=rng.choice([0.0, 0.0, 0.1]),
                    ignored=rng.choice([0.0, 0.3]),
                    train=rng.random() < 0.75)
    if op == 'ns':
        m, n = _log(rng, 1, 4096), _log(rng, 1, 4096)
        most = 1 << 33
        batch = max(1, min(_log(rng, 1, 24), most // (m * n * min(m, n))))
        return dict(op=op, batch=batch, m=m, n=n, dtype=dtype)
    if op == 'muon':
        shapes = ['%dx%d' % (_log(rng, 8, 2048), _log(rng, 8, 2048))
                  for _ in range(rng.randint(1, 4))]
        return dict(op=op, shapes=','.join(shapes * rng.randint(1, 4)))
    d = 2 * _log(rng, 4, 128)
    r = d if rng.random() < 0.5 else 2 * rng.randint(1, d // 2)
    hk = _log(rng, 1, 16)
    h = hk * rng.choice([1, 1, 2, 4])
    t = _log(rng, 1, 32768)
    b = max(1, min(_log(rng, 1, 128), (1 << 27) // (t * (h + hk) * d)))
    t = max(1, min(t, (1 << 27) // (b * (h + hk) * d)))
    return dict(op=op, b=b, t=t, h=h, hk=hk, d=d, r=r,
                interleaved=rng.random() < 0.5, scaled=rng.random() < 0.5,
                places=65536, dtype=dtype, train=rng.random() < 0.6)


# -- inputs -------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _zipf(n, v, g):
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    ids = torch.exp(u * math.log(v + 1.0)) - 1.0
    return ids.long().clamp_(0, v - 1)


def _update(shape, g):
    """What an optimizer's momentum holds: a few strong directions over
    noise, rows of different strength."""
    m, n = shape[-2:]
    rank = min(8, m, n)
    lead = shape[:-2]
    a = torch.randn(*lead, m, rank, generator=g, device=DEV)
    b = torch.randn(*lead, rank, n, generator=g, device=DEV)
    noise = torch.randn(*lead, m, n, generator=g, device=DEV)
    rows = torch.exp(0.5 * torch.randn(*lead, m, 1, generator=g, device=DEV))
    return 1e-3 * rows * (noise + (a @ b) * rank ** -0.5)


def _tables(r, places, scaled):
    """cos/sin of every place, from 64-bit angles; `scaled` stretches the
    slow angles eightfold and leaves the fast ones."""
    i = torch.arange(0, r, 2, dtype=torch.float64, device=DEV)
    inv = 10000.0 ** (-i / r)
    if scaled:
        turns = 4096.0 * inv / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0, 1)
        inv = inv * keep + inv / 8.0 * (1 - keep)
    ang = torch.arange(places, dtype=torch.float64, device=DEV)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _shapes(case):
    return [tuple(int(x) for x in s.split('x'))
            for s in case['shapes'].split(',')]


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case['op'] == 'lce':
        dt = TYPES[case['dtype']]
        n, v, d = case['n'], case['v'], case['d']
        s['x'] = torch.randn(n, d, generator=g, device=DEV).to(dt)
        w = torch.randn(v, d, generator=g, device=DEV)
        s['w'] = w.mul_(1.5 * d ** -0.5).to(dt)
        del w
        s['bias'] = None
        if case['bias']:
            rank = torch.arange(v, device=DEV, dtype=torch.float32)
            s['bias'] = (-0.5 * torch.log(rank + 2.0)
                         + 0.1 * torch.randn(v, generator=g,
                                             device=DEV)).to(dt)
        s['y'] = _zipf(n, v, g)
        if case['ignored']:
            out = torch.rand(n, generator=g, device=DEV) < case['ignored']
            out[0] = False
            s['y'] = torch.where(out, -100, s['y'])
        if own and case['train']:
            for k in ('x', 'w', 'bias'):
                if s[k] is not None:
                    s[k].requires_grad_()
    elif case['op'] == 'ns':
        lead = (case['batch'],) if case['batch'] > 1 else ()
        s['g'] = _update(lead + (case['m'], case['n']),
                         g).to(TYPES[case['dtype']])
    elif case['op'] == 'muon':
        s['p'], s['gr'], s['buf'] = [], [], []
        for sh in _shapes(case):
            p = torch.randn(*sh, generator=g, device=DEV) * sh[1] ** -0.5
            s['p'].append(torch.nn.Parameter(p))
            s['gr'].append(_update(sh, g))
            s['buf'].append(5.0 * _update(sh, g))
        if own:
            from parallax_amd import optim
            s['opt'] = optim.Muon(s['p'], lr=MUON_LR,
                                  momentum=MUON_MOMENTUM,
                                  weight_decay=MUON_DECAY)
            for p, gr, buf in zip(s['p'], s['gr'], s['buf']):
                p.grad = gr
                s['opt'].state[p]['momentum_buffer'] = buf
    else:
        dt = TYPES[case['dtype']]
        b, t, h, hk, d = (case[k] for k in ('b', 't', 'h', 'hk', 'd'))
        qkv = torch.randn(b, t, (h + 2 * hk) * d, generator=g,
                          device=DEV).to(dt)
        s['q'] = qkv[..., :h * d].view(b, t, h, d).detach()
        s['k'] = qkv[..., h * d:(h + hk) * d].view(b, t, hk, d).detach()
        first = torch.randint(0, case['places'] - t + 1, (b, 1), generator=g,
                              device=DEV)
        s['pos'] = first + torch.arange(t, device=DEV)
        s['cos'], s['sin'] = _tables(case['r'], case['places'],
                                     case['scaled'])
        if case['train']:
            s['gq'] = torch.randn(b, t, h, d, generator=g, device=DEV).to(dt)
            s['gk'] = torch.randn(b, t, hk, d, generator=g,
                                  device=DEV).to(dt)
            if own:
                s['q'].requires_grad_()
                s['k'].requires_grad_()
    return s


# -- plain forms --------------------------------------------------------------


def _lce_plain(s):
    x, w, b, y = s['x'], s['w'], s['bias'], s['y']
    x32, w32 = x.float(), w.float()
    z = x32 @ w32.t()
    if b is not None:
        z = z + b.float()
    live = y != -100
    yc = torch.where(live, y, 0)[:, None]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    tot = e.sum(1, keepdim=True)
    lse = top + torch.log(tot)
    eps = s['smooth']
    loss = lse - (1 - eps) * z.gather(1, yc)
    if eps:
        loss = loss - eps * z.mean(1, keepdim=True)
    count = live.sum()
    loss = torch.where(live, loss[:, 0], 0.0).sum()
    if not s['train']:
        return loss
    loss = loss / count
    gz = e / tot
    if eps:
        gz = gz - eps / w.shape[0]
    gz.scatter_add_(1, yc, torch.full_like(yc, eps - 1.0,
                                           dtype=torch.float32))
    gz = gz * (live / count)[:, None]
    dx = (gz @ w32).to(x.dtype)
    dw = (gz.t() @ x32).to(w.dtype)
    db = None if b is None else gz.sum(0).to(b.dtype)
    return [loss, dx, dw] + ([] if db is None else [db])


def _ns_plain(g, steps=5):
    a, b, c = NS_COEFFS
    wide = g.shape[-2] <= g.shape[-1]
    x = g.double()
    x = (x / (x.square().sum((-2, -1), keepdim=True).sqrt()
              + NS_EPS)).float()
    x = x if wide else x.transpose(-2, -1).contiguous()
    for _ in range(steps):
        p = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * p + c * (p @ p)) @ x
    return (x if wide else x.transpose(-2, -1)).to(g.dtype)


def _muon_plain(s):
    with torch.no_grad():
        for p, gr, buf in zip(s['p'], s['gr'], s['buf']):
            buf.mul_(MUON_MOMENTUM).add_(gr)
            o = _ns_plain(gr + MUON_MOMENTUM * buf)
            p.mul_(1 - MUON_LR * MUON_DECAY)
            p.sub_(MUON_LR * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * o)
    return [p.detach() for p in s['p']] + s['buf']


def _turn(x, cos, sin, interleaved, back=False):
    """Rotates the leading 2 * cos.shape[-1] values of each head."""
    r = 2 * cos.shape[-1]
    x32 = x[..., :r].float()
    if interleaved:
        u, v = x32[..., 0::2], x32[..., 1::2]
    else:
        u, v = x32[..., :r // 2], x32[..., r // 2:]
    if back:
        sin = -sin
    lo, hi = u * cos - v * sin, u * sin + v * cos
    rot = torch.stack((lo, hi), -1).flatten(-2) if interleaved \
        else torch.cat((lo, hi), -1)
    return torch.cat((rot.to(x.dtype), x[..., r:]), -1)


def _rotary_plain(s):
    cos, sin = s['cos'][s['pos']][:, :, None], s['sin'][s['pos']][:, :, None]
    it = s['interleaved']
    out = [_turn(s['q'], cos, sin, it), _turn(s['k'], cos, sin, it)]
    if s['train']:
        out += [_turn(s['gq'], cos, sin, it, True),
                _turn(s['gk'], cos, sin, it, True)]
    return out


def run(s):
    op = s['op']
    if own:
        from parallax_amd import ops
        if op == 'lce':
            loss = ops.linear_cross_entropy(
                s['x'], s['w'], s['bias'], s['y'],
                reduction='mean' if s['train'] else 'sum',
                label_smoothing=s['smooth'])
            if not s['train']:
                return loss
            wrt = [t for t in (s['x'], s['w'], s['bias']) if t is not None]
            return [loss.detach()] + list(torch.autograd.grad(loss, wrt))
        if op == 'ns':
            return ops.newton_schulz(s['g'])
        if op == 'muon':
            s['opt'].step()
            return [p.detach() for p in s['p']] + s['buf']
        q, k = ops.apply_rotary(s['q'], s['k'], s['cos'], s['sin'],
                                positions=s['pos'],
                                interleaved=s['interleaved'])
        if not s['train']:
            return [q, k]
        return [q.detach(), k.detach()] + list(torch.autograd.grad(
            (q, k), (s['q'], s['k']), (s['gq'], s['gk'])))
    return {'lce': _lce_plain, 'ns': lambda t: _ns_plain(t['g']),
            'muon': _muon_plain, 'rotary': _rotary_plain}[op](s)


# -- what a pass cannot do without --------------------------------------------


def _ns_flops(batch, m, n):
    m, n = min(m, n), max(m, n)
    # two symmetric products, of which one half each, and a full one
    return 5.0 * batch * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    if case['op'] == 'lce':
        n, v, d = case['n'], case['v'], case['d']
        size = TYPES[case['dtype']].itemsize
        inputs = (n * d + v * d + (v if case['bias'] else 0)) * size
        both = 2 if case['train'] else 1
        return {'bytes': both * inputs + n * 8 + 4,
                'flops': (6.0 if case['train'] else 2.0) * n * v * d}
    if case['op'] == 'ns':
        size = TYPES[case['dtype']].itemsize
        return {'bytes': 2 * case['batch'] * case['m'] * case['n'] * size,
                'flops': _ns_flops(case['batch'], case['m'], case['n'])}
    if case['op'] == 'muon':
        sh = _shapes(case)
        return {'bytes': 5 * 4 * sum(m * n for m, n in sh),
                'flops': sum(_ns_flops(1, m, n) for m, n in sh)}
    heads = case['h'] + case['hk']
    values = case['b'] * case['t'] * heads * case['d']
    turned = case['b'] * case['t'] * heads * case['r']
    passes = 2 if case['train'] else 1
    return {'bytes': passes * (2 * values * TYPES[case['dtype']].itemsize
                               + case['b'] * case['t'] * (8 + 4 * case['r'])),
            'flops': passes * 3.0 * turned}


# -- the definitions, in 64 bits ----------------------------------------------


def _lce_exact(s):
    x, y = s['x'].detach().double(), s['y']
    v, eps, rows = s['w'].shape[0], s['smooth'], torch.arange(len(y))
    rows = rows.to(y.device)
    step = max(1, (1 << 28) // max(1, len(y)))
    spans = [(i, min(v, i + step)) for i in range(0, v, step)]

    def logits(i, j):
        w = s['w'][i:j].detach().double()
        z = torch.mm(x, w.t())
        if s['bias'] is not None:
            z += s['bias'][i:j].detach().double()
        return z, w

    parts, total, hit = [], 0.0, torch.zeros_like(x[:, 0])
    for i, j in spans:
        z, _ = logits(i, j)
        parts.append(torch.logsumexp(z, 1))
        total = total + z.sum(1)
        here = (y >= i) & (y < j)
        hit = hit + torch.where(
            here, z[rows, torch.where(here, y - i, 0)], 0.0)
    lse = torch.logsumexp(torch.stack(parts), 0)
    live = (y >= 0).double()
    loss = (live * (lse - (1 - eps) * hit - eps * total / v)).sum()
    if not s['train']:
        return loss
    scale = live / live.sum()
    dx, dw, db = torch.zeros_like(x), [], []
    for i, j in spans:
        z, w = logits(i, j)
        p = torch.exp(z - lse[:, None]) - eps / v
        here = (y >= i) & (y < j)
        p[rows[here], y[here] - i] -= 1 - eps
        p *= scale[:, None]
        dx += p @ w
        dw.append(p.t() @ x)
        db.append(p.sum(0))
    out = [loss / live.sum(), dx, torch.cat(dw)]
    return out + ([] if s['bias'] is None else [torch.cat(db)])


def _ns_exact(g):
    a, b, c = NS_COEFFS
    x = g.double()
    flip = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if flip else x
    norm = torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True)
    x = x / (norm + NS_EPS)
    for _ in range(5):
        p = torch.matmul(x, x.mT.contiguous())
        q = torch.matmul(p, x)
        x = a * x + b * q + c * torch.matmul(p, q)
    return x.mT if flip else x


def _rotary_exact(x, s, sign):
    r = s['r']
    i = torch.arange(r // 2, dtype=torch.float64, device=x.device)
    freq = torch.exp(-2.0 * i / r * math.log(10000.0))
    if s['scaled']:
        keep = ((4096.0 * freq / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / 8.0)
    ang = sign * s['pos'].double()[:, :, None, None] * freq
    turn = torch.polar(torch.ones_like(ang), ang)
    z = x.detach().double().clone()
    pair = slice(0, r, 2), slice(1, r, 2)
    if not s['interleaved']:
        pair = slice(0, r // 2), slice(r // 2, r)
    u = torch.complex(z[..., pair[0]].contiguous(),
                      z[..., pair[1]].contiguous()) * turn
    z[..., pair[0]], z[..., pair[1]] = u.real, u.imag
    return z


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'lce':
        return _lce_exact(s)
    if case['op'] == 'ns':
        return _ns_exact(s['g'])
    if case['op'] == 'muon':
        new, bufs = [], []
        for p, gr, buf in zip(s['p'], s['gr'], s['buf']):
            m = MUON_MOMENTUM * buf.double() + gr.double()
            o = _ns_exact(gr.double() + MUON_MOMENTUM * m)
            ratio = max(1.0, p.shape[0] / p.shape[1]) ** 0.5
            new.append(p.detach().double() * (1 - MUON_LR * MUON_DECAY)
                       - MUON_LR * ratio * o)
            bufs.append(m)
        return new + bufs
    out = [_rotary_exact(s[k], s, 1.0) for k in ('q', 'k')]
    if case['train']:
        out += [_rotary_exact(s[k], s, -1.0) for k in ('gq', 'gk')]
    return out
