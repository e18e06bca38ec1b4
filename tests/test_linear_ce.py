"""linear_cross_entropy against its definition in 64 bits.

Bounds.  With u half a step of the inputs' type and e = 2^-24:
  * a logit is a sum of D products (and the bias) in fp32, or of three such
    sums over 22-bit parts (2^-22 of a product, twice, and its rounding):
    dz = (D + 32) e (|x| |w|^T + |b|);
  * exp2((z - l) log2 e) turns an argument rounded to fp32 into a relative
    error of 3 e |z - l| + 4 e; a sum of V positive terms adds at most V e;
  * so lse and p are off by dz and those (`rel`), G by that times p, and by
    u |G| for its one rounding (2^-22 for fp32, whose G is split);
  * a gradient adds (K + 32) e of the sum of magnitudes over its K terms,
    plus the rounding u of the result (fp16: at least 2^-25, half a step of
    its subnormal numbers).
"""

import math

import pytest
import torch

from parallax_amd import ops

E = 2.0 ** -24
GPU = pytest.mark.gpu
DEVICES = ['cpu', pytest.param('cuda', marks=GPU)]
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11,
     torch.float32: 2.0 ** -24}


def _inputs(n, v, d, dtype, dev, bias=True, seed=0, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g).to(dtype)
    w = (torch.randn(v, d, generator=g) * scale * d ** -0.5).to(dtype)
    b = torch.randn(v, generator=g).to(dtype) if bias else None
    y = torch.randint(0, v, (n,), generator=g)
    return [t if t is None else t.to(dev) for t in (x, w, b, y)]


def _exact(x, w, b, y, dloss, eps=0.0, ignore=-100):
    """losses, dx, dw, db for the rows' upstream gradients, each with its
    bound, in 64 bits on the host."""
    u = U[x.dtype]
    ug = u if x.dtype != torch.float32 else 2.0 ** -22
    x, w, y, dl = (t.detach().cpu() for t in (x, w, y, dloss))
    live = y != ignore
    x = torch.where(live[:, None], x.double(), 0.0)
    w, dl = w.double(), dl.double()
    n, v, d = x.shape[0], w.shape[0], x.shape[1]
    bb = torch.zeros(v, dtype=torch.float64) if b is None \
        else b.detach().cpu().double()
    z = x @ w.t() + bb
    fin = torch.where(torch.isfinite(bb), bb.abs(), 0.0)
    dz = (d + 32) * E * (x.abs() @ w.abs().t() + fin)
    lse = torch.logsumexp(z, 1, keepdim=True)
    yc = torch.where(live, y.clamp(0, v - 1), 0)
    hit = torch.zeros(n, v, dtype=torch.float64)
    hit[torch.arange(n), yc] = 1.0
    zy = z.gather(1, yc[:, None])
    loss = lse - (1 - eps) * zy
    if eps:
        loss = loss - eps * z.mean(1, keepdim=True)
    loss = torch.where(live, loss[:, 0], 0.0)
    p = torch.exp(z - lse)
    span = torch.where(p > 0, (z - lse).abs(), 0.0)
    rel = dz + dz.amax(1, keepdim=True) + (3 * span + 4 + v) * E \
        + (3 * span.amax(1, keepdim=True) + 4) * E
    dloss_ = rel.amax(1) + dz.amax(1) + 8 * E * (lse.abs() + zy.abs())[:, 0]
    if eps:
        dloss_ = dloss_ + eps * v * E * z.abs().mean(1)
    g = torch.where(live, dl, torch.zeros_like(dl))[:, None]
    G = torch.where(live[:, None], (p - (1 - eps) * hit - eps / v) * g, 0.0)
    dG = torch.where(live[:, None], ug * G.abs() + g.abs() * (
        p * rel + 4 * E * (p + hit + eps)), 0.0)
    tiny = 2.0 ** -25 if u == U[torch.float16] else 1e-30

    def out(val, mag, err, k):
        return val, err + (k + 32) * E * mag + U16(val, u) + tiny

    def U16(val, u):
        return u * val.abs()

    dx = out(G @ w, G.abs() @ w.abs(), dG @ w.abs(), v)
    dw = out(G.t() @ x, G.abs().t() @ x.abs(), dG.t() @ x.abs(), n)
    db = out(G.sum(0), G.abs().sum(0), dG.sum(0), n)
    return (loss, dloss_), dx, dw, db


def _close(got, want, what):
    val, tol = want
    off = (got.detach().cpu().double() - val).abs()
    worst = (off / tol.clamp_min(1e-300)).max() if off.numel() else 0.0
    assert bool((off <= tol).all()), (what, float(worst), float(off.max()))


def _check(x, w, b, y, eps=0.0, reduction='mean'):
    leaves = [t if t is None else t.detach().requires_grad_()
              for t in (x, w, b)]
    xl, wl, bl = leaves
    loss = ops.linear_cross_entropy(xl, wl, bl, y, reduction=reduction,
                                    label_smoothing=eps)
    assert loss.dtype == torch.float32
    n = x.shape[0]
    live = y != -100
    if reduction == 'none':
        up = torch.linspace(-1.0, 2.0, n, device=x.device)
        loss.backward(up)
    else:
        loss.backward()
        up = torch.ones(n, device=x.device)
        if reduction == 'mean':
            up = up / live.sum()
    (l, dl), dx, dw, db = _exact(x, w, b, y, up, eps)
    if reduction == 'none':
        _close(loss, (l, dl), 'loss')
    else:
        k = 1.0 if reduction == 'sum' else float(live.sum())
        _close(loss, (l.sum() / k, (dl.sum() + 4 * E * l.abs().sum()) / k),
               'loss')
    _close(xl.grad, dx, 'dx')
    _close(wl.grad, dw, 'dw')
    if bl is not None:
        _close(bl.grad, db, 'db')
    for t, src in zip(leaves, (x, w, b)):
        if t is not None:
            assert t.grad.dtype == src.dtype and t.grad.shape == src.shape


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize('n,v,d', [
    (1, 1, 1), (1, 7, 64), (3, 1000, 33), (17, 257, 64), (64, 300, 128),
    (65, 513, 72), (129, 1025, 192), (300, 2000, 100), (257, 129, 640)])
def test_matches_definition(dev, dtype, n, v, d):
    if dev == 'cpu' and dtype != torch.float32:
        pytest.skip('one type is enough for the host path')
    _check(*_inputs(n, v, d, dtype, dev))


@GPU
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('eps', [0.0, 0.1])
def test_reductions_and_smoothing(dtype, reduction, eps):
    x, w, b, y = _inputs(150, 700, 64, dtype, 'cuda', seed=3)
    y[5:40] = -100
    _check(x, w, b, y, eps, reduction)
    _check(x, w, None, y, eps, reduction)


@GPU
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16,
                                   torch.float16])
def test_several_pieces(dtype, monkeypatch):
    """Enough rows that G is made in pieces of the vocabulary."""
    x, w, b, y = _inputs(40000, 1300, 16, dtype, 'cuda', seed=4)
    y[::7] = -100
    _check(x, w, b, y)


@GPU
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_strides(dtype):
    x, w, b, y = _inputs(70, 260, 128, dtype, 'cuda', seed=5)
    big = torch.zeros(70, 300, dtype=dtype, device='cuda')
    big[:, 3:131] = x
    _check(big[:, 3:131], w, b, y)
    _check(x.t().contiguous().t(), w.t().contiguous().t(), b, y)
    wide = torch.zeros(520, 136, dtype=dtype, device='cuda')
    wide[::2, 8:] = w
    _check(x, wide[::2, 8:], b, y)
    wide = torch.zeros(260, 129, dtype=dtype, device='cuda')
    wide[:, 1:] = w
    _check(x, wide[:, 1:], b, y)
    bb = torch.zeros(520, dtype=dtype, device='cuda')
    bb[::2] = b
    _check(x, w, bb[::2], y)
    one = x[:1].expand(70, 128)
    loss = ops.linear_cross_entropy(one, w, b, y)
    same = ops.linear_cross_entropy(one.contiguous(), w, b, y)
    assert torch.equal(loss, same)


@pytest.mark.parametrize('dev', DEVICES)
def test_leading_dimensions_and_mixed_types(dev):
    x, w, b, y = _inputs(24, 90, 64, torch.float32, dev, seed=6)
    flat = ops.linear_cross_entropy(x, w, b, y, reduction='none')
    cube = ops.linear_cross_entropy(x.view(4, 6, 64), w, b, y.view(4, 6),
                                    reduction='none')
    assert cube.shape == (4, 6) and torch.equal(cube.flatten(), flat)
    # an fp32 table under a bf16 body: cast as the layer norm casts its own
    wl = w.clone().requires_grad_()
    mixed = ops.linear_cross_entropy(x.bfloat16(), wl, b, y.int())
    same = ops.linear_cross_entropy(x.bfloat16(), w.bfloat16(), b, y)
    assert torch.equal(mixed.detach(), same)
    mixed.backward()
    assert wl.grad.dtype == torch.float32
    with torch.autocast(dev, dtype=torch.bfloat16):
        auto = ops.linear_cross_entropy(x, w, b, y)
    assert torch.equal(auto, same) and auto.dtype == torch.float32


@GPU
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_ignored_rows_reach_nothing(dtype):
    x, w, b, y = _inputs(140, 300, 64, dtype, 'cuda', seed=7)
    y[::3] = -100
    bad = x.clone()
    bad[::3] = float('nan')
    bad[3] = float('inf')
    outs = []
    for t in (x, bad):
        leaf = [s.clone().requires_grad_() for s in (t, w, b)]
        loss = ops.linear_cross_entropy(*leaf, y)
        loss.backward()
        outs.append([loss.detach()] + [s.grad for s in leaf])
    for p, q in zip(*outs):
        assert torch.equal(p, q)
    assert not outs[0][1][::3].any()


@pytest.mark.parametrize('dev', DEVICES)
def test_no_row_counts(dev):
    x, w, b, y = _inputs(5, 40, 64, torch.float32, dev, seed=8)
    y[:] = -100
    leaf = [s.clone().requires_grad_() for s in (x, w, b)]
    ops.linear_cross_entropy(*leaf, y, reduction='sum').backward()
    assert all(not s.grad.any() for s in leaf)
    assert math.isnan(ops.linear_cross_entropy(x, w, b, y))
    assert not ops.linear_cross_entropy(x, w, b, y, reduction='none').any()
    none = ops.linear_cross_entropy(x[:0], w, b, y[:0], reduction='sum')
    assert float(none) == 0.0
    assert math.isnan(ops.linear_cross_entropy(x[:0], w, b, y[:0]))


@pytest.mark.parametrize('dev', DEVICES)
def test_masked_words(dev):
    """A bias of -inf takes words out; one of the type's lowest value nearly
    does; a label on a masked word has an infinite loss."""
    x, w, b, y = _inputs(40, 500, 64, torch.float32, dev, seed=9)
    b[100:420] = float('-inf')
    y = y % 100
    if dev == 'cuda':
        _check(x, w, b, y)
    keep = torch.cat([torch.arange(100), torch.arange(420, 500)]).to(dev)
    leaf = [s.clone().requires_grad_() for s in (x, w, b)]
    loss = ops.linear_cross_entropy(*leaf, y)
    loss.backward()
    part = ops.linear_cross_entropy(x, w[keep], b[keep], y)
    assert torch.allclose(loss.detach(), part, rtol=64 * E, atol=0)
    assert not leaf[1].grad[100:420].any() and not leaf[2].grad[100:420].any()
    assert all(torch.isfinite(s.grad).all() for s in leaf)
    low = b.clamp_min(torch.finfo(torch.float32).min)
    assert torch.allclose(ops.linear_cross_entropy(x, w, low, y), part,
                          rtol=64 * E, atol=0)
    y2 = y.clone()
    y2[0] = 200
    each = ops.linear_cross_entropy(x, w, b, y2, reduction='none')
    assert float(each[0]) == float('inf') and torch.isfinite(each[1:]).all()
    every = torch.full_like(b, float('-inf'))
    assert torch.isnan(ops.linear_cross_entropy(x, w, every, y,
                                                reduction='none')).all()


@pytest.mark.parametrize('dev', DEVICES)
def test_labels_outside_are_clamped(dev):
    x, w, b, y = _inputs(6, 50, 64, torch.float32, dev, seed=10)
    y = torch.tensor([-1, 0, 49, 50, 10 ** 12, -10 ** 12], device=dev)
    c = y.clamp(0, 49)
    res = []
    for t in (y, c):
        leaf = [s.clone().requires_grad_() for s in (x, w, b)]
        loss = ops.linear_cross_entropy(*leaf, t)
        loss.backward()
        res.append([loss.detach()] + [s.grad for s in leaf])
    for p, q in zip(*res):
        assert torch.equal(p, q)


@GPU
@pytest.mark.parametrize('scale', [1e-30, 1e-12, 1e6, 1e18])
def test_fp32_range(scale):
    """The powers of two that bring fp32 values into fp16's range."""
    x, w, b, y = _inputs(33, 200, 64, torch.float32, 'cuda', seed=11)
    _check(x * scale, w / scale, b, y)


@GPU
def test_fp32_rows_of_different_size():
    x, w, b, y = _inputs(33, 200, 64, torch.float32, 'cuda', seed=12)
    x[::2] *= 1e-4
    w[::3] *= 1e-3
    w[7] = 0
    _check(x, w, b, y, reduction='none')


@GPU
@pytest.mark.parametrize('up', [0.0, 1e-20, 1e20])
def test_upstream_range(up):
    x, w, b, y = _inputs(33, 200, 64, torch.float32, 'cuda', seed=13)
    leaf = [s.clone().requires_grad_() for s in (x, w, b)]
    (ops.linear_cross_entropy(*leaf, y, reduction='sum') * up).backward()
    want = _exact(x, w, b, y, torch.full((33,), up, dtype=torch.float64))
    for t, e in zip(leaf, want[1:]):
        _close(t.grad, e, up)


@pytest.mark.parametrize('dev', DEVICES)
def test_against_differences(dev):
    """Central differences along random directions.  The loss is off by
    about dl each, and the third derivative of a log-sum-exp along a
    direction is at most 2 (range of the logits' change)^3."""
    x, w, b, y = _inputs(20, 120, 64, torch.float32, dev, seed=14)
    leaf = [s.clone().requires_grad_() for s in (x, w, b)]

    def f(*t):
        return ops.linear_cross_entropy(*t, y, reduction='sum',
                                        label_smoothing=0.1)

    f(*leaf).backward()
    (_, dl), *_ = _exact(x, w, b, y, torch.ones(20), 0.1)
    h = 2.0 ** -5
    for k in range(3):
        to = leaf[k].grad / leaf[k].grad.norm()

        def at(s):
            t = [q.detach() for q in leaf]
            t[k] = t[k] + s * h * to
            return float(f(*t))

        got = (at(1) - at(-1)) / (2 * h)
        d64 = [q.detach().double() for q in leaf]
        dz = (to.double() @ d64[1].t() if k == 0 else
              d64[0] @ to.double().t() if k == 1 else
              to.double()[None].expand(20, -1))
        span = dz.amax(1) - dz.amin(1)
        # the inputs moved by h are rounded to fp32: E of their size
        moved = E * float((leaf[k].detach().abs() * leaf[k].grad.abs())
                          .sum()) / h
        tol = float(dl.sum()) / h + h * h / 3 * float((span ** 3).sum()) \
            + moved
        want = float((leaf[k].grad * to).sum())
        assert abs(got - want) <= tol, (k, got, want, tol)
        assert tol < 0.1 * abs(want), (k, tol, want)


@GPU
def test_same_bits_every_time():
    x, w, b, y = _inputs(300, 3001, 128, torch.bfloat16, 'cuda', seed=16)
    res = []
    for _ in range(3):
        leaf = [s.clone().requires_grad_() for s in (x, w, b)]
        loss = ops.linear_cross_entropy(*leaf, y)
        loss.backward()
        res.append([loss.detach()] + [s.grad for s in leaf])
    for r in res[1:]:
        assert all(torch.equal(p, q) for p, q in zip(res[0], r))


@GPU
def test_only_what_is_asked_for():
    x, w, b, y = _inputs(90, 500, 64, torch.bfloat16, 'cuda', seed=17)
    full = [s.clone().requires_grad_() for s in (x, w, b)]
    ops.linear_cross_entropy(*full, y).backward()
    for k in range(3):
        part = [s.clone().requires_grad_(i == k)
                for i, s in enumerate((x, w, b))]
        ops.linear_cross_entropy(*part, y).backward()
        assert torch.equal(part[k].grad, full[k].grad)
        assert all(part[i].grad is None for i in range(3) if i != k)


@GPU
def test_on_another_stream_and_in_a_graph():
    x, w, b, y = _inputs(200, 1000, 128, torch.bfloat16, 'cuda', seed=18)

    def step(x, w, b, y):
        leaf = [s.detach().requires_grad_() for s in (x, w, b)]
        loss = ops.linear_cross_entropy(*leaf, y)
        return [loss.detach()] + list(torch.autograd.grad(loss, leaf))

    want = step(x, w, b, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = step(x, w, b, y)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    sx = x.clone()
    with torch.cuda.graph(graph):
        out = step(sx, w, b, y)
    for seed in range(3):
        x2 = _inputs(200, 1000, 128, torch.bfloat16, 'cuda',
                     seed=30 + seed)[0]
        sx.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(x2, w, b, y)
        assert all(torch.equal(p, q) for p, q in zip(out, eager))


@GPU
def test_table_past_32_bits():
    """Words whose rows lie behind 2^31 elements of the table."""
    v, d, n = (1 << 22) + 700, 520, 6
    w = torch.empty(v, d, dtype=torch.bfloat16, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(19)
    for i in range(0, v, 1 << 20):
        w[i:i + (1 << 20)] = torch.randn(
            w[i:i + (1 << 20)].shape, generator=g, device='cuda') * 0.05
    x = torch.randn(n, d, generator=g, device='cuda').bfloat16()
    y = torch.tensor([v - 1, v - 2, 5, v - 600, 1 << 22, 0], device='cuda')
    bias = torch.full((v,), -20.0, dtype=torch.bfloat16, device='cuda')
    bias[-700:] = 0
    bias[:10] = 0
    rows = torch.cat([torch.arange(10), torch.arange(v - 700, v)]).cuda()
    xl, wl = x.clone().requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(xl, wl, bias, y, reduction='none')
    loss.sum().backward()
    z = torch.cat([x.double() @ w[i:i + (1 << 18)].detach().double().t()
                   + bias[i:i + (1 << 18)].double()
                   for i in range(0, v, 1 << 18)], 1)
    lse = torch.logsumexp(z, 1)
    want = lse - z.gather(1, y[:, None])[:, 0]
    # terms add up in fp32 along chains far shorter than 2^13
    tol = 2.0 ** -11 + 600 * E * 0.05 * 520
    assert float((loss.double() - want).abs().max()) < tol
    p = torch.exp(z[:, rows] - lse[:, None])
    p[y[:, None] == rows] -= 1
    dw = p.t() @ x.double()
    off = (wl.grad[rows].double() - dw).abs()
    bound = 2.0 ** -7 * (p.abs().t() @ x.double().abs()) + 1e-4
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize('dev', DEVICES)
def test_refusals(dev):
    x, w, b, y = _inputs(6, 50, 64, torch.float32, dev, seed=20)
    f = ops.linear_cross_entropy
    with pytest.raises(ValueError, match='reduction'):
        f(x, w, b, y, reduction='avg')
    with pytest.raises(ValueError, match='label_smoothing'):
        f(x, w, b, y, label_smoothing=1.0)
    with pytest.raises(ValueError, match='weight'):
        f(x, w[:, :60], b, y)
    with pytest.raises(ValueError, match='labels'):
        f(x, w, b, y[:5])
    with pytest.raises(ValueError, match='bias'):
        f(x, w, b[:7], y)
    with pytest.raises(TypeError, match='labels'):
        f(x, w, b, y.float())
    with pytest.raises(TypeError, match='inputs'):
        f(x.long(), w, b, y)
    if dev == 'cuda':
        with pytest.raises(RuntimeError, match='bf16, fp16 or fp32'):
            f(x.double(), w, b, y)
        with pytest.raises(RuntimeError, match='GPU|device'):
            f(x, w.cpu(), b, y)


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('asked', [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_only_the_asked_gradients(dev, asked):
    x, w, b, y = _inputs(70, 300, 64, torch.float32, dev, seed=21)
    every = [t.clone().requires_grad_() for t in (x, w, b)]
    ops.linear_cross_entropy(*every, y).backward()
    some = [t.clone().requires_grad_(i in asked)
            for i, t in enumerate((x, w, b))]
    ops.linear_cross_entropy(*some, y).backward()
    for i, (s, t) in enumerate(zip(some, every)):
        if i in asked:
            assert torch.equal(s.grad, t.grad)
        else:
            assert s.grad is None


@pytest.mark.parametrize('dev', DEVICES)
def test_no_rows_give_no_gradient(dev):
    x, w, b, y = _inputs(5, 40, 64, torch.float32, dev, seed=22)
    w[3] = float('nan')
    for reduction in ('mean', 'sum', 'none'):
        leaf = [t.clone().requires_grad_() for t in (x[:0], w, b)]
        ops.linear_cross_entropy(*leaf, y[:0], reduction=reduction).sum() \
            .backward()
        assert not leaf[1].grad.any() and not leaf[2].grad.any()


@GPU
def test_second_derivatives_are_refused():
    x, w, b, y = _inputs(9, 40, 64, torch.float32, 'cuda', seed=23)
    leaf = [t.clone().requires_grad_() for t in (x, w, b)]
    loss = ops.linear_cross_entropy(*leaf, y)
    first = torch.autograd.grad(loss, leaf, create_graph=True)
    plain = torch.autograd.grad(ops.linear_cross_entropy(*leaf, y), leaf)
    for p, q in zip(first, plain):
        assert torch.equal(p, q)
        with pytest.raises(RuntimeError, match='again'):
            torch.autograd.grad(p.sum(), leaf, retain_graph=True)


@GPU
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('eps', [0.0, 0.1])
def test_equal_rows_are_not_rounded_alike(dtype, eps):
    """A mean over 45 or 53 rows gives every row 1/45 or 1/53, and a label
    without probability -(1 - eps) of that: rounded to 8 or 11 bits, all
    labels' parts of the gradients would be off by the same.  Relative to
    that value they are 1 and round to themselves: G is off by D = what
    rounding G / up / (1 - eps) changes, dx by D w and dw by D^T x, and each
    by its own rounding, so in norm by at most the sum of both.  The other
    bounds above, of 2^-24, are below a hundredth of it."""
    for n in (45, 53):
        x, w, b, y = _inputs(n, 3000, 256, dtype, 'cuda', seed=24)
        leaf = [t.clone().requires_grad_() for t in (x, w, b)]
        ops.linear_cross_entropy(*leaf, y, label_smoothing=eps).backward()
        up = torch.full((n,), 1.0 / n, dtype=torch.float64)
        _, dx, dw, _ = _exact(x, w, b, y, up, eps)
        x, w, b, y = (t.cpu() for t in (x, w, b, y))
        x, w, b = x.double(), w.double(), b.double()
        G = torch.softmax(x @ w.t() + b, 1) - eps / 3000
        G[torch.arange(n), y] -= 1 - eps
        G = G / (1 - eps) * (1.0 if dtype == torch.bfloat16 else 8192.0)
        D = (G.to(dtype).double() - G) * ((1 - eps) / n)
        if dtype == torch.float16:
            D = D / 8192.0
        for t, (want, _), part in zip(leaf, (dx, dw), (D @ w, D.t() @ x)):
            own = (want.to(dtype).double() - want).norm()
            off = (t.grad.cpu().double() - want).norm()
            assert float(off) < 1.01 * float(own + part.norm())


@GPU
def test_piece_at_the_largest_offset():
    """A table of 2^31 bytes and more: the last values before that."""
    last = (1 << 31) // 8192 - 1
    v, d = last + 300, 4096
    g = torch.Generator(device='cuda').manual_seed(25)
    w = torch.empty(v, d, dtype=torch.bfloat16, device='cuda')
    w.normal_(0, 1 / 64, generator=g)
    x = torch.randn(3, d, generator=g, device='cuda').bfloat16()
    xl = x.clone().requires_grad_()
    y = torch.full((3,), last, device='cuda')
    ops.linear_cross_entropy(xl, w, None, y, reduction='sum').backward()
    # E[w exp(x w)] / E[exp(x w)] = x / 64^2 for words of deviation 1 / 64;
    # about it the mean over V words with logits of deviation 1 has one of
    # sqrt(e / V) / 64, which the second term is 4.8 times; bf16 rounds by
    # 2^-8 of the result
    tol = 2.0 ** -8 * w[last].float().abs() + 8 * v ** -0.5 / 64
    off = (xl.grad.float() + w[last].float() - x.float() / 4096).abs()
    assert bool((off <= tol).all()), float((off - tol).max())
    assert float(w[last, -8:].abs().max()) > 4 * float(tol.max())


@GPU
def test_refused_sizes():
    f = ops.linear_cross_entropy
    big = torch.zeros(1, 1, device='cuda').expand(1 << 20, 512)
    y = torch.zeros(1, dtype=torch.long, device='cuda').expand(1 << 20)
    w = torch.zeros(4, 512, device='cuda')
    with pytest.raises(RuntimeError, match='fewer rows'):
        f(big, w, None, y)
    with pytest.raises(RuntimeError, match='2.20 rows'):
        f(big[:, :1].expand(1 << 20, 1).repeat(2, 1), w[:, :1], None,
          y.repeat(2))
    with pytest.raises(RuntimeError, match='32768'):
        f(torch.zeros(2, 40000, device='cuda'),
          torch.zeros(3, 40000, device='cuda'), None, y[:2])


@GPU
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n', [128, 130, 192, 193, 256, 320, 321, 440, 449])
def test_every_tile_of_rows(dtype, n):
    _check(*_inputs(n, 600, 128, dtype, 'cuda', seed=26))


@GPU
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n', [193, 256, 320, 350, 385, 512])
@pytest.mark.parametrize('eps', [0.0, 0.1])
def test_larger_tiles(dtype, n, eps):
    """Enough words that the large tiles of rows run, whole and cut."""
    x, w, b, y = _inputs(n, 8310, 64, dtype, 'cuda', seed=27)
    y[3:9] = -100
    _check(x, w, b, y, eps)


@pytest.mark.parametrize('dev', DEVICES)
def test_no_words_are_refused(dev):
    x, w, b, y = _inputs(5, 7, 4, torch.float32, dev, seed=28)
    with pytest.raises(ValueError, match='one word'):
        ops.linear_cross_entropy(x, w[:0], b[:0], y)
    with pytest.raises(ValueError, match='one word'):
        ops.linear_cross_entropy(x[:, :0], w[:, :0], b, y)
