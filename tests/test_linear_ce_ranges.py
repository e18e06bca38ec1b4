"""linear_cross_entropy over sizes and values that a small case does not
reach, against its definition in 64 bits on the same device.

Bounds.  With u half a step of the results' type, ug one of G's and
e = 2^-24: a logit is off by dz = (D + 32) e (|x| |w|^T + |b|), so the
logarithm of a probability by dz, the largest dz of its row (for lse) and the
rounding of exp2's argument, 3 e |z - lse| + 4 e; lse adds V e for the sum of
V positive terms.  G is off by that times p and by ug |G|, the products by
the sums of that and by (K + 32) e of the magnitudes of their K terms, and
the results are rounded by u.
"""

import pytest
import torch

from parallax_amd import ops

E = 2.0 ** -24
GPU = pytest.mark.gpu
DEVICES = ['cpu', pytest.param('cuda', marks=GPU)]
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11,
     torch.float32: 2.0 ** -24}


def _exact(x, w, b, y, up):
    """{name: (value, bound)} of dx, dw and db for the rows' upstream
    gradients ``up``."""
    u = U[x.dtype]
    ug = u if x.dtype != torch.float32 else 2.0 ** -22
    x, w, up = x.detach().double(), w.detach().double(), up.double()
    n, d = x.shape
    v = w.shape[0]
    z = x @ w.t()
    dz = x.abs() @ w.abs().t()
    if b is not None:
        z += b.detach().double()
        dz += b.detach().double().abs()
    dz *= (d + 32) * E
    z -= torch.logsumexp(z, 1, keepdim=True)
    rel = dz + (3 * z.abs() + 4) * E
    rel += dz.amax(1, keepdim=True) + v * E
    p = z.exp()
    g = up[:, None]
    G = p * g
    dG = g.abs() * p * (rel + 4 * E)
    rows = torch.arange(n, device=x.device)
    G[rows, y] -= up
    dG[rows, y] += 4 * E * up.abs()
    dG += ug * G.abs()

    def out(val, mag, err, k):
        return val, err + (k + 32) * E * mag + u * val.abs() + 1e-30

    A = G.abs()
    return dict(dx=out(G @ w, A @ w.abs(), dG @ w.abs(), v),
                dw=out(G.t() @ x, A.t() @ x.abs(), dG.t() @ x.abs(), n),
                db=out(G.sum(0), A.sum(0), dG.sum(0), n))


def _inside(got, want, what):
    val, tol = want
    off = (got.double() - val).abs()
    assert bool((off <= tol).all()), (what, float((off / tol).max()))


@GPU
@pytest.mark.parametrize('asked', [(0, 1, 2), (0,), (1,)])
@pytest.mark.parametrize('n,v,d', [(4000, 22600, 640), (4000, 21800, 640)])
def test_widths_that_do_not_divide_a_piece(n, v, d, asked):
    """Rows of 640 values are three tiles of 256, of which 256 CUs hold
    21,845 words' worth, no multiple of a tile: the pieces of the vocabulary
    have to be, whether there are several or one."""
    g = torch.Generator(device='cuda').manual_seed(0)
    x = torch.randn(n, d, generator=g, device='cuda').bfloat16()
    w = (torch.randn(v, d, generator=g, device='cuda') * d ** -0.5) \
        .bfloat16()
    b = torch.randn(v, generator=g, device='cuda').bfloat16()
    y = torch.randint(0, v, (n,), generator=g, device='cuda')
    leaf = [t.clone().requires_grad_(i in asked)
            for i, t in enumerate((x, w, b))]
    ops.linear_cross_entropy(*leaf, y, reduction='sum').backward()
    want = _exact(x, w, b, y, torch.ones(n, device='cuda'))
    for i, name in enumerate(('dx', 'dw', 'db')):
        if i in asked:
            _inside(leaf[i].grad, want[name], name)


def _spread(dev, n=300, v=3000, d=96, seed=1):
    """Words whose probabilities go from 1e-1 to 1e-16."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g)
    w = torch.randn(v, d, generator=g) * d ** -0.5
    b = -30.0 * torch.rand(v, generator=g)
    y = torch.randint(0, v, (n,), generator=g)
    b[y] = b[y] / 4
    return [t.to(dev) for t in (x, w, b, y)]


def _gradients_inside(x, w, b, y, up):
    leaf = [t.clone().requires_grad_() for t in (x, w, b)]
    ops.linear_cross_entropy(*leaf, y, reduction='none').backward(up)
    want = _exact(x, w, b, y, up)
    for t, name in zip(leaf, ('dx', 'dw', 'db')):
        _inside(t.grad, want[name], name)
    return want


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('n', [5, 300, 5000])
def test_fp32_words_of_tiny_probability(dev, n):
    """Each word's gradient is as exact as fp32 values are, however rare the
    word: _exact's bounds are relative to the word's own terms."""
    x, w, b, y = _spread(dev, n=n)
    up = torch.ones(n, device=dev)
    dw = _gradients_inside(x, w, b, y, up)['dw'][0]
    size = dw.norm(dim=1)
    assert float(size.min()) < 1e-11 * float(size.max())


@pytest.mark.parametrize('dev', DEVICES)
def test_fp32_rows_of_tiny_gradient(dev):
    """Rows whose upstream gradients differ by 1e15."""
    x, w, b, y = _spread(dev, seed=2)
    up = 10.0 ** torch.linspace(-12, 3, 300, device=dev)
    _gradients_inside(x, w, b, y, up)
    up[::3] = 0.0
    _gradients_inside(x, w, b, y, -up)


@pytest.mark.parametrize('dev', DEVICES)
def test_fp32_rows_of_tiny_inputs(dev):
    """A word that only rows of tiny inputs make likely has a gradient as
    exact as the others'."""
    x, w, b, y = _spread(dev, seed=3)
    x[:150] *= 1e-7
    y[:150] = torch.arange(150, device=dev) + 2000
    y[150:] %= 2000
    b[2000:2150] = -30.0
    dw = _gradients_inside(x, w, b, y, torch.ones(300, device=dev))['dw'][0]
    size = dw.norm(dim=1)
    assert float(size[2000:2150].max()) < 1e-5 * float(size[:2000].max())


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('ignore', [-100, 7])
def test_what_ignored_rows_hold_is_not_read(dev, reduction, ignore):
    """NaN and infinities in the rows of a padded batch, whatever the label
    that marks them."""
    x, w, b, y = _spread(dev, n=40, v=200, d=24, seed=4)
    y[y == 7] = 8
    y[::3] = ignore
    bad = x.clone()
    bad[::3] = float('nan')
    bad[3] = float('inf')
    bad[6, 5] = -float('inf')
    outs = []
    for t in (x, bad):
        leaf = [s.clone().requires_grad_() for s in (t, w, b)]
        loss = ops.linear_cross_entropy(*leaf, y, reduction=reduction,
                                        ignore_index=ignore,
                                        label_smoothing=0.1)
        loss.sum().backward()
        outs.append([loss.detach()] + [s.grad for s in leaf])
    for p, q in zip(*outs):
        assert torch.isfinite(p).all() and torch.equal(p, q)
    assert not outs[1][1][::3].any() and outs[1][1][1::3].any()


def test_fp64_on_the_host():
    """64 bits stay 64 bits, so torch's own check against differences
    holds; the GPU refuses them."""
    x, w, b, y = _spread('cpu', n=6, v=20, d=5, seed=5)
    y[2] = -100
    x, w, b = (t.double().requires_grad_() for t in (x, w, b / 10))
    for reduction in ('mean', 'none'):
        def f(x, w, b):
            return ops.linear_cross_entropy(x, w, b, y, reduction=reduction,
                                            label_smoothing=0.2)

        assert f(x, w, b).dtype == torch.float64
        assert torch.autograd.gradcheck(f, (x, w, b))
        assert ops.linear_cross_entropy(
            x[:0], w, b, y[:0], reduction=reduction).dtype == torch.float64
    z = x @ w.t() + b
    want = torch.nn.functional.cross_entropy(z, y)
    got = ops.linear_cross_entropy(x, w, b, y)
    assert abs(float(got - want)) < 1e-13


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('eps', [0.0, 1e-9])
def test_no_loss_is_negative(dev, dtype, eps):
    """Labels of a probability that rounds to 1: lse and the label's logit
    are sums in different orders, each off by its rounding."""
    g = torch.Generator().manual_seed(6)
    w = torch.randn(200, 96, generator=g)
    y = torch.randint(0, 200, (300,), generator=g)
    x = w[y] * 20 + torch.randn(300, 96, generator=g)
    x, w, y = x.to(dtype).to(dev), w.to(dtype).to(dev), y.to(dev)
    each = ops.linear_cross_entropy(x, w, None, y, reduction='none',
                                    label_smoothing=eps)
    z = x.double() @ w.double().t()
    want = (1 - eps) * (torch.logsumexp(z, 1)
                        - z.gather(1, y[:, None])[:, 0]) \
        + eps * (torch.logsumexp(z, 1) - z.mean(1))
    tol = 2 * (96 + 32) * E * (x.double().abs() @ w.double().abs().t()) \
        .amax(1) + 8 * E * z.abs().amax(1)
    assert float(z.amax(1).min()) > 500
    assert bool((each >= 0).all()), float(each.min())
    assert bool(((each.double() - want).abs() <= tol).all())
    assert bool(torch.isnan(ops.linear_cross_entropy(
        x * float('nan'), w, None, y, reduction='none')).all())


@GPU
@pytest.mark.parametrize('n', [40, 130, 256, 300, 1000])
@pytest.mark.parametrize('v,d', [(13001, 200), (700, 600)])
def test_fp32_every_tile_of_both_gradients(n, v, d):
    """Tiles of 64 and 128 rows behind one another, whose scales differ, in
    the large and the small tile of dw."""
    x, w, b, y = _spread('cuda', n=n, v=v, d=d, seed=n)
    up = 10.0 ** torch.linspace(3, -12, n, device='cuda')
    x *= 10.0 ** torch.linspace(-3, 0, n, device='cuda')[:, None]
    _gradients_inside(x, w, b, y, up)


@GPU
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_the_most_rows(dtype):
    """2^20 rows: a piece is 256 words, of which G takes up to 1 GB twice.
    (dw is a sum of 2^20 terms, whose order the bound allows for.)"""
    n, v, d = 1 << 20, 300, 16
    g = torch.Generator(device='cuda').manual_seed(7)
    x = torch.randn(n, d, generator=g, device='cuda').to(dtype)
    w = torch.randn(v, d, generator=g, device='cuda').to(dtype)
    b = torch.randn(v, generator=g, device='cuda').to(dtype)
    y = torch.randint(0, v, (n,), generator=g, device='cuda')
    up = torch.rand(n, generator=g, device='cuda') * 2.0 ** -20
    _gradients_inside(x, w, b, y, up)
