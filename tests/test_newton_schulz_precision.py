"""How many bits newton_schulz keeps.

fp32: the kernels multiply two fp16 parts of each operand (22 bits) and add
up in fp32.  Their results are held against 64 bits with the bound

    2 (error of the same formula in plain fp32 + error of rounding every
       operand to 22 bits, sums exact) + 52 2^-24

on the very input: fp32 sums in another order have errors of the same size,
and where those happen to vanish (a 1 x 1 matrix) one rounding of X a step
is left, which the five steps let grow by at most 10, 18, 11, 8 and 5.
test_what_the_bound_notices plants the mistakes that the kernels could make
in the formula and shows that they are outside.

bf16, from 256 rows on: the first two steps round operands to 11 bits.  The
bound is twice the error of just that, plus the above.
"""

import pytest
import torch

from parallax_amd import ops, optim

GPU = pytest.mark.gpu
A, B, C = 3.4445, -4.7750, 2.0315
SCALE = 4096.0  # of the parts: what lies below fp16's range


def _parts(v):
    hi = (v * SCALE).half().double() / SCALE
    return hi, ((v - hi) * SCALE).half().double() / SCALE


def _mm(a, b, kind):
    if kind == 'exact':
        return a @ b
    (ah, al), (bh, bl) = _parts(a), _parts(b)
    if kind == 'one':
        return ah @ bh
    out = ah @ bh + al @ bh
    return out if kind == 'dropped' else out + ah @ bl


def _wide(g):
    return g.mT.contiguous() if g.shape[-2] > g.shape[-1] else g


def _steps(g, kinds):
    """kinds(step): what the three products of a step are."""
    x = _wide(g.double())
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + 1e-7)
    for i in range(5):
        k = kinds(i)
        p = _mm(x, x.mT.contiguous(), k[0])
        x = A * x + _mm(B * p + C * _mm(p, p, k[1]), x, k[2])
    return x


def _exact(g):
    return _steps(g, lambda i: ('exact',) * 3)


def _two(i):
    return ('two',) * 3


def _one_in_two_steps(i):
    return ('one',) * 3 if i < 2 else _two(i)


MISTAKES = dict(
    one_part_in_two_steps=_one_in_two_steps,
    low_part_of_x=lambda i: ('dropped', 'two', 'two'),
    low_part_of_a=lambda i: ('two', 'dropped', 'two'),
    low_part_of_b=lambda i: ('two', 'two', 'dropped'))


def _plain(g):
    x = _wide(g.double())
    x = (x / (torch.linalg.matrix_norm(x)[..., None, None] + 1e-7)).float()
    for _ in range(5):
        p = x @ x.mT.contiguous()
        x = A * x + (B * p + C * (p @ p)) @ x
    return x.double()


def _off(got, want):
    """of each matrix of a batch, relative to its norm"""
    return torch.linalg.matrix_norm(got - want) \
        / torch.linalg.matrix_norm(want)


def _bound(g, want):
    return 2 * (_off(_plain(g), want) + _off(_steps(g, _two), want)) \
        + 52 * 2.0 ** -24


def _matrices(b, m, n, kind, dev, seed=1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, m, n, generator=g)
    if kind == 'rows':
        x = x * torch.exp(torch.randn(b, m, 1, generator=g))
    if kind == 'rank':
        r = min(4, m, n)
        x = 0.1 * x + torch.randn(b, m, r, generator=g) \
            @ torch.randn(b, r, n, generator=g)
    return (x * 1e-3).to(dev)


# tiles of 32 (uncut, long k cut), of 64 (uncut, cut) and of 128 (uncut, cut)
SHAPES = [(1, 3, 5), (1, 33, 17), (1, 100, 1000), (1, 100, 4000),
          (11, 8, 687), (1, 257, 300), (20, 448, 520), (3, 1100, 1300),
          (1, 1024, 8192), (6, 1100, 1300), (12, 512, 2048)]


@GPU
@pytest.mark.parametrize('kind', ['noise', 'rows', 'rank'])
@pytest.mark.parametrize('b,m,n', SHAPES)
def test_fp32_keeps_22_bits(b, m, n, kind):
    g = _matrices(b, m, n, kind, 'cuda')
    want = _exact(g)
    tol = _bound(g, want)
    got = _wide(ops.newton_schulz(g)).double()
    assert bool((_off(got, want) <= tol).all()), (_off(got, want), tol)
    got = _wide(ops.newton_schulz(g.mT.contiguous())).double()
    assert got.shape == want.shape
    assert bool((_off(got, want) <= tol).all()), (_off(got, want), tol)


@pytest.mark.parametrize('mistake', sorted(MISTAKES))
@pytest.mark.parametrize('b,m,n', [
    (b, m, n) for b, m, n in SHAPES if m < 1024] + [(1, 1100, 1300)])
def test_what_the_bound_notices(b, m, n, mistake):
    """Rows of different size have small singular values, where the steps
    make the most of an error."""
    g = _matrices(min(b, 2), m, n, 'rows', 'cpu')
    want = _exact(g)
    off = _off(_steps(g, MISTAKES[mistake]), want)
    assert bool((off > 2 * _bound(g, want)).all())


def _step_of(w, g, **kw):
    """What one step of Muon takes a zero parameter's fp32 value to."""
    ps = [torch.nn.Parameter(torch.zeros(t.shape, dtype=w, device=t.device))
          for t in g]
    for p, t in zip(ps, g):
        p.grad = t.to(w)
    opt = optim.Muon(ps, lr=1.0, momentum=0.0, **kw)
    opt.step()
    return [-(opt.state[p].get('master', p)).detach().double() for p in ps]


@GPU
@pytest.mark.parametrize('m,n', [(33, 170), (256, 300), (300, 520)])
def test_muon_fp32_keeps_22_bits(m, n):
    g = _matrices(1, m, n, 'rows', 'cuda')
    got, = _step_of(torch.float32, [g[0]])
    want = _exact(g)
    assert bool((_off(got[None], want) <= _bound(g, want)).all())


@GPU
@pytest.mark.parametrize('kind', ['noise', 'rows', 'rank'])
@pytest.mark.parametrize('m,n', [(255, 300), (256, 300), (300, 520),
                                 (1100, 1300)])
def test_muon_bf16_masters_of_any_size(m, n, kind):
    """The masters' step is in 22 bits below 256 rows and has two steps in
    11 bits from there on, no fewer."""
    g = _matrices(1, m, n, kind, 'cuda').bfloat16()
    got, = _step_of(torch.bfloat16, [g[0]])
    want = _exact(g)
    tol = _bound(g, want)
    if m >= 256:
        tol = tol + 2 * _off(_steps(g, _one_in_two_steps), want)
    assert bool((_off(got[None], want) <= tol).all())


@GPU
def test_precision_is_of_the_matrix_not_of_its_company():
    """Matrices of 129 to 256 rows go through the products in one list, but
    only those of 256 have steps in 11 bits."""
    small = _matrices(1, 200, 300, 'rows', 'cuda', seed=2)[0]
    large = _matrices(1, 256, 300, 'rows', 'cuda', seed=3)[0]
    alone = [_step_of(torch.bfloat16, [t])[0] for t in (small, large)]
    for order in (1, -1):
        both = _step_of(torch.bfloat16, [small, large][::order])[::order]
        for p, q in zip(alone, both):
            assert torch.equal(p, q)


@GPU
def test_a_list_of_two_precisions_is_refused():
    f = ops.ext().newton_schulz_list
    mats = [torch.ones(200, 300, device='cuda'),
            torch.ones(256, 300, device='cuda')]
    with pytest.raises(RuntimeError, match='256'):
        f(mats, 5, A, B, C, 1e-7, False)
    f(mats, 5, A, B, C, 1e-7, True)
