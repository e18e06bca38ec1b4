"""apply_rotary and its tables against rotations of complex numbers in 64
bits.

Bound: cos and sin are fp32 (2^-24 of at most 1); two products and a sum in
fp32 add 3 * 2^-24 of |u| + |v|; the result is rounded once, half a step of
its type (fp16: at least 2^-25, half a step of its subnormal numbers).
"""

import math

import pytest
import torch

from parallax_amd import ops

GPU = pytest.mark.gpu
DEVICES = ['cpu', pytest.param('cuda', marks=GPU)]
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11,
     torch.float32: 2.0 ** -24}
E = 2.0 ** -24


def _exact(x, pos, r, interleaved, sign=1.0, inv=None):
    """x [B, T, H, D] on the host, pos [B, T]; the value and |u| + |v|."""
    z = x.detach().cpu().double().clone()
    mag = torch.zeros_like(z)
    if inv is None:
        inv = 10000.0 ** (-torch.arange(0, r, 2).double() / r)
    ang = sign * pos.cpu().double()[:, :, None, None] * inv
    w = torch.polar(torch.ones_like(ang), ang)
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved \
        else (slice(0, r // 2), slice(r // 2, r))
    u, v = z[..., first].clone(), z[..., second].clone()
    t = torch.complex(u, v) * w
    z[..., first], z[..., second] = t.real, t.imag
    mag[..., first] = mag[..., second] = u.abs() + v.abs()
    return z, mag


def _close(got, want, u):
    z, mag = want
    off = (got.detach().cpu().double() - z).abs()
    tiny = 2.0 ** -25 if u == U[torch.float16] else 0.0
    tol = u * z.abs() + 4 * E * mag + tiny
    assert bool((off <= tol).all()), float((off - tol).max())


def _pair(b, t, h, hk, d, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, t, h, d, generator=g).to(dtype).to(dev)
    k = torch.randn(b, t, hk, d, generator=g).to(dtype).to(dev)
    return q, k


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('b,t,h,hk,d,r', [
    (1, 1, 1, 1, 2, 2), (3, 1, 8, 8, 64, 64), (2, 7, 4, 1, 128, 64),
    (2, 5, 3, 2, 33, 16), (1, 300, 6, 2, 80, 80), (2, 3, 5, 5, 30, 10),
    (1, 2, 70, 9, 256, 32)])
def test_matches_definition(dev, dtype, interleaved, b, t, h, hk, d, r):
    q, k = _pair(b, t, h, hk, d, dtype, dev)
    cos, sin = ops.rotary_tables(r, 1000, device=dev)
    g = torch.Generator().manual_seed(1)
    pos = torch.randint(0, 1000, (b, t), generator=g)
    q.requires_grad_()
    k.requires_grad_()
    a, c = ops.apply_rotary(q, k, cos, sin, positions=pos.to(dev),
                            interleaved=interleaved)
    assert a.dtype == dtype and a.shape == q.shape and c.shape == k.shape
    _close(a, _exact(q, pos, r, interleaved), U[dtype])
    _close(c, _exact(k, pos, r, interleaved), U[dtype])
    ga, gc = _pair(b, t, h, hk, d, dtype, dev, seed=2)
    dq, dk = torch.autograd.grad((a, c), (q, k), (ga, gc))
    _close(dq, _exact(ga, pos, r, interleaved, -1.0), U[dtype])
    _close(dk, _exact(gc, pos, r, interleaved, -1.0), U[dtype])


@pytest.mark.parametrize('dev', DEVICES)
def test_places(dev):
    """An offset, [T], [1, T], int32 and [B, T] say the same; places outside
    the tables go to their ends."""
    q, k = _pair(2, 6, 3, 3, 16, torch.float32, dev)
    cos, sin = ops.rotary_tables(16, 40, device=dev)
    want = ops.apply_rotary(q, k, cos, sin, offset=9)
    row = torch.arange(9, 15, device=dev)
    for pos in (row, row[None], row.int(), row.expand(2, 6),
                row.repeat(2, 1)):
        got = ops.apply_rotary(q, k, cos, sin, positions=pos)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out = torch.tensor([-5, 0, 39, 40, 10 ** 10, 7], device=dev)
    got = ops.apply_rotary(q, None, cos, sin, positions=out)
    same = ops.apply_rotary(q, None, cos, sin, positions=out.clamp(0, 39))
    assert torch.equal(got, same)
    assert ops.apply_rotary(q[:0], k[:0], cos, sin)[0].shape == q[:0].shape
    none = ops.apply_rotary(q[:, :0], k[:, :0], cos, sin,
                            positions=row[:0])
    assert none[1].shape == k[:, :0].shape


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('interleaved', [False, True])
def test_strides(dev, interleaved):
    """Views of a packed projection, heads before tokens, odd offsets,
    broadcast heads: the values of dense copies, bit for bit."""
    g = torch.Generator().manual_seed(3)
    b, t, h, d = 2, 9, 4, 64
    for dtype in (torch.float32, torch.bfloat16):
        cos, sin = ops.rotary_tables(48, 64, device=dev)
        qkv = torch.randn(b, t, 3 * h * d + 3, generator=g).to(dtype).to(dev)
        for first in (0, 1, 2, 3):
            q = qkv[..., first:first + h * d].unflatten(-1, (h, d))
            k = qkv[..., first + h * d:first + 2 * h * d] \
                .unflatten(-1, (h, d))
            views = [(q, k),
                     (q.transpose(1, 2).contiguous().transpose(1, 2), k),
                     (q, k[:, :, :1].expand(b, t, h, d)),
                     (q.flip(3).transpose(2, 3).contiguous()
                      .transpose(2, 3), k)]
            for x, y in views:
                x, y = x.detach().requires_grad_(), y.detach() \
                    .requires_grad_()
                got = ops.apply_rotary(x, y, cos, sin, offset=5,
                                       interleaved=interleaved)
                want = ops.apply_rotary(x.contiguous(), y.contiguous(), cos,
                                        sin, offset=5,
                                        interleaved=interleaved)
                up = [torch.randn(s.shape, generator=g).to(dtype).to(dev)
                      for s in got]
                for p, w in zip(got, want):
                    assert torch.equal(p, w)
                dg = torch.autograd.grad(got, (x, y), up)
                dw = torch.autograd.grad(want, (x, y), up)
                for p, w in zip(dg, dw):
                    assert torch.equal(p, w)


@pytest.mark.parametrize('dev', DEVICES)
def test_one_gradient_alone_and_broadcast(dev):
    q, k = _pair(2, 4, 3, 2, 16, torch.float32, dev)
    cos, sin = ops.rotary_tables(16, 8, device=dev)
    q.requires_grad_()
    k.requires_grad_()
    a, c = ops.apply_rotary(q, k, cos, sin)
    pos = torch.arange(4).expand(2, 4)
    ones, _ = torch.autograd.grad(a.sum(), (q, k), allow_unused=True,
                                  retain_graph=True)
    _close(ones, _exact(torch.ones_like(q), pos, 16, False, -1.0), E)
    dk, = torch.autograd.grad(c.sum(), (k,))
    _close(dk, _exact(torch.ones_like(k), pos, 16, False, -1.0), E)


@pytest.mark.parametrize('dev', DEVICES)
def test_against_differences(dev):
    """The map is linear: differences are exact up to rounding."""
    q, _ = _pair(1, 5, 2, 1, 32, torch.float32, dev)
    cos, sin = ops.rotary_tables(32, 100, device=dev)
    up, step = _pair(1, 5, 2, 2, 32, torch.float32, dev, seed=4)

    def f(x):
        y = ops.apply_rotary(x, None, cos, sin, offset=50)
        return (y.double() * up.double()).sum()

    q.requires_grad_()
    dq, = torch.autograd.grad(f(q), q)
    with torch.no_grad():
        got = float(f(q + step) - f(q - step)) / 2
    want = float((dq.double() * step.double()).sum())
    # 5 E of |u| + |v| for each of the values, in both passes
    tol = 20 * E * float((up.abs() * (q.detach().abs() + step.abs())).sum()) * 2
    assert abs(got - want) < tol and tol < 1e-3


@pytest.mark.parametrize('scaling', [None, 'linear', 'ntk', 'yarn'])
def test_tables(scaling):
    r, f, n = 32, 4.0, 200000
    cos, sin = ops.rotary_tables(r, n, base=500.0, scaling=scaling, factor=f,
                                 original_places=256)
    i = torch.arange(r // 2).double()
    plain = 500.0 ** (-2 * i / r)
    m = 1.0
    if scaling == 'linear':
        inv = plain / f
    elif scaling == 'ntk':
        inv = (500.0 * f ** (r / (r - 2.0))) ** (-2 * i / r)
        assert abs(float(inv[-1] / plain[-1]) * f - 1) < 1e-12
        assert float(inv[0]) == 1.0
    elif scaling == 'yarn':
        m = 0.1 * math.log(f) + 1
        # 256 places: an angle that turns 32 times has index < 0, once: 9.5
        lo = max(math.floor(r * math.log(256 / (2 * math.pi * 32))
                            / (2 * math.log(500.0))), 0)
        hi = math.ceil(r * math.log(256 / (2 * math.pi))
                       / (2 * math.log(500.0)))
        part = ((i - lo) / (hi - lo)).clamp(0, 1)
        inv = plain * (1 - part) + plain / f * part
        assert float(inv[0]) == 1.0 and float(inv[-1] * f / plain[-1]) == 1
    else:
        inv = plain
    at = torch.tensor([0, 1, 77, 131072, n - 1])
    ang = at.double()[:, None] * inv
    # rounded to fp32 once; the angle in 64 bits is off by 2^-52 of itself
    tol = m * (E + n * 2.0 ** -50)
    assert float((cos[at].double() - m * ang.cos()).abs().max()) <= tol
    assert float((sin[at].double() - m * ang.sin()).abs().max()) <= tol


@pytest.mark.parametrize('dev', DEVICES)
def test_module(dev):
    q, k = _pair(2, 6, 4, 2, 32, torch.bfloat16, dev)
    rot = ops.ParallaxRotary(32, 64, rotary_dim=16, interleaved=True,
                             scaling='linear', factor=2.0).to(dev)
    assert not rot.state_dict()
    before = rot.cos.clone()
    rot.to(torch.bfloat16)
    assert rot.cos.dtype == torch.float32 and torch.equal(rot.cos, before)
    a, c = rot(q, k, offset=3)
    pos = torch.arange(3, 9).expand(2, 6)
    inv = 10000.0 ** (-torch.arange(0, 16, 2).double() / 16) / 2
    _close(a, _exact(q, pos, 16, True, inv=inv), U[torch.bfloat16])
    assert torch.equal(rot(q, offset=3), a)
    assert torch.equal(rot(k, offset=3), c)


def test_scores_depend_on_distance():
    g = torch.Generator().manual_seed(5)
    q, k = torch.randn(2, 1, 8, 1, 32, generator=g)
    cos, sin = ops.rotary_tables(32, 600)
    a = ops.apply_rotary(q, k, cos, sin, offset=0)
    b = ops.apply_rotary(q, k, cos, sin, offset=500)
    sa, sb = (x[0][0, :, 0] @ x[1][0, :, 0].t() for x in (a, b))
    assert torch.allclose(sa, sb, atol=64 * E * 32 * 4)


@GPU
def test_long_and_past_32_bits():
    """Far places, and a batch whose last values lie behind 2^31."""
    cos, sin = ops.rotary_tables(64, 1 << 20, device='cuda')
    big = torch.empty(3, 180000, 32, 128, dtype=torch.bfloat16,
                      device='cuda')
    assert big.numel() > 1 << 31
    g = torch.Generator(device='cuda').manual_seed(6)
    tail = torch.randn(20, 32, 128, generator=g, device='cuda').bfloat16()
    big.zero_()
    big[2, -20:] = tail
    pos = torch.zeros(3, 180000, dtype=torch.long, device='cuda')
    pos[2, -20:] = torch.arange((1 << 20) - 20, 1 << 20, device='cuda')
    out = ops.apply_rotary(big, None, cos, sin, positions=pos)
    _close(out[2:, -20:], _exact(tail[None], pos[2:, -20:], 64, False),
           U[torch.bfloat16])
    assert not out[:2].any() and not out[2, :-20].any()


@GPU
def test_other_stream_and_graph():
    q, k = _pair(2, 16, 4, 2, 64, torch.bfloat16, 'cuda')
    cos, sin = ops.rotary_tables(64, 100, device='cuda')
    pos = torch.arange(16, device='cuda').repeat(2, 1)

    def step(q, k, pos):
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        out = ops.apply_rotary(q, k, cos, sin, positions=pos)
        return list(out) + list(torch.autograd.grad(out, (q, k), out))

    want = step(q, k, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(q, k, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(q, k, pos)
    for i in range(3):
        pos += 5
        graph.replay()
        torch.cuda.synchronize()
        eager = step(q, k, pos)
        assert all(torch.equal(x, y) for x, y in zip(out, eager))


@pytest.mark.parametrize('dev', DEVICES)
def test_refusals(dev):
    q, k = _pair(2, 6, 4, 2, 16, torch.float32, dev)
    cos, sin = ops.rotary_tables(16, 8, device=dev)
    f = ops.apply_rotary
    with pytest.raises(ValueError, match='q '):
        f(q[0], None, cos, sin)
    with pytest.raises(TypeError, match='type'):
        f(q.long(), None, cos, sin)
    with pytest.raises(ValueError, match='does not match'):
        f(q, k[:, :3], cos, sin)
    with pytest.raises(ValueError, match='does not match'):
        f(q, k.bfloat16(), cos, sin)
    with pytest.raises(ValueError, match='tables'):
        f(q[..., :14], None, cos, sin)
    with pytest.raises(ValueError, match='tables'):
        f(q, k, cos, sin[:, :4])
    with pytest.raises(ValueError, match='places'):
        f(q, k, cos, sin, offset=3)
    with pytest.raises(ValueError, match='places'):
        f(q, k, cos, sin, offset=-1)
    pos = torch.arange(6, device=dev)
    with pytest.raises(ValueError, match='not both'):
        f(q, k, cos, sin, positions=pos, offset=1)
    with pytest.raises(ValueError, match='positions'):
        f(q, k, cos, sin, positions=pos[:5])
    with pytest.raises(TypeError, match='positions'):
        f(q, k, cos, sin, positions=pos.float())
    with pytest.raises(ValueError, match='even'):
        ops.rotary_tables(7, 8)
    with pytest.raises(ValueError, match='scaling'):
        ops.rotary_tables(8, 8, scaling='dynamic')
    with pytest.raises(ValueError, match='factor'):
        ops.rotary_tables(8, 8, scaling='linear', factor=0.5)
    with pytest.raises(ValueError, match='original_places'):
        ops.rotary_tables(8, 8, scaling='yarn', factor=2.0)
    with pytest.raises(ValueError, match='place'):
        ops.rotary_tables(8, 0)
    with pytest.raises(ValueError, match='rotary_dim'):
        ops.ParallaxRotary(16, 8, rotary_dim=32)


@pytest.mark.parametrize('dev', DEVICES)
def test_tables_get_no_gradient(dev):
    cos, sin = ops.rotary_tables(16, 8, device=dev)
    q, k = _pair(2, 4, 3, 2, 16, torch.float32, dev)
    want = ops.apply_rotary(q, k, cos, sin)
    got = ops.apply_rotary(q, k, cos.requires_grad_(), sin.requires_grad_())
    for a, b in zip(got, want):
        assert torch.equal(a, b) and not a.requires_grad


@GPU
def test_refused_on_the_gpu():
    cos, sin = ops.rotary_tables(16, 8, device='cuda')
    q, k = _pair(2, 4, 3, 2, 16, torch.float32, 'cuda')
    with pytest.raises(RuntimeError, match='bf16, fp16 or fp32'):
        ops.apply_rotary(q.double(), k.double(), cos, sin)
    q.requires_grad_()
    a, _ = ops.apply_rotary(q, k, cos, sin)
    up = torch.ones_like(a, requires_grad=True)
    dq, = torch.autograd.grad(a, q, up, create_graph=True)
    with pytest.raises(RuntimeError, match='again'):
        torch.autograd.grad(dq.sum(), up)
