"""newton_schulz and optim.Muon against their definitions in 64 bits.

Bounds, as the 2-norm of the difference over that of the result:
  * bf16: its rounding is at most 2^-8 of each value, so of the norm too.
    From 256 rows on the first two steps multiply one-part operands (2^-12
    of each value): three products of two operands, of independent errors
    of 2^-12 / sqrt(3) each, grow by at most 10 and 18 as below.
  * fp16: the rounding, 2^-11, and two-part products as for fp32.
  * fp32: each product and each stored X is off by (k + 8) 2^-24 (fp32 sums
    of k terms, independent ones, so the square root of k; 22-bit operands
    count as 4 each).  A relative error of a singular value that is made
    before step 1..5 grows by at most 10, 18, 11, 8 and 5 (the largest
    |s f'(s) / f(s)| of what is left of the five steps, over all s in
    (0, 1]): 52 for all of them.  One that is small against the whole matrix
    but not against a small singular value grows by a^5 = 485, out of a
    matrix of norm 1 into one of norm sqrt(min(m, n)).
"""

import math

import pytest
import torch

from parallax_amd import ops, optim

GPU = pytest.mark.gpu
DEVICES = ['cpu', pytest.param('cuda', marks=GPU)]
A, B, C = 3.4445, -4.7750, 2.0315


def _exact(g, steps=5, eps=1e-7, coeffs=(A, B, C)):
    a, b, c = coeffs
    x = g.detach().cpu().double()
    flip = x.shape[-2] > x.shape[-1]
    x = x.mT if flip else x
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    for _ in range(steps):
        p = x @ x.mT
        x = a * x + b * p @ x + c * p @ (p @ x)
    return x.mT if flip else x


def _bound(dtype, m, n):
    k = max(m, n)
    grown = 52 + 485 / math.sqrt(min(m, n))
    fine = grown * 2.0 ** -24 * 3 * (math.sqrt(k) + 8)
    if dtype == torch.bfloat16 and min(m, n) >= 256:
        fine += (10 + 18) * 2.0 ** -12 * math.sqrt(6 / 3)
    return fine + {torch.bfloat16: 2.0 ** -8,
                   torch.float16: 2.0 ** -11,
                   torch.float32: 0.0}[dtype]


def _off(got, want):
    d = got.detach().cpu().double() - want
    return float(d.norm() / want.norm().clamp_min(1e-300))


def _matrix(m, n, kind='noise', seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=g)
    if kind == 'rows':
        x = x * torch.exp(torch.randn(m, 1, generator=g))
    if kind == 'rank':
        r = min(4, m, n)
        x = 0.1 * x + torch.randn(m, r, generator=g) \
            @ torch.randn(r, n, generator=g)
    return x * 1e-3


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize('m,n', [
    (1, 1), (1, 50), (50, 1), (3, 5), (33, 17), (64, 64), (65, 130),
    (128, 128), (100, 1000), (700, 90), (257, 300)])
@pytest.mark.parametrize('kind', ['noise', 'rows', 'rank'])
def test_matches_definition(dev, dtype, m, n, kind):
    g = _matrix(m, n, kind).to(dtype).to(dev)
    if dtype == torch.float16:
        g = g * 64  # away from fp16's subnormal numbers
    got = ops.newton_schulz(g)
    assert got.shape == g.shape and got.dtype == dtype
    assert _off(got, _exact(g)) < _bound(dtype, m, n), _off(got, _exact(g))


@GPU
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_wide_tiles(dtype):
    """Enough of them that the larger tile runs, on and off its edges."""
    for shape in [(3, 1100, 1300), (20, 448, 520)]:
        g = torch.stack([_matrix(*shape[1:], seed=i)
                         for i in range(shape[0])]).to(dtype).cuda()
        got = ops.newton_schulz(g)
        want = _exact(g)
        for i in range(shape[0]):
            assert _off(got[i], want[i]) < _bound(dtype, *shape[1:])


@GPU
def test_more_than_go_through_together():
    g = torch.randn(70, 2048, 2048, dtype=torch.bfloat16, device='cuda')
    got = ops.newton_schulz(g)
    for i in (0, 69):
        off = _off(got[i], _exact(g[i]))
        assert off < _bound(torch.bfloat16, 2048, 2048), off
    g = torch.randn(70000, 2, 3, device='cuda')
    got = ops.newton_schulz(g)
    for i in (0, 20000, 69999):
        assert _off(got[i], _exact(g[i])) < _bound(torch.float32, 2, 3)


@pytest.mark.parametrize('dev', DEVICES)
def test_batches_are_separate(dev):
    g = torch.stack([_matrix(40, 70, k, i) * 10.0 ** (3 * i - 3)
                     for i, k in enumerate(('noise', 'rows', 'rank'))])
    g = g.to(dev)
    got = ops.newton_schulz(g.view(3, 1, 40, 70))
    assert got.shape == (3, 1, 40, 70)
    for i in range(3):
        assert torch.allclose(got[i, 0], ops.newton_schulz(g[i]),
                              rtol=0, atol=1e-6)


@pytest.mark.parametrize('dev', DEVICES)
def test_range_and_special_values(dev):
    g = _matrix(40, 70).to(dev)
    want = _exact(g)
    for s in (1e-12, 1e15, 1e30):  # the norm's squares need 64 bits
        # the scaled entries are rounded once more, 2^-24 of each
        assert _off(ops.newton_schulz(g * s, eps=0.0), want) < \
            _bound(torch.float32, 40, 70)
    zero = torch.zeros(5, 7, device=dev)
    assert not ops.newton_schulz(zero).any()
    assert ops.newton_schulz(g[:0]).shape == (0, 70)
    assert ops.newton_schulz(g[None][:0]).shape == (0, 40, 70)
    bad = torch.stack([g, g])
    bad[0, 3, 3] = float('nan')
    got = ops.newton_schulz(bad)
    assert torch.isnan(got[0]).any() and torch.isfinite(got[1]).all()
    bad[0, 3, 3] = float('inf')
    assert torch.isnan(ops.newton_schulz(bad)[0]).any()


@pytest.mark.parametrize('dev', DEVICES)
def test_strides_steps_and_coefficients(dev):
    g = _matrix(60, 90).to(dev)
    want = ops.newton_schulz(g)
    wide = torch.zeros(120, 95, device=dev)
    wide[::2, 5:] = g
    assert torch.equal(ops.newton_schulz(wide[::2, 5:]), want)
    t = g.t().contiguous().t()
    assert torch.equal(ops.newton_schulz(t), want)
    assert _off(ops.newton_schulz(g.t()), want.cpu().double().t()) < 1e-5
    soft = (1.875, -1.25, 0.375)  # 15/8, -10/8, 3/8: rises to 1 from below
    for steps in (1, 2, 8):
        got = ops.newton_schulz(g, steps=steps, coefficients=soft)
        assert _off(got, _exact(g, steps, coeffs=soft)) < \
            _bound(torch.float32, 60, 90)


def test_singular_values_come_near_one():
    """In 64 bits: where the definition leads is what the name says."""
    o = _exact(_matrix(40, 80))
    s = torch.linalg.svdvals(o)
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


@pytest.mark.parametrize('dev', DEVICES)
def test_refusals(dev):
    g = _matrix(6, 9).to(dev)
    f = ops.newton_schulz
    with pytest.raises(ValueError, match='matrix'):
        f(g[0])
    with pytest.raises(TypeError, match='floating'):
        f(g.int())
    for steps in (0, 65, 2.5):
        with pytest.raises(ValueError, match='steps'):
            f(g, steps=steps)
    with pytest.raises(ValueError, match='three'):
        f(g, coefficients=(1.0, 2.0))
    if dev == 'cuda':
        with pytest.raises(RuntimeError, match='bf16, fp16 or fp32'):
            f(g.double())
        with pytest.raises(RuntimeError, match='32768'):
            f(torch.zeros(1, 40000, device=dev))


@GPU
def test_same_bits_other_stream_and_graph():
    g = torch.stack([_matrix(200, 130, seed=i) for i in range(3)]).cuda()
    want = ops.newton_schulz(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.newton_schulz(g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    buf = g.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.newton_schulz(buf)
    for i in range(3):
        buf.copy_(torch.stack([_matrix(200, 130, seed=10 * i + j)
                               for j in range(3)]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.newton_schulz(buf))


# -- the optimizer ------------------------------------------------------------


def _muon_exact(w, buf, g, lr=0.02, mom=0.95, wd=0.0, nesterov=True):
    """One step on 64-bit (rows, cols) matrices."""
    buf.mul_(mom).add_(g)
    o = _exact(g + mom * buf if nesterov else buf)
    w.mul_(1 - lr * wd).sub_(lr * max(1.0, w.shape[0] / w.shape[1]) ** 0.5
                             * o)


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('nesterov,wd', [(True, 0.0), (False, 0.1)])
def test_muon_fp32(dev, nesterov, wd):
    shapes = [(40, 24), (24, 40), (40, 24), (16, 5, 3, 3), (1, 9), (7, 1),
              (0, 4)]
    g = torch.Generator().manual_seed(1)
    ps = [torch.nn.Parameter((torch.randn(s, generator=g) * 0.1).to(dev))
          for s in shapes]
    # a transposed and a channels-last parameter
    ps.append(torch.nn.Parameter(torch.randn(30, 20, generator=g)
                                 .to(dev).t()))
    ps.append(torch.nn.Parameter(
        torch.randn(12, 6, 3, 3, generator=g).to(dev)
        .to(memory_format=torch.channels_last)))
    opt = optim.Muon(ps, nesterov=nesterov, weight_decay=wd)
    ref = [(p.detach().cpu().double().flatten(1).clone(),
            torch.zeros_like(p.detach().cpu().double().flatten(1)))
           for p in ps]
    for step in range(3):
        for p, (w, b) in zip(ps, ref):
            gr = torch.randn(p.shape, generator=g) * 10.0 ** (step - 2)
            if not p.numel():
                p.grad = gr.to(dev)
                continue
            p.grad = gr.to(dev)  # contiguous: another layout than some p's
            _muon_exact(w, b, gr.double().reshape(w.shape), wd=wd,
                        nesterov=nesterov)
        opt.step()
    for p, (w, b) in zip(ps, ref):
        if not p.numel():
            continue
        o = _bound(torch.float32, *w.shape) * 3 * 0.02 \
            * max(1.0, w.shape[0] / w.shape[1]) ** 0.5 \
            * min(w.shape) ** 0.5 * 1.25
        off = (p.detach().cpu().double().reshape(w.shape) - w).norm()
        assert float(off) < o + 6 * 2.0 ** -24 * float(w.norm()), p.shape
        buf = opt.state[p]['momentum_buffer'].cpu().double()
        assert torch.allclose(buf.reshape(w.shape), b, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_muon_many_of_about_one_size(dev, dtype):
    """Wide, tall, odd ones and vectors as matrices, more than go together;
    each as if it were the only one."""
    g = torch.Generator().manual_seed(6)
    shapes = [(5 + i, 60 - i) for i in range(55)] + [(1, 128), (128, 128),
                                                     (3, 129), (129, 3)]
    ws = [torch.randn(s, generator=g).to(dtype) for s in shapes]
    gs = [torch.randn(s, generator=g).to(dtype) for s in shapes]
    ps = [torch.nn.Parameter(w.clone().to(dev)) for w in ws]
    for p, gr in zip(ps, gs):
        p.grad = gr.to(dev)
    opt = optim.Muon(ps)
    opt.step()
    for p, w, gr in zip(ps, ws, gs):
        w, b = w.double(), torch.zeros(w.shape, dtype=torch.float64)
        _muon_exact(w, b, gr.double())
        got = opt.state[p]['master'] if dtype == torch.bfloat16 else p
        step = 0.02 * max(1.0, w.shape[0] / w.shape[1]) ** 0.5 \
            * 1.25 * min(w.shape) ** 0.5
        off = float((got.detach().cpu().double() - w).norm())
        assert off < step * _bound(torch.float32, *w.shape) \
            + 2 * 2.0 ** -24 * float(w.norm()), p.shape


def test_list_refusals():
    f = ops.ext().newton_schulz_list
    with pytest.raises(RuntimeError, match='GPU'):
        f([torch.zeros(4, 4)], 5, A, B, C, 1e-7, True)
    with pytest.raises(RuntimeError, match='steps'):
        f([torch.zeros(4, 4)], 0, A, B, C, 1e-7, True)
    f([], 5, A, B, C, 1e-7, True)


@GPU
def test_list_refusals_on_the_gpu():
    f = ops.ext().newton_schulz_list
    z = torch.zeros(8, 8, device='cuda')
    for other in (torch.zeros(8, 200, device='cuda'),
                  torch.zeros(200, 8, device='cuda')):
        with pytest.raises(RuntimeError, match='padded'):
            f([z, other], 5, A, B, C, 1e-7, True)
    for other in (z[:, :4], z.bfloat16(), z.cpu(), z[:0], z[0]):
        with pytest.raises(RuntimeError, match='one type'):
            f([z, other], 5, A, B, C, 1e-7, True)


@pytest.mark.parametrize('dev', DEVICES)
def test_muon_bf16_masters(dev):
    """bf16 parameters keep fp32 masters: ten steps, each smaller than the
    parameters' rounding, arrive."""
    g = torch.Generator().manual_seed(2)
    w0 = torch.randn(48, 80, generator=g).bfloat16()
    p = torch.nn.Parameter(w0.to(dev))
    opt = optim.Muon([p], lr=1e-3)
    w, b = w0.double(), torch.zeros(48, 80, dtype=torch.float64)
    moved = w.clone()
    for _ in range(10):
        gr = torch.randn(48, 80, generator=g).bfloat16()
        p.grad = gr.to(dev)
        _muon_exact(w, b, gr.double(), lr=1e-3)
        opt.step()
    master = opt.state[p]['master'].cpu().double()
    per_step = 1e-3 * 1.25 * 48 ** 0.5
    # the update stays fp32 behind the products: no 2^-8 of a rounding
    assert float((master - w).norm()) < 10 * (
        per_step * _bound(torch.float32, 48, 80)
        + 2.0 ** -24 * float(w.norm()))
    assert float((w - moved).norm()) > 3 * per_step
    assert torch.equal(p.detach().cpu(), master.float().bfloat16())


@pytest.mark.parametrize('dev', DEVICES)
def test_muon_vectors_groups_and_rows_take_adam(dev):
    g = torch.Generator().manual_seed(3)

    def leaf(*s):
        return torch.nn.Parameter(torch.randn(*s, generator=g).to(dev))

    mat, vec, head, table = leaf(20, 30), leaf(30), leaf(10, 30), leaf(50, 8)
    opt = optim.Muon([dict(params=[mat, vec, table]),
                      dict(params=[head], muon=False, adam_lr=1e-2)],
                     weight_decay=0.5)
    twins = [torch.nn.Parameter(t.detach().clone()) for t in (vec, head)]
    adam = [optim.Adam([twins[0]], lr=3e-4, betas=(0.9, 0.95)),
            optim.Adam([twins[1]], lr=1e-2, betas=(0.9, 0.95))]
    rows = torch.nn.Parameter(table.detach().clone())
    lazy = optim.Adam([rows], lr=3e-4, betas=(0.9, 0.95))
    ids = torch.tensor([3, 7], device=dev)
    before = mat.detach().clone()
    for _ in range(3):
        for t in (mat, vec, head):
            t.grad = torch.randn(t.shape, generator=g).to(dev)
        vals = torch.randn(2, 8, generator=g).to(dev)
        table.grad = torch.sparse_coo_tensor(ids[None], vals, (50, 8))
        twins[0].grad, twins[1].grad = vec.grad.clone(), head.grad.clone()
        rows.grad = table.grad.clone()
        opt.step()
        for a in adam + [lazy]:
            a.step()
    assert torch.equal(vec, twins[0]) and torch.equal(head, twins[1])
    assert torch.equal(table, rows)
    assert not torch.equal(mat, before)
    assert 'exp_avg' not in opt.state[mat]
    assert 'momentum_buffer' not in opt.state[vec]


@pytest.mark.parametrize('dev', DEVICES)
def test_muon_state_round_trip(dev):
    g = torch.Generator().manual_seed(4)
    ws = [torch.randn(12, 20, generator=g).bfloat16(),
          torch.randn(20, generator=g)]
    grads = [[torch.randn(w.shape, generator=g).to(w.dtype).to(dev)
              for w in ws] for _ in range(4)]

    def fresh(src):
        ps = [torch.nn.Parameter(w.detach().clone().to(dev)) for w in src]
        return ps, optim.Muon(ps)

    def go(ps, opt, some):
        for gs in some:
            for p, q in zip(ps, gs):
                p.grad = q.clone()
            opt.step()

    p1, o1 = fresh(ws)
    go(p1, o1, grads)
    p2, o2 = fresh(ws)
    go(p2, o2, grads[:2])
    p3, o3 = fresh(p2)
    o3.load_state_dict(o2.state_dict())
    go(p3, o3, grads[2:])
    for p, q in zip(p1, p3):
        assert torch.equal(p, q)


def test_muon_refusals():
    p = torch.nn.Parameter(torch.randn(4, 4))
    with pytest.raises(ValueError, match='momentum'):
        optim.Muon([p], momentum=1.0)
    with pytest.raises(ValueError, match='ns_steps'):
        optim.Muon([p], ns_steps=0)
    odd = torch.nn.Parameter(torch.randn(4, 6, 8).permute(2, 0, 1)[:, :, ::2])
    odd.grad = torch.randn(8, 4, 3)
    with pytest.raises(ValueError, match='does not lie'):
        optim.Muon([odd]).step()
    opt = optim.Muon([p])
    p.grad = torch.randn(4, 4)
    opt.state[p]['momentum_buffer'] = torch.zeros(4, 5)
    with pytest.raises(ValueError, match='momentum buffer'):
        opt.step()


@GPU
def test_muon_in_a_graph():
    g = torch.Generator().manual_seed(5)
    w = torch.randn(70, 40, generator=g).cuda()
    p = torch.nn.Parameter(w.clone())
    q = torch.nn.Parameter(w.clone())
    op, oq = optim.Muon([p]), optim.Muon([q])
    grad = torch.randn(70, 40, generator=g).cuda()
    p.grad, q.grad = grad.clone(), grad.clone()
    op.step()
    oq.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.step()
    for _ in range(3):
        nxt = torch.randn(70, 40, generator=g).cuda()
        p.grad.copy_(nxt)
        q.grad.copy_(nxt)
        graph.replay()
        torch.cuda.synchronize()
        oq.step()
        assert torch.equal(p, q)


@GPU
def test_muon_fp16():
    g = torch.Generator().manual_seed(7)
    w0 = torch.randn(30, 50, generator=g).half()
    gr = torch.randn(30, 50, generator=g).half()
    p = torch.nn.Parameter(w0.cuda())
    p.grad = gr.cuda()
    opt = optim.Muon([p])
    opt.step()
    w, b = w0.double(), torch.zeros(30, 50, dtype=torch.float64)
    _muon_exact(w, b, gr.double())
    off = (opt.state[p]['master'].cpu().double() - w).norm()
    assert float(off) < 0.02 * 1.25 * 30 ** 0.5 \
        * _bound(torch.float32, 30, 50) + 2 * 2.0 ** -24 * float(w.norm())
    assert torch.equal(p.detach(), opt.state[p]['master'].half())


@GPU
def test_two_streams_at_once():
    """Calls that run side by side share nothing."""
    g = [_matrix(300, 500, seed=i).cuda() for i in range(2)]
    want = [ops.newton_schulz(t) for t in g]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for s, t in zip(streams, g):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(ops.newton_schulz(t))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])
