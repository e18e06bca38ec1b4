"""The ways a program calls linear_cross_entropy, newton_schulz and
apply_rotary in: without autograd, through checkpointing and hooks that move
what is saved, on two streams at once.  All are the plain call, to the bit."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from parallax_amd import ops

GPU = pytest.mark.gpu
DEVICES = ['cpu', pytest.param('cuda', marks=GPU)]


def _loss(dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(150, 128, generator=g)
    w = torch.randn(900, 128, generator=g) * 0.1
    b = torch.randn(900, generator=g)
    y = torch.randint(0, 900, (150,), generator=g).to(dev)

    def call(*leaf):
        return ops.linear_cross_entropy(*leaf, y, label_smoothing=0.1)

    return call, [t.to(dtype).to(dev) for t in (x, w, b)]


def _turn(dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(2, 9, 4, 32, generator=g).to(dtype).to(dev)
    k = torch.randn(2, 9, 2, 32, generator=g).to(dtype).to(dev)
    cos, sin = ops.rotary_tables(32, 9, device=dev)

    def call(q, k):
        a, b = ops.apply_rotary(q, k, cos, sin)
        return a.float().square().sum() + b.float().sin().sum()

    return call, [q, k]


def _with_gradients(call, args):
    leaf = [t.clone().requires_grad_() for t in args]
    out = call(*leaf)
    return [out.detach()] + list(torch.autograd.grad(out, leaf))


def _same(a, b):
    assert len(a) == len(b)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('make', [_loss, _turn])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_without_autograd_and_recomputed(make, dtype, dev):
    call, args = make(dtype, dev)
    want = _with_gradients(call, args)
    with torch.no_grad():
        _same([call(*args)], want[:1])
    with torch.inference_mode():
        _same([call(*[t.clone() for t in args])], want[:1])
    _same(_with_gradients(
        lambda *t: checkpoint(call, *t, use_reentrant=False), args), want)
    with torch.autograd.graph.save_on_cpu():
        _same(_with_gradients(call, args), want)
    # of a graph that is kept, twice
    leaf = [t.clone().requires_grad_() for t in args]
    out = call(*leaf)
    for _ in range(2):
        _same(list(torch.autograd.grad(out, leaf, retain_graph=True)),
              want[1:])


@pytest.mark.parametrize('dev', DEVICES)
def test_newton_schulz_without_autograd(dev):
    g = torch.randn(3, 40, 70, generator=torch.Generator().manual_seed(1))
    g = g.to(dev)
    want = ops.newton_schulz(g)
    with torch.inference_mode():
        assert torch.equal(ops.newton_schulz(g.clone()), want)
    assert not ops.newton_schulz(g.requires_grad_()).requires_grad


@GPU
def test_a_changed_input_is_noticed():
    """Autograd's check of what the backward reads (the host keeps copies)."""
    call, args = _loss(torch.float32, 'cuda')
    for i in (0, 1):
        leaf = [t.clone().requires_grad_() for t in args]
        live = [t * 1 for t in leaf]
        out = call(*live)
        with torch.no_grad():
            live[i].add_(1)
        with pytest.raises(RuntimeError, match='modified'):
            out.backward()


@GPU
@pytest.mark.parametrize('make', [_loss, _turn])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_two_streams_at_once(make, dtype):
    cases = [make(dtype, 'cuda', seed) for seed in range(2)]
    want = [_with_gradients(*c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for s, c in zip(streams, cases):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(_with_gradients(*c))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for i, o in enumerate(got):
        _same(o, want[i % 2])
