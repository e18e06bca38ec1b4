"""optim.SGD with momentum over bf16 parameters: fp32 masters and buffers,
against the update in 64 bits."""

import pytest
import torch

from parallax_amd import ops, optim

GPU = pytest.mark.gpu
DEVICES = ['cpu', pytest.param('cuda', marks=GPU)]
E = 2.0 ** -24


@pytest.mark.parametrize('dev', DEVICES)
@pytest.mark.parametrize('nesterov,wd', [(False, 0.0), (True, 0.0),
                                         (True, 0.01)])
def test_masters_and_buffers(dev, nesterov, wd):
    """Each of the steps rounds the buffer, the update and the master to
    fp32 (at most six roundings of values of their sizes); the buffer's
    errors stay with it, as it shrinks by 0.9 a step: 10 of them."""
    lr, mom, steps = 0.05, 0.9, 6
    g = torch.Generator().manual_seed(0)
    shapes = [(33, 17), (129,), (4, 3, 5), (1,)]
    types = [torch.bfloat16, torch.bfloat16, torch.bfloat16, torch.float32]
    ws = [torch.randn(s, generator=g).to(t) for s, t in zip(shapes, types)]
    ps = [torch.nn.Parameter(w.clone().to(dev)) for w in ws]
    opt = optim.SGD(ps, lr=lr, momentum=mom, nesterov=nesterov,
                    weight_decay=wd)
    want = [w.double() for w in ws]
    bufs = [torch.zeros(s, dtype=torch.float64) for s in shapes]
    most = [w.abs().max() for w in want]
    for _ in range(steps):
        for i, p in enumerate(ps):
            gr = torch.randn(shapes[i], generator=g).to(types[i])
            p.grad = gr.to(dev)
            gr = gr.double() + wd * want[i]
            bufs[i].mul_(mom).add_(gr)
            want[i] -= lr * (gr + mom * bufs[i] if nesterov else bufs[i])
            most[i] = torch.maximum(most[i], want[i].abs().max()
                                    + bufs[i].abs().max())
        opt.step()
    for p, w, b, top, t in zip(ps, want, bufs, most, types):
        st = opt.state[p]
        assert st['momentum_buffer'].dtype == torch.float32
        tol = 10 * 6 * E * float(top)
        off = (st['momentum_buffer'].cpu().double() - b).abs().max()
        assert float(off) <= tol
        got = st['master'] if t == torch.bfloat16 else p.detach()
        assert got.dtype == torch.float32
        off = (got.cpu().double() - w).abs().max()
        assert float(off) <= steps * tol
        assert torch.equal(p.detach(), got.to(t))


@GPU
def test_buffers_of_another_type_are_refused():
    p = torch.zeros(8, dtype=torch.bfloat16, device='cuda')
    f = ops.ext().multi_tensor_momentum
    for buf in (torch.zeros_like(p), torch.zeros(7, device='cuda')):
        with pytest.raises(RuntimeError, match='fp32'):
            f([p], [p.clone()], [buf], 0.1, 0.9, 0.0, False, [])
