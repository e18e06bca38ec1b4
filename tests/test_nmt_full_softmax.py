"""The NMT transformer with rotary positions, the full-vocabulary loss and
Muon: the operators run together as a user's program has them."""

import os
import subprocess
import sys

import pytest
import torch

import parallax_amd
from parallax_amd.config import ParallaxConfig
from parallax_amd.models import nmt
from parallax_amd.tagging import classify_params, split_dense_sparse

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GPU = pytest.mark.gpu
DEVICES = ['cpu', pytest.param('cuda', marks=GPU)]


@pytest.fixture(autouse=True)
def _destroy_pg():
    yield
    import torch.distributed as dist
    if dist.is_initialized():
        dist.destroy_process_group()


def _env(monkeypatch, port):
    monkeypatch.setenv('WORLD_SIZE', '1')
    monkeypatch.setenv('RANK', '0')
    monkeypatch.setenv('LOCAL_RANK', '0')
    monkeypatch.setenv('MASTER_ADDR', '127.0.0.1')
    monkeypatch.setenv('MASTER_PORT', str(port))


def _graph(**kw):
    torch.manual_seed(0)
    g = nmt.build_nmt_graph(
        arch='transformer', src_vocab=90, tgt_vocab=110, d_model=32,
        heads=4, ffn=64, enc_layers=2, dec_layers=2, min_partitions=2,
        optimizer='muon', positions='rotary', softmax='full',
        label_smoothing=0.1, **kw)
    for m in g.model.modules():
        if isinstance(m, nmt._Block):
            m.p = 0.0
    return g


def _model(dev='cpu'):
    return _graph().model.to(dev)


@pytest.mark.parametrize('dev', DEVICES)
def test_session(monkeypatch, free_port, dev):
    if dev == 'cpu' and torch.cuda.is_available():
        pytest.skip('the session takes the GPU')
    _env(monkeypatch, free_port)
    sess, *_ = parallax_amd.parallel_run(
        lambda: _graph(use_bf16=False), None,
        parallax_config=ParallaxConfig(run_option='HYBRID'))
    sparse, dense = split_dense_sparse(classify_params(sess.graph.model))
    assert {gi.name for gi in sparse} == {'src_emb.weight', 'tgt_emb.weight'}
    assert 'out_w' in {gi.name for gi in dense}
    assert 'pos' not in {gi.name for gi in dense}
    model, opt = sess.graph.model, sess.graph.optimizer
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    batch = nmt.synthetic_batch(4, 6, 7, 90, 110, device=dev)
    for _ in range(3):
        out = sess.run(batch)
        assert torch.isfinite(out['loss'])
    for n, p in model.named_parameters():
        assert not torch.equal(p, before[n]) and torch.isfinite(p).all(), n
        muon = 'momentum_buffer' in opt.state[p]
        assert muon == (p.dim() == 2 and n.split('.')[0] in ('enc', 'dec'))
    sess.close()


@GPU
def test_gradients_of_the_gpu_are_those_of_the_cpu():
    """fp32 on both sides: sums of at most 110 terms through about 20 layers
    of products, each off by some 2^-24 of its terms' magnitudes and passed
    on by maps that do not grow errors much: 2^-24 * 110 * 20 = 1.3e-4 of a
    gradient's norm, taken four times for what they do grow."""
    cpu, gpu = _model(), _model('cuda')
    src, tin, tout = nmt.synthetic_batch(4, 9, 7, 90, 110)
    tout[0, 4:] = -100
    cpu(src, tin, tout).backward()
    gpu(src.cuda(), tin.cuda(), tout.cuda()).backward()
    for (n, p), q in zip(cpu.named_parameters(), gpu.parameters()):
        a, b = (t.to_dense() if t.layout != torch.strided else t
                for t in (p.grad, q.grad.cpu()))
        assert float((a - b).norm()) <= 4 * 1.3e-4 * float(a.norm()), n


def test_gradient_against_differences():
    """Along the gradient, in fp32: the loss of about 5 is off by some 100
    roundings of 2^-24 of it, 3e-5, which over 2h = 2^-5 is 1e-3; the third
    derivative's share was seen to be below that by halving h."""
    m = _model()
    batch = nmt.synthetic_batch(4, 6, 7, 90, 110)
    ps = [p for n, p in m.named_parameters() if 'emb' not in n]
    m(*batch).backward()
    norm = float(sum(p.grad.double().square().sum() for p in ps)) ** 0.5
    to = [p.grad / norm for p in ps]

    def at(h):
        with torch.no_grad():
            for p, t in zip(ps, to):
                p.add_(t, alpha=h)
            out = float(m(*batch))
            for p, t in zip(ps, to):
                p.sub_(t, alpha=h)
        return out

    wide, near = ((at(h) - at(-h)) / (2 * h) for h in (2.0 ** -6, 2.0 ** -7))
    third = abs(wide - near) * 4 / 3
    assert abs(wide - norm) < third + 2e-3, (wide, near, norm)
    assert third + 2e-3 < 0.1 * norm


@GPU
def test_graphed_session_is_the_eager_one(monkeypatch, free_port):
    _env(monkeypatch, free_port)
    batches = [nmt.synthetic_batch(8, 16, 16, 90, 110, device='cuda')
               for _ in range(8)]
    seen = []
    for graphed in (False, True):
        sess, *_ = parallax_amd.parallel_run(
            lambda: _graph(use_bf16=True, pure_bf16=True), None,
            parallax_config=ParallaxConfig(run_option='HYBRID'))
        for i, b in enumerate(batches):
            if graphed and i == 2:
                sess.enable_cuda_graph(b)
            out = sess.run(b)
            assert torch.isfinite(out['loss'])
        seen.append({n: p.detach().float().clone()
                     for n, p in sess.graph.model.named_parameters()})
        sess.close()
        import torch.distributed as dist
        if dist.is_initialized():
            dist.destroy_process_group()
    for n in seen[0]:
        # bf16 gradients of sums in another order (the embeddings' rows are
        # added up with atomics): a step's direction may differ by 2^-8 of
        # it; eight steps of at most 0.02 * 2 each in a matrix's values
        d = (seen[0][n] - seen[1][n]).norm()
        assert float(d) <= 0.05 * float(seen[0][n].norm()) + 1e-3, n


def test_decoding_runs_with_both_options():
    m = _model()
    m.eval()
    src = torch.randint(3, 90, (2, 5))
    a = m.greedy_decode(src, max_len=6)
    b = m.beam_decode(src, beam_width=1, max_len=6)
    assert a == b
    with pytest.raises(ValueError, match='places'):
        m.encode(torch.zeros(1, 513, dtype=torch.long))


def test_options_are_checked():
    kw = dict(src_vocab=20, tgt_vocab=20, d_model=16, heads=2, ffn=16,
              enc_layers=1, dec_layers=1, min_partitions=1)
    with pytest.raises(ValueError, match='positions'):
        nmt.NMTTransformer(positions='sine', **kw)
    with pytest.raises(ValueError, match='softmax'):
        nmt.NMTTransformer(softmax='hard', **kw)
    with pytest.raises(ValueError, match='label_smoothing'):
        nmt.NMTTransformer(label_smoothing=0.1, **kw)
    with pytest.raises(ValueError, match='optimizer'):
        nmt.build_nmt_graph(optimizer='lamb', **kw)
    with pytest.raises(ValueError, match='transformer'):
        nmt.build_nmt_graph(arch='gnmt', softmax='full')


def test_driver_runs():
    cmd = [sys.executable,
           os.path.join(REPO, 'examples', 'nmt',
                        'nmt_distributed_driver.py'), '--max_steps', '2',
           '--batch_size', '2', '--src_len', '5', '--tgt_len', '5',
           '--d_model', '16', '--heads', '2', '--ffn', '16', '--layers', '1',
           '--log_frequency', '1', '--optimizer', 'muon', '--positions',
           'rotary', '--softmax', 'full', '--label_smoothing', '0.1']
    env = dict(os.environ, WORLD_SIZE='1', RANK='0', LOCAL_RANK='0',
               MASTER_ADDR='127.0.0.1', MASTER_PORT='29583',
               PARALLAX_RUN_OPTION='HYBRID')
    out = subprocess.run(cmd, capture_output=True, text=True, timeout=300,
                         env=env)
    assert out.returncode == 0, out.stderr[-2000:]
    assert 'loss' in out.stdout + out.stderr
