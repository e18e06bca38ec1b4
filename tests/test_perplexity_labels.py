"""The perplexity tools refuse labels that are no words of the model's
vocabulary: clamped, they would give a plausible perplexity."""

import importlib.util
import os
import sys

import numpy as np
import pytest
import torch

from parallax_amd.models.lm1b import LM1BModel
from parallax_amd.models.skip_thoughts import SkipThoughts, synthetic_batch
from parallax_amd.ops.linear_ce import check_labels

GPU = pytest.mark.gpu
DEVICES = ['cpu', pytest.param('cuda', marks=GPU)]
EXAMPLES = os.path.join(os.path.dirname(os.path.dirname(
    os.path.abspath(__file__))), 'examples')


def _tool(*path):
    path = os.path.join(EXAMPLES, *path)
    sys.path.insert(0, os.path.dirname(path))
    try:
        spec = importlib.util.spec_from_file_location(
            os.path.splitext(os.path.basename(path))[0], path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    finally:
        sys.path.pop(0)
    return mod


class _Stream:
    """Windows of words below 50, one of which has the given label."""

    def __init__(self, label):
        self.label = label

    def iterate_forever(self, batch, steps):
        rng = np.random.RandomState(0)
        while True:
            x = rng.randint(0, 50, (batch, steps)).astype(np.int64)
            y = rng.randint(0, 50, (batch, steps)).astype(np.int64)
            y[1, 2] = self.label
            yield x, y, np.ones_like(y)


@pytest.mark.parametrize('dev', DEVICES)
def test_lm1b(dev):
    torch.manual_seed(0)
    model = LM1BModel(vocab_size=50, emb_dim=16, state_size=32,
                      proj_size=16, num_sampled=8, min_partitions=2).to(dev)
    run = _tool('lm1b', 'lm1b_eval.py').evaluate_perplexity

    def go(label):
        return run(model, _Stream(label), batch_size=3, num_steps=4,
                   max_batches=2, device=dev)

    assert go(49)[1] == 24
    for label in (50, -1):
        with pytest.raises(IndexError, match='vocabulary'):
            go(label)


@pytest.mark.parametrize('dev', DEVICES)
def test_skip_thoughts(dev):
    torch.manual_seed(0)
    model = SkipThoughts(vocab=64, emb_dim=16, units=32, num_sampled=8,
                         min_partitions=2).to(dev)
    run = _tool('skip_thoughts', 'track_perplexity.py').evaluate_perplexity
    batch = [t.to(dev) for t in synthetic_batch(4, 6, vocab=64)]
    assert run(model, [batch])[1] == 2 * 4 * 5
    batch[2][1, -1] = 64
    with pytest.raises(IndexError, match='vocabulary'):
        run(model, [batch])


def test_check_labels():
    y = torch.tensor([[0, 9], [-100, 3]])
    check_labels(y, 10)
    with pytest.raises(IndexError, match='label 9 .* 9 words'):
        check_labels(y, 9)
    with pytest.raises(IndexError, match='label -100'):
        check_labels(y, 10, ignore_index=3)
    check_labels(y[:0], 1)
