"""Softmax cross entropy of a projection onto a large vocabulary.

``linear_cross_entropy(inputs, weight, bias, labels)`` is
``softmax_cross_entropy(inputs @ weight.t() + bias, labels)`` without the
[N, V] logits: for LM1B's 793,470 words and 2,560 tokens they would take
8.1 GB in fp32.  Beside the sampled softmax it gives the exact loss, for
held-out perplexity and for training on the whole vocabulary.

GPU: hand-written MFMA kernels (ops/hip/csrc/linear_ce.hip); the backward
computes the logits again, piece by piece of the vocabulary.  CPU: torch
reference, which does keep them.
"""

import torch

from parallax_amd import ops as _ops

_REDUCTIONS = {'none': 0, 'mean': 1, 'sum': 2}


def _check(inputs, weight, bias, labels, label_smoothing, reduction):
    if reduction not in _REDUCTIONS:
        raise ValueError("linear_cross_entropy: reduction is 'mean', 'sum' "
                         "or 'none', got %r" % (reduction,))
    if not 0.0 <= label_smoothing < 1.0:
        raise ValueError('linear_cross_entropy: label_smoothing in [0, 1) '
                         'expected, got %r' % (label_smoothing,))
    if weight.dim() != 2 or inputs.dim() < 2 \
            or inputs.shape[-1] != weight.shape[1]:
        raise ValueError('linear_cross_entropy: inputs [..., D] and weight '
                         '[V, D] expected, got %s and %s'
                         % (tuple(inputs.shape), tuple(weight.shape)))
    if not weight.numel():
        raise ValueError('linear_cross_entropy: at least one word of one '
                         'value expected, got a weight of %s'
                         % (tuple(weight.shape),))
    if labels.shape != inputs.shape[:-1]:
        raise ValueError('linear_cross_entropy: labels %s expected, got %s'
                         % (tuple(inputs.shape[:-1]), tuple(labels.shape)))
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError('linear_cross_entropy: bias %s expected, got %s'
                         % (tuple(weight.shape[:1]), tuple(bias.shape)))
    for t, name in ((inputs, 'inputs'), (weight, 'weight'), (bias, 'bias')):
        if t is not None and not t.is_floating_point():
            raise TypeError('linear_cross_entropy: %s of type %s'
                            % (name, t.dtype))
    if labels.is_floating_point() or labels.dtype == torch.bool:
        raise TypeError('linear_cross_entropy: labels of type %s'
                        % labels.dtype)


def check_labels(labels, words, ignore_index=-100):
    """Raises IndexError where a label is neither a word nor
    ``ignore_index``.  The loss clamps such labels, since it does not wait
    for the GPU; what reads its result on the host anyway, as a perplexity
    does, asks here first."""
    out = (labels != ignore_index) & ((labels < 0) | (labels >= words))
    if bool(out.any()):
        raise IndexError('label %d outside the vocabulary of %d words'
                         % (int(labels[out][0]), words))


def _wide(t):
    """In 32 bits, or 64 where it has them (on the host alone)."""
    return t.to(torch.promote_types(t.dtype, torch.float32))


def _plain(x, weight, bias, labels, ignore_index, smoothing, reduction):
    live = labels != ignore_index
    # a product with what ignored rows hold would carry it into the gradients
    x = torch.where(live[:, None], _wide(x), 0.0)
    logits = x @ _wide(weight).t()
    if bias is not None:
        logits = logits + bias.to(logits.dtype)
    # labels outside the vocabulary go to its nearest end, as on the GPU
    y = torch.where(live, labels.clamp(0, weight.shape[0] - 1), 0)
    lse = torch.logsumexp(logits, 1)
    losses = lse - logits.gather(1, y[:, None])[:, 0]
    if smoothing:
        losses = (1 - smoothing) * losses + smoothing * (lse - logits.mean(1))
    losses = torch.where(live, losses, torch.zeros_like(losses))
    if reduction == 'none':
        return losses
    total = losses.sum()
    return total / live.sum() if reduction == 'mean' else total


def linear_cross_entropy(inputs, weight, bias, labels, reduction='mean',
                         ignore_index=-100, label_smoothing=0.0):
    """loss[i] = lse_i - (1 - e) z_i[labels_i] - e mean_v z_i[v] with
    z = inputs @ weight.t() + bias and e = label_smoothing.

    inputs [..., D], weight [V, D], bias [V] or None, labels [...] integer.
    Rows whose label is ``ignore_index`` have no loss and no gradient, and
    their inputs are not read; other labels are clamped to the vocabulary.
    'mean' is over the rows that count (NaN where none does).  The loss is
    fp32 (fp64 of fp64 inputs, which the host takes and the GPU refuses): a
    scalar, or the shape of ``labels`` for 'none'; none is negative.
    ``weight`` is
    cast to the type of ``inputs`` where the two differ; under autocast
    both are cast to its type, as a product's operands are.
    """
    _check(inputs, weight, bias, labels, label_smoothing, reduction)
    x = inputs.reshape(-1, inputs.shape[-1])
    if torch.is_autocast_enabled(x.device.type):
        x = x.to(torch.get_autocast_dtype(x.device.type))
    y = labels.reshape(-1).long()
    if weight.dtype != x.dtype:
        weight = weight.to(x.dtype)
    if x.shape[0] == 0:  # no rows: what a sum over nothing is
        z = _wide(x).sum() + _wide(weight[:0]).sum()
        if bias is not None:
            z = z + bias[:0].to(z.dtype).sum()
        if reduction == 'none':
            return (_wide(x).sum(-1) + z).reshape(labels.shape)
        return z / 0 if reduction == 'mean' else z
    if _ops.use_native(x):
        losses = _ops.ext().linear_ce(x, weight, bias, y.contiguous(),
                                      ignore_index, label_smoothing,
                                      _REDUCTIONS[reduction])
    else:
        with torch.autocast(x.device.type, enabled=False):
            losses = _plain(x, weight, bias, y, ignore_index,
                            label_smoothing, reduction)
    return losses.view(labels.shape) if reduction == 'none' else losses
