"""Newton-Schulz orthogonalisation of update matrices.

``newton_schulz(g)`` brings every singular value of ``g / |g|`` near 1 and
keeps the singular vectors: the polar factor of the update, which the Muon
optimizer (optim.Muon) takes its steps along.  Five steps of
s -> a s + b s^3 + c s^5 with the steep coefficients below lift singular
values from 1e-3 of the norm into [0.7, 1.2].

GPU: hand-written MFMA products (ops/hip/csrc/newton_schulz.hip), a batch of
matrices at a time.  CPU: the same products in torch.
"""

import torch

from parallax_amd import ops as _ops

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _plain(g, steps, coefficients, eps):
    """[batch, rows, cols]; norm in 64 bits, products in at least 32."""
    a, b, c = coefficients
    x = g.double()
    norm = x.square().sum((1, 2), keepdim=True).sqrt()
    x = (x / (norm + eps)).to(torch.promote_types(g.dtype, torch.float32))
    flip = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2).contiguous() if flip else x
    for _ in range(steps):
        p = x @ x.transpose(1, 2).contiguous()
        x = a * x + (b * p + c * (p @ p)) @ x
    return (x.transpose(1, 2) if flip else x).to(g.dtype)


def _into(g, out, steps, coefficients, eps, exact):
    """``g`` [batch, rows, cols] into ``out`` (which may be ``g``)."""
    if _ops.use_native(g):
        _ops.ext().newton_schulz(g, out, steps, *coefficients, eps, exact)
    else:
        with torch.autocast(g.device.type, enabled=False):
            out.copy_(_plain(g, steps, coefficients, eps))
    return out


@torch.no_grad()
def newton_schulz(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """g [..., rows, cols] -> the same shape and type, each matrix made
    orthogonal by itself (rows of a wide one, columns of a tall one).

    ``coefficients`` (a, b, c) have to keep singular values of at most 1
    below about 2, as the default does.  No gradient flows through it.
    bf16 results are exact to bf16's rounding.  fp32 ones are as near as
    products in fp32 come, on the GPU too: to about 2e-6 of the norm, to 1e-5
    for large matrices near low rank."""
    if g.dim() < 2:
        raise ValueError('newton_schulz: a matrix or a batch of matrices '
                         'expected, got shape %s' % (tuple(g.shape),))
    if not g.is_floating_point():
        raise TypeError('newton_schulz: floating type expected, got %s'
                        % g.dtype)
    if int(steps) != steps or not 1 <= steps <= 64:
        raise ValueError('newton_schulz: 1 to 64 steps expected, got %r'
                         % (steps,))
    if len(coefficients) != 3:
        raise ValueError('newton_schulz: three coefficients expected')
    if not g.numel():
        return torch.empty_like(g)
    flat = g.detach().reshape(-1, *g.shape[-2:]).contiguous()
    out = _into(flat, torch.empty_like(flat), int(steps), coefficients, eps,
                g.dtype != torch.bfloat16)
    return out.view(g.shape)
