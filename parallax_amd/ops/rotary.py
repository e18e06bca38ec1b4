"""Rotary positions of queries and keys.

``apply_rotary(q, k, cos, sin)`` turns pairs of values of each head by the
angle of the token's place; ``ParallaxRotary`` holds the tables for it,
stretched for contexts longer than the model was trained on where asked.
Scores then depend on the distance of two tokens alone, so a transformer
needs no table of learned positions (models/nmt.py, ``positions='rotary'``).

GPU: one hand-written launch for queries and keys, and one for their
gradients (ops/hip/csrc/rotary.hip).  CPU: the same formula in torch.
"""

import math

import torch
import torch.nn as nn

from parallax_amd import ops as _ops


def _turn(x, cos, sin, interleaved):
    """x [B, T, H, D]; cos and sin [B or 1, T, 1, R/2]."""
    r = 2 * cos.shape[-1]
    y = x[..., :r].float() if x.dtype != torch.float64 else x[..., :r]
    if interleaved:
        u, v = y[..., 0::2], y[..., 1::2]
    else:
        u, v = y[..., :r // 2], y[..., r // 2:]
    u, v = u * cos - v * sin, u * sin + v * cos
    y = torch.stack((u, v), -1).flatten(-2) if interleaved \
        else torch.cat((u, v), -1)
    return torch.cat((y.to(x.dtype), x[..., r:]), -1)


def _last_dense(t):
    return t if t.stride(-1) == 1 else t.contiguous()


def _check(q, k, cos, sin, positions, offset):
    if q.dim() != 4:
        raise ValueError('apply_rotary: q [B, T, H, D] expected, got %s'
                         % (tuple(q.shape),))
    if not q.is_floating_point():
        raise TypeError('apply_rotary: q of type %s' % q.dtype)
    if k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2]
                          or k.shape[3] != q.shape[3]
                          or k.dtype != q.dtype):
        raise ValueError('apply_rotary: k %s of type %s does not match q %s '
                         'of type %s' % (tuple(k.shape), k.dtype,
                                         tuple(q.shape), q.dtype))
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] < 1 \
            or not 2 <= 2 * cos.shape[1] <= q.shape[3]:
        raise ValueError('apply_rotary: tables [places, R/2] with R of at '
                         'most %d expected, got %s and %s'
                         % (q.shape[3], tuple(cos.shape), tuple(sin.shape)))
    if positions is None:
        if offset < 0 or offset + q.shape[1] > cos.shape[0]:
            raise ValueError('apply_rotary: places %d to %d, but the tables '
                             'have %d' % (offset, offset + q.shape[1],
                                          cos.shape[0]))
        return
    if offset:
        raise ValueError('apply_rotary: positions or an offset, not both')
    if positions.is_floating_point() or positions.dtype == torch.bool:
        raise TypeError('apply_rotary: positions of type %s'
                        % positions.dtype)
    if positions.shape not in ((q.shape[1],), tuple(q.shape[:2]),
                               (1, q.shape[1])):
        raise ValueError('apply_rotary: positions [T] or [B, T] expected, '
                         'got %s' % (tuple(positions.shape),))


def apply_rotary(q, k, cos, sin, positions=None, offset=0,
                 interleaved=False):
    """(q', k'), or q' where ``k`` is None.

    q [B, T, H, D], k [B, T, Hk, D] (Hk of its own), in any strides; cos and
    sin [places, R/2] fp32, R <= D: the rest of a head passes through.
    Pairs are (i, i + R/2), or (2i, 2i+1) where ``interleaved``.  Token t of
    a sequence stands at ``positions[b, t]`` (integers [T] or [B, T],
    clamped to the tables) or at ``offset + t``.  No gradient flows to the
    tables."""
    _check(q, k, cos, sin, positions, offset)
    if cos.requires_grad or sin.requires_grad:
        cos, sin = cos.detach(), sin.detach()
    if positions is not None:
        positions = positions.long()
        positions = positions[None] if positions.dim() == 1 else positions
    if _ops.use_native(q):
        cos, sin = cos.float().contiguous(), sin.float().contiguous()
        q = _last_dense(q)
        k = _last_dense(k) if k is not None else None
        out = _ops.ext().rotary(q, k, cos, sin, positions, offset,
                                interleaved)
        return out[0] if k is None else tuple(out)
    if positions is None:
        c, s = (t[offset:offset + q.shape[1]][None, :, None]
                for t in (cos, sin))
    else:
        at = positions.clamp(0, cos.shape[0] - 1)
        c, s = cos[at][:, :, None], sin[at][:, :, None]
    a = _turn(q, c, s, interleaved)
    return a if k is None else (a, _turn(k, c, s, interleaved))


def rotary_tables(rotary_dim, places, base=10000.0, scaling=None, factor=1.0,
                  original_places=None, beta_fast=32.0, beta_slow=1.0,
                  device=None):
    """cos and sin [places, rotary_dim/2] fp32 of angles in 64 bits.

    scaling  None: angle = place base^(-2i/R).
             'linear': places divided by ``factor``.
             'ntk': a larger base, base factor^(R/(R-2)), so that the
             slowest angle is divided by ``factor`` and the fastest stays.
             'yarn': angles that turn less than ``beta_slow`` times within
             ``original_places`` are divided by ``factor``, those that turn
             more than ``beta_fast`` times stay, a ramp over i in between,
             and cos and sin are multiplied by 0.1 ln(factor) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError('rotary_tables: an even rotary_dim expected, got %r'
                         % (rotary_dim,))
    if places < 1:
        raise ValueError('rotary_tables: at least one place expected, got '
                         '%r' % (places,))
    if scaling not in (None, 'linear', 'ntk', 'yarn'):
        raise ValueError("rotary_tables: scaling is None, 'linear', 'ntk' or "
                         "'yarn', got %r" % (scaling,))
    if scaling is not None and not factor >= 1.0:
        raise ValueError('rotary_tables: a factor of at least 1 expected, '
                         'got %r' % (factor,))
    r, scale = rotary_dim, 1.0
    i = torch.arange(0, r, 2, dtype=torch.float64, device=device)
    if scaling == 'ntk' and r > 2:
        base = base * factor ** (r / (r - 2.0))
    inv = base ** (-i / r)
    if scaling == 'linear':
        inv = inv / factor
    elif scaling == 'yarn':
        if not original_places or original_places < 1:
            raise ValueError("rotary_tables: 'yarn' needs original_places")

        def index(turns):  # of the angle that turns so often
            return r * math.log(original_places / (2 * math.pi * turns)) \
                / (2 * math.log(base))

        lo = max(math.floor(index(beta_fast)), 0)
        hi = min(math.ceil(index(beta_slow)), r - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
        scale = 0.1 * math.log(factor) + 1.0
    at = torch.arange(places, dtype=torch.float64, device=device)
    angle = at[:, None] * inv
    return (angle.cos() * scale).float(), (angle.sin() * scale).float()


class ParallaxRotary(nn.Module):
    """The tables of ``rotary_tables`` and the call that uses them:
    ``rotary(q, k, positions=None, offset=0)``.  The tables are no state of
    a checkpoint and stay fp32 under ``.to(torch.bfloat16)``."""

    def __init__(self, head_dim, places, rotary_dim=None, interleaved=False,
                 **scaling):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim > head_dim:
            raise ValueError('ParallaxRotary: rotary_dim %d of a head of %d'
                             % (rotary_dim, head_dim))
        self.interleaved = interleaved
        cos, sin = rotary_tables(rotary_dim, places, **scaling)
        self.register_buffer('cos', cos, persistent=False)
        self.register_buffer('sin', sin, persistent=False)

    def _apply(self, fn, recurse=True):
        tables = self.cos, self.sin
        super()._apply(fn, recurse)
        if self.cos.dtype != torch.float32:  # a change of type: device only
            self.cos, self.sin = (t.to(self.cos.device) for t in tables)
        return self

    def forward(self, q, k=None, positions=None, offset=0):
        return apply_rotary(q, k, self.cos, self.sin, positions, offset,
                            self.interleaved)
