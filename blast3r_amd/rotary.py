"""Rotary positions of a transformer's queries and keys on the device (``ba_rotary``, libba_hip.so).

The depth and matching networks in front of a bundle adjustment place the patches of an image by row and column (two or
three axes, each with its part of the head; the reference has an extension for it, src/blast3r/extensions/curope, with
which parity is unpinned); sequence models place tokens by one position, with pairs half a head apart or side by side, and
may scale their frequencies for long contexts.  ``Rotary`` holds one such choice::

    rot = Rotary(64, axes=2)                    # a head of 64, rows in its first half, columns in the other
    q, k = rot(positions, q, k)                 # one launch for both; differentiable

Nothing here falls back to torch: the rotation runs in libba_hip.so on device tensors.
"""
import math

import torch

from ._lib import BaRotaryArgs, dual_level, has_tangent, launch, lib, overlaps, written

__all__ = ['Rotary', 'rotary_frequencies']

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def rotary_frequencies(n, base=10000.0, scaling=None):
    """(angle per position of each of the n / 2 pairs of a section of n elements, factor of the result), 64 bits.

    base^(-2p/n) for pair p, and with ``scaling``
      dict(kind='linear', factor=s)   divided by s: positions are squeezed into the trained range;
      dict(kind='base', factor=s)     with base * s^(n / (n - 2)): the slowest pair turns s times slower, the fastest as
                                      before;
      dict(kind='ramp', factor=s, length=L, fast=32, slow=1)
                                      by the turns that a pair makes over the trained length L: as before from `fast`
                                      turns on, divided by s up to `slow`, a mixture in between; the result is
                                      multiplied by 0.1 ln s + 1.
    """
    if n < 2 or n % 2:
        raise ValueError(f'rotary: a section must be whole pairs, got {n} elements')
    if not base > 0:
        raise ValueError(f'rotary: base must be positive, got {base}')
    kind = scaling['kind'] if scaling else None
    s = float(scaling['factor']) if scaling else 1.0
    if kind not in (None, 'linear', 'base', 'ramp') or not s >= 1.0:
        raise ValueError(f'rotary: unknown scaling {scaling!r} (linear, base or ramp, by a factor of at least 1)')
    if kind == 'base':
        base = base * s ** (n / max(n - 2, 1))
    f = [base ** (-2.0 * p / n) for p in range(n // 2)]
    if kind == 'linear':
        f = [x / s for x in f]
    if kind == 'ramp':
        fast, slow = float(scaling.get('fast', 32.0)), float(scaling.get('slow', 1.0))
        if not fast > slow:
            raise ValueError(f'rotary: fast must exceed slow, got {fast} and {slow}')
        keep = [min(1.0, max(0.0, (scaling['length'] * x / (2 * math.pi) - slow) / (fast - slow))) for x in f]
        f = [g * x + (1.0 - g) * x / s for g, x in zip(keep, f)]
        return f, 0.1 * math.log(s) + 1.0
    return f, 1.0


class _Turn(torch.autograd.Function):
    """The rotation with its gradient, which is the opposite rotation (and so differentiable in turn), and its
    forward-mode derivative, which is the rotation of the tangents."""

    @staticmethod
    def forward(ctx, rot, positions, inverse, *xs):
        ctx.rot, ctx.inverse, ctx.shapes = rot, inverse, [x.shape for x in xs]
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        return rot._run(positions, xs, None, inverse)

    @staticmethod
    def backward(ctx, *grads):
        positions, = ctx.saved_tensors
        need = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[3 + i]]
        out = [None] * len(grads)
        if need:
            gs = [g if g.stride(-1) == 1 else g.contiguous() for g in (grads[i] for i in need)]
            for i, y in zip(need, _Turn.apply(ctx.rot, positions, not ctx.inverse, *gs)):
                out[i] = y
        return (None, None, None, *out)

    @staticmethod
    def jvp(ctx, rot, positions, inverse, *ts):
        """Tangents turn as their tensors do; without one the tangent is zero."""
        positions, = ctx.saved_tensors
        have = [i for i, t in enumerate(ts) if t is not None]
        like = ts[have[0]]
        ys = _Turn.apply(ctx.rot, positions, ctx.inverse, *(ts[i] if ts[i].stride(-1) == 1 else ts[i].contiguous() for i in have))
        out = [torch.zeros(shape, dtype=like.dtype, device=like.device) if t is None else t for t, shape in zip(ts, ctx.shapes)]
        for i, y in zip(have, ys):
            out[i] = y
        return tuple(out)


def _fixed(name):
    return property(lambda self: getattr(self, name))


class Rotary:
    """Rotary positions of heads of ``head_dim`` elements.

    rotary_dim  the first elements of a head that are rotated (default: all); the rest is copied
    base        of the frequencies base^(-2p/n)
    layout      'half': pair p of a section of n is (p, p + n/2); 'interleaved': (2p, 2p + 1)
    axes        coordinates of a position; each rotates rotary_dim / axes elements
    scaling     see ``rotary_frequencies``

    These, and ``frequencies``, ``factor`` and ``turns`` that come of them, stay as they are: another choice is another
    ``Rotary``.
    """

    head_dim, rotary_dim, layout, axes = _fixed('_head_dim'), _fixed('_rotary_dim'), _fixed('_layout'), _fixed('_axes')
    frequencies, factor, turns, device = _fixed('_frequencies'), _fixed('_factor'), _fixed('_turns'), _fixed('_device')

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, layout='half', axes=1, scaling=None, device='cuda'):
        part = head_dim if rotary_dim is None else rotary_dim
        if layout not in ('half', 'interleaved'):
            raise ValueError(f"rotary: layout must be 'half' or 'interleaved', got {layout!r}")
        if axes < 1 or part < 2 or part > head_dim or part % (2 * axes):
            raise ValueError(f'rotary: {part} of {head_dim} elements are not whole pairs for each of {axes} axes')
        if layout == 'interleaved' and head_dim % 2:
            raise ValueError('rotary: an interleaved head must be even')
        self._head_dim, self._rotary_dim, self._layout, self._axes = head_dim, part, layout, axes
        self._frequencies, self._factor = rotary_frequencies(part // axes, base, scaling)
        # turns per position in units of 2^-64 (a frequency of 2 pi or more wraps, as its angle does)
        turns = [round(x / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for x in self._frequencies]
        self._turns = torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns], dtype=torch.int64, device=device)
        if not self._turns.is_cuda:
            raise RuntimeError('rotary needs a GPU (it runs in libba_hip.so)')
        self._device = self._turns.device
        # the fields of every call
        self._args = BaRotaryArgs(n_x=1, B=1, dim=head_dim, part=part, axes=axes, interleaved=layout == 'interleaved',
                                  factor=self._factor)
        self._call = lib().ba_rotary

    def __call__(self, positions, *xs, out=None, inverse=False):
        """The rotated tensors of ``xs``: one or two of shape (tokens, heads, head_dim) or (B, T, heads, head_dim), fp32,
        fp16 or bf16, any strides with contiguous elements; a single tensor comes back as itself, two as a tuple.

        positions   int32 or int64, the tokens' shape ((T,) serves every batch), with more than one axis a last
                    dimension of ``axes``
        out         tensors to write to, one for each x (x itself rotates in place; another one may not overlap either x);
                    not differentiable, and refused where gradients are recorded and one of them requires one
        inverse     rotate by the opposite angles
        """
        if not 1 <= len(xs) <= 2:
            raise ValueError(f'rotary: one or two tensors at a time, got {len(xs)}')
        if torch.is_grad_enabled() and (xs[0].requires_grad or xs[-1].requires_grad) or dual_level() and has_tangent(*xs):
            if out is not None:
                raise ValueError('rotary: out cannot be given where gradients are recorded')
            ys = _Turn.apply(self, positions, bool(inverse), *xs)
        else:
            ys = self._run(positions, xs, out, inverse)
        return ys if len(xs) == 2 else ys[0]

    def _run(self, positions, xs, out, inverse):
        x = xs[0]
        dtype, shape, dev = x.dtype, x.shape, self._device
        lead = shape[:-2]
        n_lead = len(lead)
        if n_lead != 1 and n_lead != 2:
            raise ValueError(f'rotary: tensors are (tokens, heads, dim) or (B, T, heads, dim), got {tuple(shape)}')
        code = DTYPES.get(dtype)
        if code is None:
            raise ValueError(f'rotary: fp32, fp16 or bf16 tensors, got {dtype}')
        wide = positions.dtype is torch.int64
        if not wide and positions.dtype is not torch.int32 or positions.device != dev:
            raise ValueError(f'rotary: positions must be int32 or int64 on {dev}')
        p_lead, p_stride = positions.shape, positions.stride()
        if self._axes > 1:
            if len(p_lead) < 2 or p_lead[-1] != self._axes:
                raise ValueError(f'rotary: positions need a last dimension of {self._axes} axes, got {tuple(p_lead)}')
            p_lead = p_lead[:-1]
        if p_lead != lead and (n_lead == 1 or p_lead != lead[1:]):
            raise ValueError(f'rotary: positions of shape {tuple(positions.shape)} for tokens {tuple(lead)}')
        if out is None:
            ys = [torch.empty_like(x) for x in xs]
            for i, y in enumerate(ys):
                if y.stride()[-1] != 1:                     # expanded tensors may come back in another order
                    ys[i] = torch.empty(y.shape, dtype=dtype, device=dev)
        else:
            ys = list(out) if isinstance(out, (tuple, list)) else [out]
            if len(ys) != len(xs):
                raise ValueError(f'rotary: {len(ys)} outputs for {len(xs)} tensors')
            for x, y in zip(xs, ys):
                if y.shape != x.shape or y.dtype != x.dtype or y.device != x.device or y.stride(-1) != 1:
                    raise ValueError('rotary: an output must be like its tensor, with contiguous elements of a head')
                if y.requires_grad and torch.is_grad_enabled() or dual_level() and has_tangent(y):
                    raise ValueError('rotary: out must not require a gradient where gradients are recorded, nor have a tangent')
                if overlaps(y, x):
                    raise ValueError('rotary: out overlaps itself or, not in its place, the tensor that it is the rotation of')
            if len(xs) == 2 and x.numel():
                at = ys[0].data_ptr(), ys[1].data_ptr()
                if at[0] == at[1] or at[0] == xs[1].data_ptr() or at[1] == xs[0].data_ptr():
                    raise ValueError('rotary: an out overlaps the other tensor or its out')
        a = BaRotaryArgs.from_buffer_copy(self._args)
        t, y = xs[0], ys[0]
        xs_, ys_ = self._strides(t, lead, dtype), y.stride()
        a.x0, a.y0, a.heads0 = t.data_ptr(), y.data_ptr(), t.shape[-2]
        a.x_sh0, a.x_st0, a.y_sh0, a.y_st0 = xs_[-2], xs_[-3], ys_[-2], ys_[-3]
        if n_lead == 2:
            a.x_sb0, a.y_sb0, a.B = xs_[0], ys_[0], lead[0]
        if len(xs) == 2:
            t, y = xs[1], ys[1]
            xs_, ys_ = self._strides(t, lead, dtype), y.stride()
            a.x1, a.y1, a.heads1 = t.data_ptr(), y.data_ptr(), t.shape[-2]
            a.x_sh1, a.x_st1, a.y_sh1, a.y_st1 = xs_[-2], xs_[-3], ys_[-2], ys_[-3]
            a.n_x = 2
            if n_lead == 2:
                a.x_sb1, a.y_sb1 = xs_[0], ys_[0]
        a.dtype, a.T, a.turns = code, lead[-1], self._turns.data_ptr()
        if inverse:
            a.inverse = 1
        if wide:
            a.pos_int64 = 1
        a.positions, a.pos_st = positions.data_ptr(), p_stride[len(p_lead) - 1]
        if self._axes > 1:
            a.pos_sa = p_stride[-1]
        if len(p_lead) == 2:
            a.pos_sb = p_stride[0]
        if a.T and a.B:
            launch(self._call, a, dev)
            if out is not None:
                written(ys)
        return tuple(ys)

    def _strides(self, t, lead, dtype):
        shape, stride = t.shape, t.stride()
        if (len(shape) != len(lead) + 2 or shape[:-2] != lead or shape[-1] != self._head_dim or shape[-2] == 0 or
                t.dtype is not dtype or t.device != self._device):
            raise ValueError(f'rotary: tensors must share tokens, type and device, with heads of {self._head_dim}: got '
                             f'{tuple(shape)} {t.dtype} on {t.device}')
        if stride[-1] != 1:
            raise ValueError('rotary: the elements of a head must be contiguous')
        return stride
