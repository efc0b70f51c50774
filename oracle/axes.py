"""Rotary embedding at positions of several axes, in 64 bits. TEST INFRASTRUCTURE ONLY.

Pair i of a row turns by t = position[axis(i)] * scale * freq(i), as the complex number x + i y times e^(i t). The
operator has no counterpart in the reference; on one axis it is oracle/rope.py with exact angles.
"""

from __future__ import annotations

import numpy as np


def pair_axes(sections, interleaved: bool):
    """The axis of every pair: section by section, or dealt in turn to the axes that still lack pairs."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def freqs(dims: int, sections, base: float, interleaved: bool, restart: bool):
    axes = pair_axes(sections, interleaved)
    seen = [0] * len(sections)
    out = []
    for i, a in enumerate(axes):
        e = seen[a] / sections[a] if restart else i / (dims // 2)
        seen[a] += 1
        out.append(base ** -e)
    return np.array(axes), np.array(out, np.float64)


def rotate(x: np.ndarray, positions: np.ndarray, dims: int, sections, traditional=False, base=10000.0, scale=1.0,
           interleaved=False, restart=False):
    """x [B, H, L, D] float64, positions int [axes, B, L] -> the rotated rows, float64, not rounded; and |x| + |y| of
    every element's pair (what its error scales with)."""
    axes, f = freqs(dims, sections, base, interleaved, restart)
    t = np.transpose(np.asarray(positions, np.float64)[axes], (1, 2, 0)) * (scale * f)  # [B, L, pairs]
    turn = np.exp(1j * t)[:, None]
    out = np.array(x, np.float64)
    size = np.abs(out)
    a, b = (slice(0, dims, 2), slice(1, dims, 2)) if traditional else (slice(0, dims // 2), slice(dims // 2, dims))
    z = (out[..., a] + 1j * out[..., b]) * turn
    total = size[..., a] + size[..., b]
    out[..., a], out[..., b] = z.real, z.imag
    size[..., a] = size[..., b] = total
    return out, size
