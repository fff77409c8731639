"""Rotary positions over several axes, in 64 bits, feature by feature."""
import torch


def rotary_axes(x, cos, sin, positions, sections=None, interleaved=True, back=False):
    """x (tokens, heads, 128); cos / sin (rows, dim / 2); positions (axes, tokens) or (tokens,).  float64."""
    positions = positions if positions.dim() == 2 else positions[None]
    half = cos.shape[1]
    axis = [a for a, n in enumerate(sections or (half,)) for _ in range(n)]
    y = x.double().clone()
    for i in range(half):
        at = positions[axis[i]].long().clamp(0, cos.shape[0] - 1)
        c, s = cos[at, i].double()[:, None], sin[at, i].double()[:, None]
        s = -s if back else s
        f0, f1 = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        x0, x1 = x[..., f0].double(), x[..., f1].double()
        y[..., f0], y[..., f1] = x0 * c - x1 * s, x0 * s + x1 * c
    return y
