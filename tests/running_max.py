"""Scores at which the running maximum of tree attention has to move, worked
out in 32 bits on the CPU."""
from __future__ import annotations

import numpy as np

F = np.float32
LOG2E = F(1.4426950408889634)
HEADROOM = F(8.0)


def step(x, n):
    """``x`` moved by ``n`` representable numbers."""
    for _ in range(abs(n)):
        x = np.nextafter(x, F(np.inf if n > 0 else -np.inf), dtype=F)
    return x


def at_headroom(s0, scale_log2, n):
    """A score ``n`` steps beside the one that lies the headroom above ``s0``."""
    return step(F(s0 + F(HEADROOM / scale_log2)), n)


def split_window(s0, scale_log2):
    """A score that lies more than the headroom above ``s0`` if the difference
    of the scaled scores is rounded once, and not if the scaled score and its
    limit are each rounded before they are compared; None where none is found."""
    m = F(s0 * scale_log2)
    limit = F(m + HEADROOM)
    s = F(np.float64(limit) / np.float64(scale_log2))
    for n in range(-6, 7):
        c = step(s, n)
        once = F(np.longdouble(c) * np.longdouble(scale_log2) - np.longdouble(m))
        if once > HEADROOM and not F(c * scale_log2) > limit:
            return c
    return None
