"""Rotary positions by plain numpy, for the tests: angles in 80 bits (exact
modulo a turn to about 2^-30 at 2^31 positions), frequencies from the
published formulas."""
import math

import numpy as np

LD = np.longdouble
TWO_PI = LD("6.283185307179586476925286766559005768")


def frequencies(dim, theta, scaling=None):
    """(radians a position [dim / 2], amplitude), one pair at a time."""
    kind, *args = scaling or ("plain",)
    out = []
    for i in range(dim // 2):
        f = theta ** (-2.0 * i / dim)
        if kind == "linear":
            f = f / args[0]
        elif kind == "base":
            f = (theta * args[0] ** (dim / (dim - 2.0))) ** (-2.0 * i / dim) if dim > 2 else 1.0
        elif kind in ("parts", "bands"):
            factor, original, low, high = args if len(args) == 4 else (*args, 1.0, 32.0 if kind == "parts" else 4.0)
            if kind == "bands":
                keep = (original / (2 * math.pi / f) - low) / (high - low)
            else:
                index = lambda turns: dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
                first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), dim - 1)
                keep = 1.0 - (i - first) / max(last - first, 0.001)
            keep = min(max(keep, 0.0), 1.0)
            f = f * keep + f / factor * (1.0 - keep)
        out.append(f)
    return np.array(out), 0.1 * math.log(args[0]) + 1.0 if kind == "parts" else 1.0


def cos_sin(positions, freqs, amplitude):
    """amplitude cos, amplitude sin [rows][pairs], in 80 bits."""
    turns = np.asarray(positions, LD)[:, None] * (np.asarray(freqs, LD) / TWO_PI)[None]
    angle = (turns - np.round(turns)) * TWO_PI
    return LD(amplitude) * np.cos(angle), LD(amplitude) * np.sin(angle)


def halves(dim, layout):
    """The indices of the pairs' firsts and seconds."""
    n = dim // 2
    return (np.arange(n), np.arange(n) + n) if layout == "half" else (2 * np.arange(n), 2 * np.arange(n) + 1)


def turn(x, positions, freqs, amplitude=1.0, layout="half", transposed=False):
    """x [rows][heads][d] turned, in 80 bits."""
    c, s = (v[:, None] for v in cos_sin(positions, freqs, amplitude))
    a, b = halves(2 * len(freqs), layout)
    y = np.asarray(x, LD).copy()
    xa, xb = y[..., a].copy(), y[..., b].copy()
    s = -s if transposed else s
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y


def turn32(x, positions, freqs, amplitude=1.0, layout="half"):
    """The same by the 32-bit rule: f32 cosines, every product and sum rounded."""
    c, s = (v.astype(np.float32)[:, None] for v in cos_sin(positions, freqs, amplitude))
    a, b = halves(2 * len(freqs), layout)
    y = np.asarray(x, np.float32).copy()
    xa, xb = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y
