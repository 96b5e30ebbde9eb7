"""Rotary positions and head norms in 64 bits (numpy), and how far a float32 kernel that rounds
once may be from them."""
from __future__ import annotations

import math

import numpy as np

BF16 = 2.0 ** -8      # half a step of bf16, relative
E4M3 = 2.0 ** -4      # of E4M3
E4M3_SUB = 2.0 ** -10  # half of E4M3's smallest step
# Roundings of 2^-24 each on a float32 value: up to 16 elements added in a lane and six steps of
# a tree, halved by the root (11), the division by the size and eps (1), the root's two ulps
# (4), the weight's sum and two products (3), the rotation's product and sum (2).
F32 = 21 * 2.0 ** -24


def table(positions, rotary, theta=1e4):
    """float32 table (the kernels' input, exact for the reference)."""
    ang = np.arange(positions)[:, None] * theta ** (-np.arange(0, rotary, 2) / rotary)
    return np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)


def pair_index(rotary, interleaved):
    p = np.arange(rotary // 2)
    return (2 * p, 2 * p + 1) if interleaved else (p, p + rotary // 2)


def rotate(x, positions, tab, interleaved=False, inverse=False):
    """(rotated rows [t, h, d], sum of the magnitudes that went into each element)."""
    x = np.asarray(x, np.float64)
    rotary = 2 * tab.shape[1]
    a, b = pair_index(rotary, interleaved)
    ok = (positions >= 0) & (positions < len(tab))
    cs = tab[np.where(ok, positions, 0)].astype(np.float64)
    cos = np.where(ok[:, None], cs[..., 0], 1.0)[:, None]
    sin = np.where(ok[:, None], cs[..., 1], 0.0)[:, None] * (-1 if inverse else 1)
    y, size = x.copy(), np.abs(x)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    size[..., a] = np.abs(x[..., a] * cos) + np.abs(x[..., b] * sin)
    size[..., b] = np.abs(x[..., b] * cos) + np.abs(x[..., a] * sin)
    return y, size


def norm(x, weight, eps, offset=0.0):
    x = np.asarray(x, np.float64)
    if weight is None:
        return x
    inv = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return x * inv * (np.asarray(weight, np.float64) + offset)


def row_scale(rows):
    """Smallest power of two P >= 2^-126 with max |row| <= 448 P; 0 for a row of zeros."""
    amax = np.abs(rows).max(-1)
    out = np.zeros(amax.shape)
    for i in np.ndindex(amax.shape):
        if amax[i] > 0:
            out[i] = 2.0 ** max(-126, math.ceil(math.log2(amax[i] / 448)))
    return out


def assert_bf16(got, want, size, what):
    got = np.asarray(got, np.float64)
    bound = np.abs(want) * BF16 + size * F32 * (1 + BF16) + 1e-38
    bad = np.argwhere(~(np.abs(got - want) <= bound))
    assert not len(bad), f"{what}: {len(bad)} values off, first {bad[0]}: {got[tuple(bad[0])]} " \
                         f"for {want[tuple(bad[0])]}"


def assert_fp8(values, scales, want, size, what):
    """values: stored codes as numbers (without the scale); scales, want [..., rows(, d)]."""
    p = row_scale(want)
    close = np.abs(scales / np.where(p > 0, p, 1.0) - 1.0) < 1e-9
    close |= (p == 0) & (scales == 0)
    # the next power where the largest element lies within float32's error of the border
    edge = np.abs(want).max(-1) / np.where(p > 0, p, 1.0)
    at_edge = (np.abs(edge / 448 - 1) < 64 * F32) | (np.abs(edge / 224 - 1) < 64 * F32)
    assert np.all(close | at_edge), f"{what}: scales"
    s = scales[..., None]
    bound = np.abs(want) * E4M3 + s * E4M3_SUB + size * F32 * (1 + E4M3)
    bad = np.argwhere(~(np.abs(values * s - want) <= bound))
    assert not len(bad), f"{what}: {len(bad)} values off, first {bad[0]}"
