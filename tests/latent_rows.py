"""Rows of a latent cache in 4 and 8 bits, value by value from their description: plain Python and 64-bit torch, without the package's code."""
import math
from fractions import Fraction

import torch

R = 64


def row_bytes(L, bits):
    return (L * bits // 8 + 2 * R + L // (16 if bits == 4 else 32) + 15) // 16 * 16


def nearest(x: Fraction, grid) -> Fraction:
    """The closest of an ascending grid; of two, the one with the even place."""
    best = min(range(len(grid)), key=lambda i: (abs(grid[i] - x), i % 2))
    return grid[best]


def e4m3():
    mags = [Fraction(f, 512) for f in range(8)] + [Fraction(8 + f) * Fraction(2) ** (e - 10) for e in range(1, 16) for f in range(8) if (e, f) != (15, 7)]
    return [-m for m in reversed(mags[1:])] + mags


def group_values(y, bits):
    """What one group of finite numbers reads back as, in exact arithmetic."""
    y = [Fraction(float(v)) for v in y]
    top = max(abs(v) for v in y)
    if bits == 4:
        steps = [Fraction(8 + f, 8) * Fraction(2) ** e for e in range(-20, 11) for f in range(8)]
        s = nearest(top / 7, steps)
        return [s * min(max(nearest(v / s, [Fraction(c) for c in range(-300, 301)]) if abs(v / s) < 300 else (7 if v > 0 else -7), -7), 7) for v in y]
    k = next((k for k in range(-15, 8) if top <= 448 * Fraction(2) ** k), 7)
    grid = e4m3()
    return [nearest(v / Fraction(2) ** k, grid) * Fraction(2) ** k for v in y]


def unpack(raw, L, bits):
    """Bytes of rows [n, row_bytes] (uint8) -> their values [n, L + R] in 64 bits, NaN for groups that say so."""
    raw = raw.cpu()
    per = 2 if bits == 4 else 1
    out = torch.empty(raw.shape[0], L + R, dtype=torch.float64)
    n = L * bits // 8
    for e in range(L):
        chunk, half, j = e // 64, e % 64 // 32, (e % 32) // 16 if bits == 4 else 0
        byte = raw[:, n + 2 * R + half * (L // 64) * per + chunk * per + j].long()
        if bits == 4:
            nib = (e % 8) // 2 + 4 * (e % 2)
            c = (raw[:, e // 8 * 4 + nib // 2].long() >> (4 * (nib % 2))) & 15
            v = (c - 8).double() * (8 + byte % 8).double() * torch.pow(2.0, (byte // 8).double() - 23)
        else:
            c = raw[:, e].long()
            ex, fr = (c >> 3) & 15, (c & 7).double()
            v = torch.where(ex > 0, (8 + fr) * torch.pow(2.0, ex.double() - 10), fr / 512) * (1 - 2 * (c >> 7)).double() * torch.pow(2.0, byte.double() - 127)
        out[:, e] = torch.where(byte == 255, math.nan, v)
    out[:, L:] = raw[:, n:n + 2 * R].contiguous().view(torch.bfloat16).double()
    return out


def normed(kva, w, L, eps):
    x = kva[:, :L].double()
    return x * (1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)) * (1 + w.double())


def rotated(x, pos, inv):
    ang = (pos.double()[:, None] * inv.double()[None]).view(len(pos), *([1] * (x.dim() - 2)), R // 2)
    a, b = x[..., :R // 2].double(), x[..., R // 2:].double()
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)


def attend(q, keys, L, scale):
    """One row: q [heads, L + R], keys [n, L + R], all in 64 bits -> [heads, L]."""
    if not len(keys):
        return torch.zeros(q.shape[0], L, dtype=torch.float64)
    return torch.softmax(q @ keys.t() * scale, -1) @ keys[:, :L]
