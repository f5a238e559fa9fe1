"""The 4-bit cache from its definition: norm, rotation and entries number by number in float32 with every operation rounded for itself (numpy and Python
on the host), what codes stand for in float64.  Attention over the values: cache_8bit_plain.attend."""
import math

import numpy as np
import torch

GROUP = 32


def bf16_near(x):
    return float(torch.tensor(x, dtype=torch.float32).bfloat16())


def bf16_above(x):
    """The smallest bfloat16 no smaller than x >= 0."""
    y = torch.tensor(x, dtype=torch.float32).bfloat16()
    if float(y) < x:
        y = (y.view(torch.int16) + 1).view(torch.bfloat16)
    return float(y)


def normalised(rows, weight, eps):
    """rows [n, dim] float32: over the root of the mean square plus eps (the mean in float64, the rest float32), times weight."""
    mean = (rows.double().square().sum(-1, keepdim=True) / rows.shape[-1] + eps).float()
    # (numpy's square root is the nearest float32; torch's on the host is now and then its neighbour)
    return rows * torch.from_numpy(np.float32(1.0) / np.sqrt(mean.numpy())) * weight


def turned(rows, cos, sin, rotary, pos, pairs):
    """rows [n, dim] float32 turned by position ``pos``'s angles; every product and sum rounded for itself."""
    out = rows.clone()
    for i in range(rotary // 2):
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + rotary // 2)
        c, s = cos[pos, i], sin[pos, i]
        out[:, a] = rows[:, a] * c - rows[:, b] * s
        out[:, b] = rows[:, a] * s + rows[:, b] * c
    return out


def entry(x):
    """x [dim] float32 -> (codes [dim], steps [groups], bases [groups]); None for codes of an entry that reads as NaN."""
    groups = -(-len(x) // GROUP)
    if not bool((x.abs() < 2.0 ** 96).all()):
        return None, [math.nan] * groups, [math.nan] * groups
    codes, steps, bases, f = [], [], [], np.float32
    for j in range(groups):
        part = [f(v) for v in x[GROUP * j:GROUP * (j + 1)].tolist()]
        lo, hi = min(part), max(part)
        base = f(bf16_near(lo + (hi - lo) * f(8.0 / 15.0)))
        step = f(bf16_above(float(max((hi - base) / f(7.0), (base - lo) / f(8.0)))))
        steps.append(float(step))
        bases.append(float(base))
        codes += [min(max(int(np.rint((v - base) / step)) + 8, 0), 15) if step > 0 else 8 for v in part]
    return codes, steps, bases


def unpack(units, dim):
    """units uint8 [..., 16 groups] -> codes [..., dim]: numbers 32 j + 4 g + n are nibbles n of the (g groups + j)-th two bytes."""
    groups = -(-dim // GROUP)
    codes = torch.zeros(*units.shape[:-1], dim, dtype=torch.int64)
    for d in range(dim):
        j, g, n = d // GROUP, d % GROUP // 4, d % 4
        codes[..., d] = (units[..., 2 * (g * groups + j) + n // 2].long() >> (4 * (n % 2))) & 15
    return codes


def values(units, pairs, dim):
    """What they stand for: units uint8 [..., 16 groups], pairs bfloat16 [..., 2 groups] -> float64 [..., dim]."""
    j = torch.arange(dim) // GROUP
    pairs = pairs.double()
    return (unpack(units, dim) - 8).double() * pairs[..., 2 * j] + pairs[..., 2 * j + 1]
