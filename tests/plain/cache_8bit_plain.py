"""The 8-bit cache, attention over it and the scoring of tokens, from their definitions, one request, block and row at a time in float64."""
import math

import torch


def rotated(x, cos, sin, rotary, pos):
    """x [heads, dim] (float64): numbers d and d + rotary/2 of every head turned by position ``pos``'s angle."""
    y = x.clone()
    if rotary:
        half = rotary // 2
        c, s = cos[pos].double(), sin[pos].double()
        lo, hi = x[:, :half], x[:, half:rotary]
        y[:, :half], y[:, half:rotary] = lo * c - hi * s, lo * s + hi * c
    return y


def quantise(x, scale):
    """127 x / scale before it is rounded."""
    return 127.0 * x / scale if 0 < scale < math.inf else torch.zeros_like(x)


def append(quotients, scales, rows, start, block):
    """One request and one head.  ``quotients`` [n, dim] and ``scales`` [blocks]: what its cache holds for positions below ``start``
    (whole numbers there) and gets for those from there on: codes before their rounding.  ``rows`` [new, dim] float64."""
    for b in range(start // block, -(-(start + len(rows)) // block) if len(rows) else 0):
        lo, hi = b * block, min((b + 1) * block, start + len(rows))
        new = rows[max(lo, start) - start:hi - start]
        before = 0.0 if lo >= start else float(scales[b])
        most = float(new.abs().max())
        scale = max(before, most) if math.isfinite(before) and math.isfinite(most) and not torch.isnan(new).any() else math.nan
        if lo < start and not before >= scale:
            quotients[lo:start] = quotients[lo:start] * before / scale if math.isfinite(scale) else 0.0
        quotients[max(lo, start):hi] = quantise(new, scale) if math.isfinite(scale) else 0.0
        scales[b] = scale
    return quotients, scales


def values(codes, scales, block):
    """codes [n, dim], scales [blocks] -> what they stand for."""
    return codes.double() * scales.double().repeat_interleave(block)[:len(codes), None] / 127.0


def attend(q, k, v, start, scale, window, sink):
    """q [new, heads, dim] behind ``start`` positions; k, v [start + new, kv_heads, dim]; float64 [new, heads, dim]."""
    group = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    for i in range(len(q)):
        pos = start + i
        first = max(pos - window + 1, 0) if window else 0
        for h in range(q.shape[1]):
            s = k[first:pos + 1, h // group].double() @ q[i, h].double() * scale
            if sink is not None:
                s = torch.cat([s, sink[h].double().reshape(1)])
            p = torch.softmax(s, 0)[:pos + 1 - first]
            out[i, h] = p @ v[first:pos + 1, h // group].double()
    return out


def token_logprobs(x, token, top):
    """One row: (log probability, entropy, rank, ids of the first ``top``, their log probabilities)."""
    x = [float(v) for v in x]
    number = [(-math.inf if math.isnan(v) else v, 0 if math.isnan(v) else 1) for v in x]
    order = sorted(range(len(x)), key=lambda i: (-number[i][1], -number[i][0], i))
    m = max(v for v, _ in number)
    if any(math.isnan(v) for v in x) or not math.isfinite(m):
        return math.nan, math.nan, order.index(token), order[:top], [math.nan] * top
    z = math.fsum(math.exp(v - m) for v in x)
    entropy = math.log(z) - math.fsum(math.exp(v - m) * (v - m) for v in x if v > -math.inf) / z
    # the maximum first: a logit of -1e30 would swallow the logarithm
    return x[token] - m - math.log(z), entropy, order.index(token), order[:top], [x[i] - m - math.log(z) for i in order[:top]]
