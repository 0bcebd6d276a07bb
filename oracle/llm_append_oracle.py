"""CPU oracle for the LLM's rotary, append attention and tree verification --
TEST INFRASTRUCTURE ONLY: tests compare the kernels with it, the product path never
imports it.

Everything is in float64 from the definitions in ``include/dllm.h``.  Beside the
attention's outputs it gives the bound that a kernel with fp32 scores and sums,
16-bit probabilities and a 16-bit result stays within."""
from __future__ import annotations

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# Below its smallest normal number (2^-14) fp16's values are 2^-24 apart: a result
# there is off by up to half of that, however small it is.  The other types'
# normal numbers reach below 10^-37.
FLOOR = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def rotate(x, positions, inv, factor, rot, layout):
    """x [T, heads, D] -> (rotated in float64, bound of one rounding to x's type)."""
    y = x.double().clone()
    pos = positions.double()[:, None, None]
    t = pos * inv.double()
    c, s = torch.cos(t) * factor, torch.sin(t) * factor
    pair = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else \
        (slice(0, rot, 2), slice(1, rot, 2))
    a, b = y[..., pair[0]].clone(), y[..., pair[1]].clone()
    y[..., pair[0]], y[..., pair[1]] = a * c - b * s, b * c + a * s
    # fp32 products and sums, sincospi of a 2^-31-turn angle; float64's own angle
    # error at far positions counts for the oracle
    size = torch.zeros_like(y)
    wobble = (a.abs() + b.abs()) * factor * (2.0 ** -21 + pos.abs() * inv.double() * 2.0 ** -51)
    size[..., pair[0]], size[..., pair[1]] = wobble, wobble
    return y, size + (y.abs() + size) * HALF_STEP[x.dtype] + FLOOR[x.dtype]


def visible(m, ctx, causal=True, window=0, prefix=0, first=None, tree=None):
    """bool [m, ctx]: which cached keys each of the m newest tokens sees."""
    base = ctx - m
    p = (base + torch.arange(m))[:, None]
    k = torch.arange(ctx)[None]
    if tree is not None:
        bit = torch.bitwise_right_shift(tree[:, None], (k - base).clamp(0, 63)) & 1
        return (k < base) | (bit.bool() & (k >= base))
    see = (k <= p) | (k < prefix) if causal else torch.ones(m, ctx, dtype=torch.bool)
    if window:
        see &= k > p - window
    if first is not None:
        see &= k >= first[:, None]
    return see


def attend(q, K, V, see, scale, softcap=0.0, slopes=None):
    """q [m, H, D], K / V [ctx, KVH, D], see [m, ctx] -> (out [m, H, D], bound)."""
    m, H, D = q.shape
    ctx, KVH = K.shape[:2]
    G, base = H // KVH, ctx - m
    u = HALF_STEP[q.dtype]
    out, tol = torch.zeros(m, H, D, dtype=torch.float64), torch.zeros(m, H, D, dtype=torch.float64)
    if ctx == 0 or m == 0:
        return out, tol
    some = see.any(1)
    far = (base + torch.arange(m)[:, None] - torch.arange(ctx)[None]).abs().double()
    for h in range(H):
        k, v, qq = K[:, h // G].double(), V[:, h // G].double(), q[:, h].double()
        live = see.any(0)                     # keys that nobody sees may hold anything
        k, v = torch.where(live[:, None], k, 0.0), torch.where(live[:, None], v, 0.0)
        s = qq @ k.t() * scale
        off = (qq.abs() @ k.abs().t() * scale) * ((D + 8) * 2.0 ** -24)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
            off = off + softcap * 2.0 ** -21
        if slopes is not None:
            s = s - float(slopes[h]) * far
        off = off + (s.abs() + 1) * 2.0 ** -21
        s = torch.where(see, s, -math.inf)
        top = s.amax(1, keepdim=True)
        top = torch.where(some[:, None], top, 0.0)
        # scores far below the maximum lose their absolute accuracy and their weight
        e = torch.exp(s - top)
        total = e.sum(1, keepdim=True)
        pr = torch.where(some[:, None], e / total.clamp_min(1e-300), 0.0)
        out[:, h] = pr @ v
        size = pr @ v.abs()
        drift = 2 * ((pr * torch.where(see, off, 0.0)) @ v.abs()) + \
            2 * (pr * torch.where(see, off, 0.0)).sum(1, keepdim=True) * size
        t = size * u + drift
        if q.dtype == torch.float16:          # probabilities below fp16's normal numbers
            t = t + 2.0 ** -25 * (see.double() @ v.abs()) / total.clamp_min(1.0)
        tol[:, h] = t + (out[:, h].abs() + t) * u + FLOOR[q.dtype]
    return out, tol


def gather(cache, table_row, n_pos):
    """Positions [0, n_pos) of one sequence: [n_pos, KVH, D]; missing blocks read as NaN."""
    bs = cache.shape[1]
    k = torch.arange(n_pos)
    blk = torch.as_tensor(table_row).long()[k // bs]
    out = cache[blk.clamp(min=0), k % bs].clone()
    out[blk < 0] = float("nan")
    return out
