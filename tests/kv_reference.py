"""Plain implementations in 64 bits of what the key/value cache holds and of attention over it."""
import math

import torch

TOP = {"e4m3": 448.0, "int8": 127.0}


def held(x, fmt):
    """The values that rows x (..., d) are held as, float64.  8-bit formats: blocks of 32, scale 2^e with the smallest e >= -100
    such that max |x| <= top 2^e; a block with an infinity or a NaN is NaN throughout."""
    if fmt == "bf16":
        return x.to(torch.bfloat16).double()
    y = x.double().unflatten(-1, (-1, 32))
    a = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(a > 0, a, torch.ones_like(a)) / TOP[fmt]))
    # the logarithm is off by an ulp at most: put right from both sides
    e = torch.where(a > TOP[fmt] * torch.exp2(e), e + 1, e)
    e = torch.where(a <= TOP[fmt] * torch.exp2(e - 1), e - 1, e)
    e = torch.where(a > 0, e, torch.full_like(e, -100)).clamp(min=-100)
    s = torch.exp2(e)
    y = y / s
    if fmt == "int8":
        y = torch.round(y)
    else:
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -20))), min=-6) - 3)
        y = torch.round(y / step) * step
    y = torch.where(torch.isfinite(a), y * s, torch.full_like(y, math.nan))
    return y.float().double().flatten(-2)  # every held value is an f32, but for 2^128, what the largest f32 are rounded up to: infinity


def attend(q, keys, values, scale, window=0, holes=None):
    """q (n, heads, d): the last n tokens of a sequence whose held keys and values are (ctx, kv_heads, d), float64.  holes: positions
    nothing sees.  A masked key takes no part whatever it holds."""
    n, heads, d = q.shape
    ctx, kv = keys.shape[0], keys.shape[1]
    out = torch.zeros(n, heads, d, dtype=torch.float64)
    q, keys, values = q.double().cpu(), keys.double().cpu(), values.double().cpu()
    for i in range(n):
        p = ctx - n + i
        if p < 0:
            continue
        js = [j for j in range(max(0, p - window + 1) if window else 0, p + 1) if holes is None or j not in holes]
        if not js:
            continue
        for g in range(kv):
            h0, h1 = g * heads // kv, (g + 1) * heads // kv
            s = (q[i, h0:h1] @ keys[js, g].T) * scale
            out[i, h0:h1] = torch.softmax(s, -1) @ values[js, g]
    return out
