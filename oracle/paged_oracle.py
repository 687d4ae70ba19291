"""The paged cache and its attention from their definitions, on the CPU in 64 bits (test infrastructure only)."""
import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
LARGEST = {torch.float8_e4m3fn: 1.875, torch.int8: 1.984375}


def quantise(x, form):
    """(codes as the values that they are, exponents) of x [..., hd] (fp16 or bf16): see include/metaseq_paged.h."""
    cap = LARGEST[form] * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    x = x.double().clamp(-cap, cap)
    most = torch.nan_to_num(x, nan=0.0).abs().amax(-1)
    e = torch.full(most.shape, -126)
    for k in range(-126, 121):                      # the least that is large enough
        e = torch.where(most > TOP[form] * 2.0 ** k, k + 1, e)
    y = x * 2.0 ** (-e.double()).unsqueeze(-1)
    if form == torch.int8:
        c = torch.nan_to_num(torch.round(y), nan=0.0)
    else:
        binade = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6).nan_to_num(1.0)))
        binade = torch.where(2.0 ** binade > y.abs().clamp(min=2.0 ** -6), binade - 1, binade)
        step = 2.0 ** (binade - 3)
        c = torch.round(y / step) * step
    return c, e


def positions(pages, exps, table, upto, transposed):
    """Positions 0 .. upto - 1 of one sequence, [upto, kv_heads, hd] in 64 bits, and which of them are anywhere."""
    p = pages.double().transpose(2, 3) if transposed else pages.double()
    n, kvh, page, hd = p.shape
    if exps is not None:
        p = p * 2.0 ** exps.double().unsqueeze(-1)
    out, there = torch.zeros(upto, kvh, hd, dtype=torch.float64), torch.zeros(upto, dtype=torch.bool)
    for j in range(upto):
        at = j // page
        if at < len(table) and 0 <= int(table[at]) < n:
            out[j], there[j] = p[int(table[at]), :, j % page], True
    return out, there


def attend(q, keys, values, there, pos, scale, window=0, sinks=0):
    """(outputs, sum of p |v|, largest sum of |q k| scale among the keys seen) of the rows q [t, heads, hd] at positions
    pos ..; keys, values [.., kv_heads, hd]; in 64 bits."""
    t, heads, hd = q.shape
    group = heads // keys.shape[1]
    out, weight, size = (torch.zeros(t, heads, hd, dtype=torch.float64) for _ in range(3))
    for i in range(t):
        p = pos + i
        j = torch.arange(min(p + 1, keys.shape[0]))
        see = there[:len(j)].clone()
        if window:
            see &= (j > p - window) | (j < sinks)
        j = j[see]
        if not len(j):
            continue
        for h in range(heads):
            k, v = keys[j, h // group], values[j, h // group]
            z = k @ q[i, h].double() * scale
            w = torch.softmax(z, 0)
            out[i, h] = w @ v
            weight[i, h] = w @ v.abs()
            size[i, h] = (k.abs() @ q[i, h].double().abs()).max() * scale
    return out, weight, size
