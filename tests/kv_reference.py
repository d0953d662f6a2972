"""The 8-bit key/value cache and the attention over it, from their definitions, in 64 bits on the CPU."""
import math

import torch

MAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def needed_scale(most, dtype):
    if most == 0:
        return 2.0 ** -100
    m, e = math.frexp(most / MAX[dtype])  # m in [0.5, 1)
    s = math.ldexp(1.0, e - (m == 0.5)) if dtype == torch.float8_e4m3fn else math.ldexp(math.ceil(m * 256), e - 8)
    return max(s, 2.0 ** -100)


def codes(x, dtype):
    """Nearest code of each value (64 bits), ties to even; infinities saturate, NaN becomes 0."""
    x = torch.where(x.isnan(), 0.0, x.double()).clamp(-MAX[dtype], MAX[dtype])
    if dtype == torch.int8:
        return torch.round(x)
    e = torch.frexp(x)[1]
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def write(cache, scale, x, table, start, first):
    """cache [blocks, heads, 64, 64] code values and scale [blocks, heads] (64 bits, updated in place); x [tokens, heads, 64]."""
    dtype = cache["dtype"]
    c = cache["codes"]
    for s in range(len(start)):
        n, p0 = first[s + 1] - first[s], start[s]
        for b in range(p0 // 64, -(-(p0 + n) // 64)):
            lo, hi = max(p0, 64 * b), min(p0 + n, 64 * b + 64)
            if lo >= hi:
                continue
            page = table[s][b]
            for h in range(c.shape[1]):
                new = x[first[s] + lo - p0:first[s] + hi - p0, h].double()
                fine = new[new.isfinite()].abs()
                need = needed_scale(fine.max().item() if fine.numel() else 0.0, dtype)
                was = scale[page, h].item()
                older = lo - 64 * b
                if older and need <= was:
                    now = was
                else:
                    now = need
                    c[page, h, :older] = codes(c[page, h, :older] * was / now, dtype)
                c[page, h, older:hi - 64 * b] = codes(new / now, dtype)
                scale[page, h] = now


def attention(q, k, v, table, context, first, group, scale, causal):
    """q [tokens, heads, 64]; k, v [blocks, kv_heads, 64, 64] values, all in 64 bits.  Rows outside every sequence: NaN.
    Also returns the bound's factor: the largest |v| that a row's head and sequence has."""
    out = torch.full_like(q, float("nan"))
    vmax = torch.zeros(q.shape[0], q.shape[1], 1, dtype=torch.float64)
    for s, ctx in enumerate(context):
        n = first[s + 1] - first[s]
        if n <= 0:
            continue
        pages = table[s][:-(-ctx // 64)]
        rows = slice(first[s], first[s + 1])
        if ctx == 0:
            out[rows] = 0
            continue
        kk, vv = (x[pages].transpose(1, 2).flatten(0, 1)[:ctx].repeat_interleave(group, 1) for x in (k, v))
        z = torch.einsum("thd,khd->htk", q[rows], kk) * scale
        if causal:
            seen = torch.arange(ctx)[None] <= ctx - n + torch.arange(n)[:, None]
            z = z.masked_fill(~seen, -math.inf)
        m = z.amax(-1, keepdim=True)
        p = torch.exp(z - torch.where(m.isinf(), 0.0, m))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
        # a masked place counts for nothing, whatever value it holds
        out[rows] = torch.einsum("htk,khd->thd", p, torch.where(vv.isfinite(), vv, 0.0))
        vmax[rows] = vv.abs().amax((0, 2))[None, :, None]
    return out, vmax
