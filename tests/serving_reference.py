"""Plain statements of the serving operators in 64 bits, and how far a kernel with fp32 sums may be from them."""
import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}          # half a rounding step, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}        # half a step of the smallest numbers


def rms_norm(x, gamma, residual, eps):
    """(s, y): the rounded sum and the norm, in 64 bits."""
    s = x.double() if residual is None else (x.float() + residual.float()).to(x.dtype).double()
    return s, s * torch.rsqrt(s.square().mean(1, keepdim=True) + eps) * gamma.double()


# Norm in fp32: at most 32 sequential terms a thread and 10 steps of a tree, all positive: 42 * 2^-24 of the sum,
# half of that after the root; the root 2 units, the products and the scale 4 roundings: below 2e-6 in all.
NORM_REL = 4e-6


def w4_weights(codes, scales):
    """[n, k] weights f16(code * scale) in 64 bits from packed codes and [k / 128, n] scales."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(1).to(torch.int32)
    c = torch.where(c > 7, c - 16, c).double()
    return (c * scales.double().t().repeat_interleave(128, 1)).half().double()


def gemv_tolerance(x, w, out, dtype):
    """A warp adds k / 128 products of 16 in a chain, 8 warps are joined; the tensor cores' sums of 16 are good to 2^-22 of
    the magnitudes; the epilogue adds a few roundings of the result."""
    terms = x.double().abs() @ w.abs().t()
    step = HALF.get(dtype, 2.0 ** -24)
    return (x.shape[1] / 128 + 24) * 2.0 ** -22 * terms + (step + 1e-6) * out.abs() + TINY.get(dtype, 0.0) + 1e-30


def attention(q, keys, values, positions, causal, window, scale):
    """One request: q [n, heads, d], keys and values [len, kv, d], positions [n]; (out, lse, sum p |v|, largest error
    of a score) in 64 bits.  A row that sees nothing: zeros and -inf."""
    n, heads, d = q.shape
    length, kv = keys.shape[0], keys.shape[1]
    group = heads // kv
    j = torch.arange(length, device=q.device)
    seen = torch.ones(n, length, dtype=torch.bool, device=q.device)
    if causal:
        seen &= j[None] <= positions[:, None]
    if window > 0:
        seen &= j[None] > positions[:, None] - window
    out = torch.zeros(n, heads, d, dtype=torch.float64, device=q.device)
    spread, lse = torch.zeros_like(out), torch.full((n, heads), -math.inf, dtype=torch.float64, device=q.device)
    off = 0.0
    for h in range(heads):
        k, v = keys[:, h // group].double(), values[:, h // group].double()
        qh = q[:, h].double()
        s = (qh @ k.t() * scale).masked_fill(~seen, -math.inf)
        if seen.any():
            off = max(off, float((abs(scale) * (qh.abs() @ k.abs().t())).masked_fill(~seen, 0).max()))
        top = s.amax(1, keepdim=True) if length else torch.full((n, 1), -math.inf, dtype=torch.float64, device=q.device)
        live = torch.isfinite(top[:, 0])
        p = torch.exp(s - top.masked_fill(~torch.isfinite(top), 0))
        total = p.sum(1, keepdim=True)
        p = p / total.clamp(min=1e-300)
        out[:, h], spread[:, h] = p @ v, p @ v.abs()
        lse[live, h] = (top + torch.log(total))[live, 0]
    return out, lse, spread, off


def attention_tolerance(out, spread, off, values, length, dtype):
    """Scores: d / 16 + 8 sums of 2^-22 of sum |q k| (`off`, scaled) and as much again in the exponent and its base 2
    form, twice (numerator and denominator); P rounded to the type (half a step of each weight, or half the smallest
    step where it is below the normal numbers; the row's sum is 1 at least on the same scale); the output rounded."""
    score = (16 + 8) * 2.0 ** -22 * off + 1e-5
    largest = float(values.double().abs().max()) if values.numel() else 0.0
    return (HALF[dtype] + 2 * score) * spread + HALF[dtype] * out.abs() + (length * largest + 1) * TINY[dtype] * 4


def paged(cache, table_row, length):
    """[length, kv, d] of a request from a cache [pages, page_size, kv, d]."""
    page = cache.shape[1]
    ids = table_row[:-(-length // page)].long()
    return cache[ids].flatten(0, 1)[:length] if length else cache.new_zeros((0,) + cache.shape[2:])


def plan(cached, new, table, free, page):
    """(table, starts, lengths, positions, slots, used) as lists; `table` a list of rows."""
    table, starts, positions, slots, used = [list(r) for r in table], [0], [], [], 0
    for r, (c, n) in enumerate(zip(cached, new)):
        for i in range(-(-c // page), -(-(c + n) // page)):
            table[r][i] = free[used]
            used += 1
        for p in range(c, c + n):
            positions.append(p)
            slots.append(table[r][p // page] * page + p % page)
        starts.append(starts[-1] + n)
    return table, starts, [c + n for c, n in zip(cached, new)], positions, slots, used
