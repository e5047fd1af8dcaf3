"""Timed cases of the operators of a language-model layer in serving: what stands between the
framework's GEMMs when a decoder-only model runs behind the encoder.

* `norm`: residual addition + root-mean-square norm, output in the input's type or in 8 bits with scales;
* `gemv`: product of a few rows with INT4 group-128 weights;
* `plan`: block tables, slot map and positions of a step from the request lengths;
* `attention`: the new tokens' keys and values go into a paged cache, the new tokens attend over it.

`own` selects the framework's calls; without it `run` computes the same in elementary torch operations.
"""
from __future__ import annotations

import importlib
import math
import random

import numpy as np
import torch

own = False

GROUP = 128
EPS = 1e-5
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    return importlib.import_module("l4-parakeet-rs_b200")


def listed():
    return [
        # the norm in front of a single request's projections, output in fp16: the smallest call
        dict(name="norm_1x1024_f16", kind="norm", rows=1, width=1024, type="f16", mode="same", residual=True),
        # a ragged chunk in front of an INT8 product; an odd row count and a width that is no power of two
        dict(name="norm_777x2560_int8", kind="norm", rows=777, width=2560, type="f16", mode="int8", residual=True),
        # a long prefill in front of an E4M3 product
        dict(name="norm_16384x4096_e4m3", kind="norm", rows=16384, width=4096, type="bf16", mode="e4m3", residual=True),
        # contracting projection of one token (the feed-forward width of the encoder's blocks), residual added
        dict(name="gemv_1x1024x4096", kind="gemv", rows=1, n=1024, k=4096, bias=False, act="none", residual=True),
        # a batch of 13 requests' tokens through a large expanding projection
        dict(name="gemv_13x28672x8192", kind="gemv", rows=13, n=28672, k=8192, bias=True, act="silu", residual=False),
        # one decode step of a handful of requests
        dict(name="plan_7_steps", kind="plan", requests=7, new_lo=1, new_hi=1, ctx_lo=3, ctx_hi=3000, page=16, lens=1),
        # a mixed step: a thousand requests, from single tokens to long prompts, behind nothing or long contexts
        dict(name="plan_1000_mixed", kind="plan", requests=1000, new_lo=1, new_hi=4000, ctx_lo=0, ctx_hi=30000, page=32, lens=2),
        # one token of one request, the head layout of the encoder (8 x 128): the smallest attention
        dict(name="attention_1x1_over_700", kind="attention", requests=1, new_lo=1, new_hi=1, ctx_lo=700, ctx_hi=700, heads=8,
             kv_heads=8, dim=128, page=16, type="f16", window=0, lens=3),
        # a decode step of 48 requests of very different lengths, shared key-value heads
        dict(name="attention_48x1_ragged", kind="attention", requests=48, new_lo=1, new_hi=1, ctx_lo=200, ctx_hi=16000, heads=32,
             kv_heads=8, dim=128, page=64, type="bf16", window=0, lens=4),
        # a chunk of a long prompt over what is cached of it already
        dict(name="attention_512_over_32000", kind="attention", requests=1, new_lo=512, new_hi=512, ctx_lo=32000, ctx_hi=32000,
             heads=16, kv_heads=2, dim=128, page=128, type="bf16", window=0, lens=5),
        # chunks of odd lengths in one step, own key-value heads of width 64, sliding window
        dict(name="attention_9_ragged_window", kind="attention", requests=9, new_lo=5, new_hi=1500, ctx_lo=0, ctx_hi=2500, heads=16,
             kv_heads=16, dim=64, page=32, type="f16", window=1024, lens=6),
        # two whole prompts, nothing cached: the largest
        dict(name="attention_2_prompts", kind="attention", requests=2, new_lo=7001, new_hi=8100, ctx_lo=0, ctx_hi=0, heads=16,
             kv_heads=4, dim=128, page=64, type="bf16", window=0, lens=7),
    ]


def _log_int(rng, low, high):
    if low >= high:
        return low
    return int(round(math.exp(rng.uniform(math.log(low + 1), math.log(high + 1))))) - 1


def draw(rng):
    kind = rng.choice(["norm", "gemv", "plan", "attention", "attention"])
    if kind == "norm":
        while True:
            rows, width = _log_int(rng, 1, 40000), _log_int(rng, 4, 1024) * 16
            if rows * width <= 16384 * 4096:
                break
        return dict(kind=kind, rows=rows, width=width, type=rng.choice(list(TYPES)), mode=rng.choice(["same", "int8", "e4m3"]),
                    residual=rng.random() < 0.8)
    if kind == "gemv":
        while True:
            n, k = _log_int(rng, 32, 30000), GROUP * _log_int(rng, 1, 128)
            if n * k <= 28672 * 8192:
                break
        return dict(kind=kind, rows=rng.randint(1, 16), n=n, k=k, bias=rng.random() < 0.5, act=rng.choice(["none", "silu", "relu"]),
                    residual=rng.random() < 0.5)
    if kind == "plan":
        new_hi = _log_int(rng, 1, 4000)
        return dict(kind=kind, requests=_log_int(rng, 1, 1000), new_lo=1, new_hi=new_hi, ctx_lo=0, ctx_hi=_log_int(rng, 1, 30000),
                    page=rng.choice([16, 32, 64, 128]), lens=rng.randrange(1 << 20))
    while True:
        new_hi = rng.choice([1, 1, _log_int(rng, 1, 8000)])
        case = dict(kind=kind, requests=_log_int(rng, 1, 64), new_lo=1, new_hi=new_hi, ctx_lo=0, ctx_hi=_log_int(rng, 1, 40000),
                    kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]),
                    type=rng.choice(list(TYPES)), window=rng.choice([0, 0, 0, _log_int(rng, 100, 4000)]), lens=rng.randrange(1 << 20))
        case["heads"] = case["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 8])
        new, ctx = _lengths(case)
        longest = max(a + b for a, b in zip(new, ctx))
        scores = case["requests"] * max(new) * case["heads"] * longest
        gathered = case["requests"] * longest * case["kv_heads"] * case["dim"]
        if scores <= 1.0e9 and gathered <= 4.0e8:
            return case


def _lengths(case):
    """New and cached tokens of each request: spread over the logarithm."""
    rng = random.Random(case["lens"])
    new = [_log_int(rng, case["new_lo"], case["new_hi"]) for _ in range(case["requests"])]
    ctx = [_log_int(rng, case["ctx_lo"], case["ctx_hi"]) for _ in range(case["requests"])]
    return new, ctx


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _paged(new, ctx, page, gen_np):
    """Block tables before and after a step: page ids in the order a busy allocator leaves them."""
    pages_old = [-(-c // page) for c in ctx]
    pages_all = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    total = sum(pages_all)
    ids = gen_np.permutation(total + total // 8 + 4).astype(np.int32)
    table = np.full((len(new), max(max(pages_all), 1)), -1, np.int32)
    at = 0
    for r, n in enumerate(pages_old):
        table[r, :n] = ids[at:at + n]
        at += n
    free = ids[at:]
    full, used = table.copy(), 0
    for r, (a, b) in enumerate(zip(pages_old, pages_all)):
        full[r, a:b] = free[used:used + b - a]
        used += b - a
    return table, full, free, len(ids)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    gen_np = np.random.default_rng(seed)
    kind = case["kind"]
    s = dict(case)
    if kind == "norm":
        dtype, rows, width = TYPES[case["type"]], case["rows"], case["width"]
        s["x"] = _normal(gen, (rows, width), dtype)
        # the residual stream has a few channels far above the rest
        r = torch.randn((rows, width), generator=gen, device="cuda") * (1.0 + 20.0 * (torch.rand(width, generator=gen, device="cuda") < 0.004))
        s["residual_in"] = r.to(dtype) if case["residual"] else None
        s["residual_out"] = torch.empty_like(s["x"]) if case["residual"] else None
        s["gamma"] = _normal(gen, (width,), dtype, 0.1) + 1.0
        s["out"] = torch.empty((rows, width), device="cuda", dtype={"same": dtype, "int8": torch.int8, "e4m3": torch.uint8}[case["mode"]])
        s["scales"] = None if case["mode"] == "same" else torch.empty(rows, device="cuda", dtype=torch.float32)
    elif kind == "gemv":
        rows, n, k = case["rows"], case["n"], case["k"]
        s["x"] = _normal(gen, (rows, k), torch.float16)
        nibbles = torch.randint(0, 15, (n, k // 2, 2), generator=gen, device="cuda", dtype=torch.int32) - 7     # codes in [-7, 7]
        s["codes"] = ((nibbles[..., 0] & 15) | ((nibbles[..., 1] & 15) << 4)).to(torch.uint8)
        s["scales"] = ((0.5 + torch.rand((k // GROUP, n), generator=gen, device="cuda")) * 0.01).half()
        s["b"] = torch.randn(n, generator=gen, device="cuda") if case["bias"] else None
        s["res"] = _normal(gen, (rows, n), torch.float16) if case["residual"] else None
        s["out"] = torch.empty((rows, n), device="cuda", dtype=torch.float16)
    else:
        new, ctx = _lengths(case)
        if kind == "plan":                          # other lengths for every seed, the sum as it is
            order = gen_np.permutation(len(new))
            new, ctx = [new[i] for i in order], [ctx[i] for i in order]
        before, after, free, pages = _paged(new, ctx, case["page"], gen_np)
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        s["tokens"], s["pages"], s["longest"], s["most"] = int(starts[-1]), pages, max(a + b for a, b in zip(new, ctx)), max(new)
        if kind == "plan":
            s["cached"], s["new"] = torch.tensor(ctx, dtype=torch.int32, device="cuda"), torch.tensor(new, dtype=torch.int32, device="cuda")
            s["table"], s["free"] = torch.from_numpy(before).cuda(), torch.from_numpy(free).cuda()
            s["free_count"] = torch.tensor([len(free)], dtype=torch.int32, device="cuda")
            return s
        dtype, kv, dim, tokens = TYPES[case["type"]], case["kv_heads"], case["dim"], s["tokens"]
        s["table"], s["starts"] = torch.from_numpy(after).cuda(), torch.from_numpy(starts).cuda()
        s["lengths"] = torch.tensor([a + b for a, b in zip(new, ctx)], dtype=torch.int32, device="cuda")
        positions = np.concatenate([np.arange(c, c + n) for n, c in zip(new, ctx)])
        rows = np.repeat(np.arange(len(new)), new)
        slots = after[rows, positions // case["page"]].astype(np.int64) * case["page"] + positions % case["page"]
        s["slots"] = torch.from_numpy(slots).cuda()
        s["k_cache"] = _normal(gen, (pages, case["page"], kv, dim), dtype)
        s["v_cache"] = _normal(gen, (pages, case["page"], kv, dim), dtype)
        # one projection's output holds queries, keys and values side by side
        qkv = _normal(gen, (tokens, (case["heads"] + 2 * kv) * dim), dtype)
        q, k, v = qkv.split([case["heads"] * dim, kv * dim, kv * dim], dim=1)
        s["q"], s["k"], s["v"] = q.unflatten(1, (-1, dim)), k.unflatten(1, (-1, dim)), v.unflatten(1, (-1, dim))
        s["out"] = torch.empty((tokens, case["heads"], dim), device="cuda", dtype=dtype)
    return s


# ---- plain forms: elementary operations in 32 bits
def _plain_norm(s):
    dtype = s["x"].dtype
    x, total = s["x"], None
    if s["residual_in"] is not None:
        x = total = (x.float() + s["residual_in"].float()).to(dtype)
    f = x.float()
    y = f * torch.rsqrt(f.square().mean(1, keepdim=True) + EPS) * s["gamma"].float()
    return y, total


def _norm_result(mode, y, total, dtype):
    if mode == "same":
        return [y.to(dtype), total]
    top = 448.0 if mode == "e4m3" else 127.0
    peak = y.abs().amax(1)
    scale = torch.where(peak > 0, peak / top, torch.ones_like(peak))
    q = y / scale[:, None]
    return [q.to(torch.float8_e4m3fn) if mode == "e4m3" else torch.round(q).clamp(-127, 127).half(), scale, total]


def _unpacked(codes):
    c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(1).to(torch.int8)
    return torch.where(c > 7, c - 16, c)


def _plain_gemv(s):
    codes = _unpacked(s["codes"])
    scales = s["scales"].t().repeat_interleave(GROUP, dim=1)
    v = s["x"].float() @ (codes.half() * scales).float().t()      # the weight is the fp16 product of code and scale
    if s["b"] is not None:
        v = v + s["b"]
    if s["act"] == "silu":
        v = v / (1.0 + torch.exp(-v))
    elif s["act"] == "relu":
        v = torch.relu(v)
    if s["res"] is not None:
        v = v + s["res"].float()
    return v.half()


def _plain_plan(s):
    page, device = s["page"], s["new"].device
    new, cached = s["new"].long(), s["cached"].long()
    lengths = cached + new
    ends = torch.cumsum(new, 0)
    starts = torch.cat([torch.zeros(1, dtype=torch.long, device=device), ends])
    had, has = (cached + page - 1) // page, (lengths + page - 1) // page
    first_free = torch.cumsum(has - had, 0) - (has - had)
    column = torch.arange(s["table"].shape[1], device=device)[None, :]
    fresh = (column >= had[:, None]) & (column < has[:, None])
    index = torch.where(fresh, first_free[:, None] + column - had[:, None], 0)
    s["table"].copy_(torch.where(fresh, s["free"][index], s["table"]))
    token = torch.arange(s["tokens"], device=device)
    request = torch.searchsorted(ends, token, right=True)
    positions = cached[request] + token - starts[request]
    slots = s["table"][request, positions // page].long() * page + positions % page
    return [s["table"], starts.int(), lengths.int(), positions.int(), slots, (has - had).sum().int()[None]]


def _plain_attention(s):
    R, page, dim, kv = s["requests"], s["page"], s["dim"], s["kv_heads"]
    group, longest, most, device = s["heads"] // kv, s["longest"], s["most"], s["q"].device
    flat_k, flat_v = s["k_cache"].flatten(0, 1), s["v_cache"].flatten(0, 1)
    flat_k[s["slots"]] = s["k"]
    flat_v[s["slots"]] = s["v"]
    lengths, starts = s["lengths"].long(), s["starts"].long()
    new = starts[1:] - starts[:-1]
    # keys and values of every request, and its queries, padded to the longest
    j = torch.arange(longest, device=device)
    live = j[None, :] < lengths[:, None]
    where = torch.where(live, s["table"].long().clamp(min=0)[:, j // page] * page + j % page, 0)
    k = flat_k[where].float().masked_fill(~live[:, :, None, None], 0.0).permute(0, 2, 3, 1)          # [R, kv, dim, longest]
    v = flat_v[where].float().masked_fill(~live[:, :, None, None], 0.0).permute(0, 2, 1, 3)          # [R, kv, longest, dim]
    i = torch.arange(most, device=device)
    rows = torch.where(i[None, :] < new[:, None], starts[:-1, None] + i[None, :], 0)
    q = s["q"][rows].float().unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).reshape(R, kv, group * most, dim)
    p = (lengths - new)[:, None] + i[None, :]                                                        # positions [R, most]
    seen = (j[None, None, :] <= p[:, :, None]) & live[:, None, :]
    if s["window"] > 0:
        seen &= j[None, None, :] > p[:, :, None] - s["window"]
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(dim)).unflatten(2, (group, most))
    scores.masked_fill_(~seen[:, None, None, :, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = scores.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    out = torch.matmul(w.flatten(2, 3), v).unflatten(2, (group, most)) / w.sum(-1, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4)                                                                 # [R, most, kv, group, dim]
    request = torch.searchsorted(starts[1:], torch.arange(s["tokens"], device=device), right=True)
    return out[request, torch.arange(s["tokens"], device=device) - starts[request]].flatten(1, 2).to(s["q"].dtype)


def run(s):
    kind = s["kind"]
    if kind == "norm":
        if own:
            pk = _ops()
            mode = {"same": pk.lib.LN_F16, "int8": pk.lib.LN_S8_ROW, "e4m3": pk.lib.LN_E4M3_ROW}[s["mode"]]
            out, scales, total = pk.ops.add_rms_norm(s["x"], s["gamma"], residual=s["residual_in"], residual_out=s["residual_out"],
                                                     mode=mode, out=s["out"], scales=s["scales"])
            if s["residual_in"] is None:                # the call hands its input back where it kept no sum
                total = None
            if s["mode"] == "same":
                return [out, total]
            return [out.view(torch.float8_e4m3fn) if s["mode"] == "e4m3" else out.half(), scales, total]
        return _norm_result(s["mode"], *_plain_norm(s), s["x"].dtype)
    if kind == "gemv":
        if own:
            pk = _ops()
            act = {"none": pk.lib.ACT_NONE, "silu": pk.lib.ACT_SILU, "relu": pk.lib.ACT_RELU}[s["act"]]
            return pk.ops.gemv_w4g128(s["x"], s["codes"], s["scales"], bias=s["b"], act=act, residual=s["res"], out=s["out"])
        return _plain_gemv(s)
    if kind == "plan":
        if own:
            p = _ops().ops.paged_plan(s["cached"], s["new"], s["table"], s["free"], s["free_count"], tokens=s["tokens"],
                                      page_size=s["page"])
            return [s["table"], p.starts, p.lengths, p.positions, p.slots, p.used]
        return _plain_plan(s)
    if own:
        out = _ops().ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["starts"], s["lengths"], key=s["k"],
                                         value=s["v"], slots=s["slots"], window=s["window"], max_new=s["most"], out=s["out"])
    else:
        out = _plain_attention(s)
    return [out, s["k_cache"], s["v_cache"]]


# ---- the same in 64 bits, written from the definitions
def _exact_norm(s):
    x = s["x"].double()
    total = None
    if s["residual_in"] is not None:
        x = total = (x + s["residual_in"].double()).to(s["x"].dtype).double()     # the stream is kept in its own type
    y = s["gamma"].double() * x / torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + EPS)
    if s["mode"] == "same":
        return [y, total]
    scale = y.abs().max(1, keepdim=True).values / (448 if s["mode"] == "e4m3" else 127)
    scale[scale == 0] = 1
    return [torch.round(y / scale) if s["mode"] == "int8" else y / scale, scale[:, 0], total]


def _exact_gemv(s):
    low, high = (s["codes"].int() & 15), (s["codes"].int() >> 4)
    signed = torch.stack([(low + 8) % 16 - 8, (high + 8) % 16 - 8], dim=2).reshape(s["n"], s["k"] // GROUP, GROUP)
    weight = (signed.double() * s["scales"].double().t()[:, :, None]).half().reshape(s["n"], s["k"])
    v = torch.cat([s["x"].double() @ w.double().t() for w in weight.split(4096)], dim=1)
    if s["b"] is not None:
        v += s["b"].double()
    v = v * torch.sigmoid(v) if s["act"] == "silu" else v.clamp(min=0) if s["act"] == "relu" else v
    return v if s["res"] is None else v + s["res"].double()


def _exact_plan(s):
    new, cached, table, free = (s[n].cpu().numpy() for n in ("new", "cached", "table", "free"))
    page, used, positions, slots = s["page"], 0, [], []
    for r in range(len(new)):
        for c in range(-(-int(cached[r]) // page), -(-int(cached[r] + new[r]) // page)):
            table[r, c] = free[used]
            used += 1
        at = np.arange(cached[r], cached[r] + new[r])
        positions.append(at)
        slots.append(table[r, at // page].astype(np.int64) * page + at % page)
    return [table, np.concatenate([[0], np.cumsum(new)]), cached + new, np.concatenate(positions), np.concatenate(slots), np.array([used])]


def _exact_attention(s):
    new, ctx = _lengths(s)
    group, page = s["heads"] // s["kv_heads"], s["page"]
    out, first = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    caches = []
    for cache, fresh in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
        cache = cache.clone()
        cache.reshape(-1, s["kv_heads"], s["dim"]).index_copy_(0, s["slots"], fresh.contiguous())
        caches.append(cache)
    for r, (n, c) in enumerate(zip(new, ctx)):
        ids = s["table"][r, :-(-(n + c) // page)].long()
        k, v = (cache[ids].flatten(0, 1)[:n + c].double() for cache in caches)
        place = torch.arange(c, c + n, device="cuda")[:, None]
        key = torch.arange(n + c, device="cuda")[None, :]
        hidden = key > place
        if s["window"] > 0:
            hidden |= key <= place - s["window"]
        for h in range(s["heads"]):
            score = s["q"][first:first + n, h].double() @ k[:, h // group].t() / math.sqrt(s["dim"])
            out[first:first + n, h] = torch.softmax(score.masked_fill(hidden, -math.inf), 1) @ v[:, h // group]
        first += n
    return [out, None, None]


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "gemv": _exact_gemv, "plan": _exact_plan, "attention": _exact_attention}[case["kind"]](s)


# ---- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "norm":
        elements = case["rows"] * case["width"]
        out = 2 if case["mode"] == "same" else 1
        return dict(bytes=elements * (2 + (4 if case["residual"] else 0) + out) + 2 * case["width"] + (0 if out == 2 else 4 * case["rows"]),
                    flops=6 * elements)
    if kind == "gemv":
        m, n, k = case["rows"], case["n"], case["k"]
        return dict(bytes=n * k * (0.5 + 2 / GROUP) + 2 * m * (k + n) + (4 * n if case["bias"] else 0) + (2 * m * n if case["residual"] else 0),
                    flops=2 * m * n * k)
    new, ctx = _lengths(case)
    if kind == "plan":
        page = case["page"]
        fresh = sum(-(-(n + c) // page) - -(-c // page) for n, c in zip(new, ctx))
        return dict(bytes=16 * len(new) + 12 * sum(new) + 8 * fresh, flops=4 * sum(new))
    window = case["window"] or (1 << 40)

    def visible(n, c):
        full = min(n, max(0, window - c))                                 # tokens that the window does not cut yet
        return full * c + full * (full + 1) // 2 + (n - full) * window if n > full else n * c + n * (n + 1) // 2

    pairs = sum(visible(n, c) for n, c in zip(new, ctx))
    keys = sum(min(n + c, n + window - 1) for n, c in zip(new, ctx))
    tokens = sum(new)
    return dict(bytes=2 * case["dim"] * (2 * tokens * case["heads"] + 2 * case["kv_heads"] * (keys + tokens + tokens)),
                flops=4 * case["dim"] * case["heads"] * pairs)
