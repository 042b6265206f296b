"""Serving operators around the paged key/value cache, as workloads: inputs, plain forms and exact values.

  plan      block table, slot map, positions and row offsets of a step, from the requests' lengths
  append    a step's keys and values rotated and written into their slots, its queries rotated
  attend    attention of each request's new tokens (one or many) over its pages
  addnorm   residual addition, RMSNorm with its weight, Q8_K quantization of the result

`run` computes them in elementary torch operations, or, where `own` is true, through the framework's entry points.
"""
import functools
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a serving loop's step of 48 running requests, one token each: launch latency
        dict(name="plan-decode-48", op="plan", n_req=48, page=16, cached_lo=1, cached_hi=2000, new_lo=1, new_hi=1, spare=16, pad=3,
             lens=1),
        # admission of 200 prompts at once, 16k tokens a step at most, the pool too small for the last of them
        dict(name="plan-admit-200", op="plan", n_req=200, page=16, cached_lo=0, cached_hi=40, new_lo=1, new_hi=511, spare=-100, pad=77,
             lens=2),
        # one decode step of 48 requests, grouped heads
        dict(name="append-decode-48", op="append", tokens=48, heads=32, kv_heads=8, dim=128, page=16, pages=64, dtype="bf16",
             rope="pairs", skip=1, lens=3),
        # a prompt of 8191 tokens of a 32-head, 4096-wide layer
        dict(name="append-prompt-8191", op="append", tokens=8191, heads=32, kv_heads=32, dim=128, page=64, pages=136, dtype="f16",
             rope="halves", skip=0, lens=4),
        # chat at its start: one request, a short cache, one token: latency
        dict(name="attend-one-short", op="attend", n_req=1, chunks=0, new_lo=1, new_hi=1, kv_lo=100, kv_hi=100, heads=32, kv_heads=32,
             dim=128, page=16, dtype="f16", causal=True, empty=0, lens=5),
        # a full decode batch of uneven lengths, grouped heads
        dict(name="attend-decode-64", op="attend", n_req=64, chunks=0, new_lo=1, new_hi=1, kv_lo=17, kv_hi=8192, heads=32, kv_heads=8,
             dim=128, page=16, dtype="bf16", causal=True, empty=1, lens=6),
        # one request with a very long cache, 64-wide heads in groups of eight
        dict(name="attend-one-long", op="attend", n_req=1, chunks=0, new_lo=1, new_hi=1, kv_lo=131001, kv_hi=131001, heads=32,
             kv_heads=4, dim=64, page=64, dtype="f16", causal=True, empty=0, lens=7),
        # drafted tokens checked: a few new tokens a request
        dict(name="attend-drafts-24", op="attend", n_req=24, chunks=24, new_lo=2, new_hi=6, kv_lo=300, kv_hi=4096, heads=32, kv_heads=8,
             dim=128, page=32, dtype="bf16", causal=True, empty=0, lens=8),
        # chunks of two long prompts, the earlier chunks in the cache
        dict(name="attend-chunk-2x2048", op="attend", n_req=2, chunks=2, new_lo=2048, new_hi=2048, kv_lo=7777, kv_hi=8192, heads=32,
             kv_heads=8, dim=128, page=16, dtype="bf16", causal=True, empty=0, lens=9),
        # a step that mixes a prompt's chunk with decoding requests, as many key heads as query heads
        dict(name="attend-mixed-8", op="attend", n_req=8, chunks=1, new_lo=700, new_hi=1000, kv_lo=1000, kv_hi=3000, heads=32,
             kv_heads=32, dim=128, page=16, dtype="f16", causal=True, empty=0, lens=10),
        # between two linears of one decoding request: latency
        dict(name="addnorm-1x4096", op="addnorm", rows=1, k=4096, stride=4096),
        # between two linears of a 2048-token prompt
        dict(name="addnorm-2048x4096", op="addnorm", rows=2048, k=4096, stride=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "append", "attend", "attend", "attend", "addnorm"))
    lens = rng.randrange(1 << 20)
    if op == "plan":
        return dict(op=op, n_req=_log(rng, 1, 600), page=rng.choice((1, 8, 16, 32, 64, 128)), cached_lo=0, cached_hi=_log(rng, 1, 4000),
                    new_lo=0, new_hi=_log(rng, 1, 300), spare=rng.randrange(-40, 60), pad=rng.randrange(100), lens=lens)
    group, kv_heads = rng.choice((1, 1, 2, 3, 4, 5, 7, 8)), rng.choice((1, 2, 4, 8, 8, 16, 32))
    if group * kv_heads > 64:
        group = 1
    dim, page, dtype = rng.choice((64, 80, 96, 128, 128, 256)), rng.choice((1, 8, 16, 16, 32, 64, 128)), rng.choice(("f16", "bf16"))
    if op == "append":
        tokens = _log(rng, 1, max(2, 1 << 24 >> int(math.log2(group * kv_heads * dim) + 1)))
        return dict(op=op, tokens=tokens, heads=group * kv_heads, kv_heads=kv_heads, dim=dim, page=page, pages=2 + (tokens + tokens // 3) // page,
                    dtype=dtype, rope=rng.choice(("none", "pairs", "halves")), skip=rng.randrange(3) if tokens > 8 else 0, lens=lens)
    if op == "addnorm":
        k = 256 * _log(rng, 1, 44)
        return dict(op=op, rows=_log(rng, 1, max(2, (1 << 23) // k)), k=k, stride=k + rng.choice((0, 0, 4, 256, 1)))
    kind = rng.choice(("decode", "decode", "drafts", "chunk", "mixed"))
    n_req = {"decode": _log(rng, 1, 200), "drafts": _log(rng, 1, 64), "chunk": rng.randrange(1, 4), "mixed": rng.randrange(2, 12)}[kind]
    new_hi = {"decode": 1, "drafts": rng.randrange(2, 9), "chunk": _log(rng, 20, 2000), "mixed": _log(rng, 20, 1200)}[kind]
    chunks = {"decode": 0, "drafts": n_req, "chunk": n_req, "mixed": rng.randrange(1, 3)}[kind]
    # the padded scores of the plain form and the cache stay below what the largest listed cases need
    most = min((1 << 29) // (n_req * new_hi * group * kv_heads), (1 << 28) // (n_req * kv_heads * dim), 40000)
    kv_hi = max(1, _log(rng, max(1, most // 200), max(1, most)))
    return dict(op=op, n_req=n_req, chunks=chunks, new_lo=max(1, new_hi // 3), new_hi=new_hi, kv_lo=max(1, kv_hi // rng.choice((1, 2, 10))),
                kv_hi=kv_hi, heads=group * kv_heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, causal=rng.random() < 0.85,
                empty=rng.randrange(2), lens=lens)


def _lengths(c):
    """The requests' lengths: a case's own, whatever the seed of its values."""
    r = random.Random(c["lens"])
    if c["op"] == "plan":
        cached = [r.randint(c["cached_lo"], c["cached_hi"]) for _ in range(c["n_req"])]
        return cached, [r.randint(c["new_lo"], c["new_hi"]) for _ in cached]
    new = [r.randint(c["new_lo"], c["new_hi"]) if i < c["chunks"] else 1 for i in range(c["n_req"])]
    r.shuffle(new)
    kv = [max(n, r.randint(c["kv_lo"], c["kv_hi"])) for n in new]
    if c["empty"] and c["n_req"] > 1:
        kv[r.randrange(c["n_req"])] = 0   # a request that got no pages this step: its rows see nothing
    return new, kv


def _int(values, dev, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).to(dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 1000003 + 17)
    randn = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    op, s = case["op"], {"op": case["op"]}
    if op == "plan":
        cached, new = _lengths(case)
        page = case["page"]
        held, want = [-(-c // page) for c in cached], [-(-(c + n) // page) for c, n in zip(cached, new)]
        n_free = max(1, sum(want) - sum(held) + case["spare"])
        ids = torch.randperm(sum(held) + n_free + 5, generator=g, device=dev).to(torch.int32)
        blocks = max(1, max(want)) + 2
        held_t = _int(held, dev, torch.int64)
        owned = torch.arange(blocks, device=dev)[None, :] < held_t[:, None]
        table = torch.full((case["n_req"], blocks), -1, dtype=torch.int32, device=dev)
        table[owned] = ids[:sum(held)]
        # the pool's front was handed out in earlier steps
        s.update(cached=_int(cached, dev), new=_int(new, dev), page=page, table=table, free=torch.cat([ids[-5:], ids[sum(held):-5]]).contiguous(),
                 used=_int([5], dev), used_out=_int([0], dev), tokens=sum(new) + case["pad"])
    elif op == "append":
        T, H, K, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        dtype = DTYPES[case["dtype"]]
        qkv = randn(T, (H + 2 * K) * D)           # one projection's output rows: queries, keys, values
        cache = [randn(case["pages"], K, case["page"], D).to(dtype) for _ in range(2)]
        slots = torch.randperm(case["pages"] * case["page"], generator=g, device=dev)[:T].contiguous()
        if case["skip"]:
            slots[torch.randint(T, (case["skip"],), generator=g, device=dev)] = -1   # padded rows
        pos = torch.randint(0, 8192, (T,), generator=g, device=dev).to(torch.int32)
        angle = torch.arange(8192, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
        rope = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
        s.update(q=qkv[:, :H * D].unflatten(1, (H, D)), k=qkv[:, H * D:(H + K) * D].unflatten(1, (K, D)),
                 v=qkv[:, (H + K) * D:].unflatten(1, (K, D)), k_cache=cache[0], v_cache=cache[1], slots=slots, pos=pos,
                 rope=rope if case["rope"] != "none" else None, halves=case["rope"] == "halves",
                 q_out=torch.empty((T, H, D), dtype=dtype, device=dev))
    elif op == "attend":
        new, kv = _lengths(case)
        H, K, D, page, dtype = case["heads"], case["kv_heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
        want = [-(-n // page) for n in kv]
        n_pages, blocks = sum(want) + 3, max(1, max(want))
        ids = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
        owned = torch.arange(blocks, device=dev)[None, :] < _int(want, dev, torch.int64)[:, None]
        table = torch.full((len(kv), blocks), -1, dtype=torch.int32, device=dev)
        table[owned] = ids[:sum(want)]
        k = torch.randn((n_pages, K, page, D), generator=g, device=dev, dtype=dtype)
        v = torch.randn((n_pages, K, page, D), generator=g, device=dev, dtype=dtype)
        # slots that hold no token of a request hold whatever was there before
        j = torch.arange(blocks * page, device=dev)
        live = j[None, :] < _int(kv, dev, torch.int64)[:, None]
        slot = table.long().clamp(min=0)[:, j // page] * page + j % page
        stale = torch.ones(n_pages * page, dtype=torch.bool, device=dev)
        stale[slot[live]] = False
        stale = stale.view(n_pages, 1, page, 1)
        k.masked_fill_(stale, float("nan"))
        v.masked_fill_(stale, float("nan"))
        q = (randn(sum(new), H, D) * 1.5).to(dtype)
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        s.update(q=q, k=k, v=v, table=table, q_start=_int(start, dev), kv_len=_int(kv, dev), max_new=max(new), page=page, scale=D ** -0.5,
                 causal=case["causal"])
    else:
        n, k, stride = case["rows"], case["k"], case["stride"]
        s.update(x=randn(n, stride)[:, :k], resid=randn(n, stride)[:, :k] * 4, weight=1 + 0.1 * randn(k), eps=1e-5)
    return s


# ---- plain forms -------------------------------------------------------------

def _plan(s):
    cached, new, free, table, page, T = s["cached"].long(), s["new"].long(), s["free"], s["table"], s["page"], s["tokens"]
    n, blocks = table.shape
    used = s["used"].long()
    end = torch.cumsum(new, 0)
    held, want = (cached + page - 1) // page, (cached + new + page - 1) // page
    fits = (end <= T) & (want <= blocks)
    need = torch.where(fits, want - held, 0)
    upto = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (used + upto <= free.numel()))     # in order: nobody overtakes
    used_out = used + torch.where(ok, need, 0).sum()
    kv_len = torch.where(ok, cached + new, 0)
    col = torch.arange(blocks, device=table.device)
    fresh = ok[:, None] & (col >= held[:, None]) & (col < want[:, None])
    pick = (used + upto - need - held)[:, None] + col
    table = torch.where(fresh, free[pick.clamp(0, free.numel() - 1)], table)
    t = torch.arange(T, device=table.device)
    r = torch.searchsorted(end, t, right=True)
    real = r < n
    r = r.clamp(max=n - 1)
    pos = cached[r] + t - (end - new)[r]
    slot = table[r, (pos // page).clamp(max=blocks - 1)].long() * page + pos % page
    placed = real & ok[r]
    q_start = torch.cat([end.new_zeros(1), end.clamp(max=T)])
    return [table, q_start.int(), kv_len.int(), torch.where(placed, slot, -1), torch.where(placed, pos, 0).int(), used_out.int()]


def _rotate(x, cos, sin, halves):
    a, b = (x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]) if halves else (x[..., 0::2], x[..., 1::2])
    y = a * cos - b * sin, a * sin + b * cos
    return torch.cat(y, -1) if halves else torch.stack(y, -1).flatten(-2)


def _append(s):
    q, k, v, slots = s["q"], s["k"], s["v"], s["slots"]
    if s["rope"] is not None:
        cos, sin = s["rope"][s["pos"].long()][:, None, :].chunk(2, -1)
        q, k = _rotate(q, cos, sin, s["halves"]), _rotate(k, cos, sin, s["halves"])
    k_cache, v_cache = s["k_cache"], s["v_cache"]
    page = k_cache.shape[2]
    # a row without a slot writes what the row of the highest slot writes
    at = torch.where(slots >= 0, torch.arange(len(slots), device=slots.device), slots.argmax())
    to = torch.where(slots >= 0, slots, slots.max())
    k_cache[to // page, :, to % page] = k[at].to(k_cache.dtype)
    v_cache[to // page, :, to % page] = v[at].to(v_cache.dtype)
    return [q.to(k_cache.dtype), k_cache, v_cache]


def _attend(s):
    """Padded to the longest request: scores, softmax and weighted sum of all requests at once."""
    q, table, q_start, kv_len, page, n = s["q"], s["table"].long(), s["q_start"].long(), s["kv_len"].long(), s["page"], s["max_new"]
    T, H, D = q.shape
    B, K = table.shape[0], s["k"].shape[1]
    new = q_start[1:] - q_start[:-1]
    i, j = torch.arange(n, device=q.device), torch.arange(table.shape[1] * page, device=q.device)
    live = j < kv_len[:, None]                                                  # [B, L]
    at = table.clamp(min=0)[:, j // page], j % page
    k = torch.where(live[..., None, None], s["k"][at[0], :, at[1]].float(), 0.0)    # [B, L, K, D]
    v = torch.where(live[..., None, None], s["v"][at[0], :, at[1]].float(), 0.0)
    rows = (q_start[:-1, None] + i).clamp(max=T - 1)
    qp = q[rows].float().view(B, n, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, H // K * n, D)
    scores = (qp @ k.permute(0, 2, 3, 1)).view(B, K, H // K, n, -1) * s["scale"]
    sees = live[:, None, :] & (i[:, None] < new[:, None, None])                 # [B, n, L]
    if s["causal"]:
        sees = sees & (j <= (kv_len - new)[:, None, None] + i[:, None])
    scores = scores.masked_fill_(~sees[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, K, H // K * n, -1) @ v.permute(0, 2, 1, 3)).view(B, K, H // K, n, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, n, H, D)
    t = torch.arange(T, device=q.device)
    r = torch.searchsorted(q_start[1:].contiguous(), t, right=True)
    return o[r, t - q_start[r]].to(q.dtype)


def _fold(a):
    """Pairwise sum over the last axis of 32, at distances 16, 8, 4, 2, 1: the order that RMSNorm's sum has here."""
    a = a[..., :16] + a[..., 16:]
    a = a[..., :8] + a[..., 8:]
    a = a[..., :4] + a[..., 4:]
    a = a[..., :2] + a[..., 2:]
    return a[..., 0] + a[..., 1]


def _addnorm(s):
    """Every rounding of the operator in its place: an 8-bit value next to a border takes the same side."""
    h = s["x"] + s["resid"]
    n, k = h.shape
    groups = _fold((h * h).view(n, k // 32, 32))
    groups = torch.nn.functional.pad(groups, (0, -(k // 32) % 32))
    lanes = functools.reduce(torch.add, groups.view(n, -1, 32).unbind(1))
    one = torch.ones((), device=h.device)
    inv = one / torch.sqrt(_fold(lanes) / (one * k) + s["eps"])
    y = (h * inv[:, None] * s["weight"]).view(n, k // 256, 256)
    top = torch.gather(y, 2, y.abs().argmax(2, keepdim=True))          # the value of largest magnitude
    scale = torch.where(top != 0, (-127 * one) / top, 0.0)             # 0 for a block of zeros
    q = torch.round(scale.double() * y.double()).clamp(max=127)
    sums = q.view(n, k // 256, 16, 16).sum(3).to(torch.int16)
    d = torch.where(scale != 0, one / scale, 0.0)
    return [h, (q.float() * d).view(n, k), sums.view(n, k // 16)]


# ---- one pass ------------------------------------------------------------------

def run(s):
    if not own:
        return {"plan": _plan, "append": _append, "attend": _attend, "addnorm": _addnorm}[s["op"]](s)
    paged, q2k = _framework()
    if s["op"] == "plan":
        plan = s.get("handle")
        if plan is None:
            plan = s["handle"] = paged.PagedPlan(s["table"], s["page"], s["tokens"])
        plan.build(s["cached"], s["new"], s["free"], s["used"], used_out=s["used_out"])
        return [s["table"], plan.q_start, plan.kv_len, plan.slots, plan.positions, s["used_out"]]
    if s["op"] == "addnorm":
        h, blocks = q2k.add_rms_quantize_q8k(s["x"], s["resid"], s["eps"], norm_w=s["weight"])
        n, k = h.shape
        blocks = blocks.view(n, k // 256, 292)
        values = blocks[:, :, 4:260].view(torch.int8) * blocks[:, :, :4].view(torch.float32)   # what the 8 bits stand for
        return [h, values.view(n, k), blocks[:, :, 260:].view(torch.int16).reshape(n, k // 16)]
    kv = s.get("handle")
    if kv is None:
        kv = s["handle"] = paged.PagedKV(*((s["k_cache"], s["v_cache"]) if s["op"] == "append" else (s["k"], s["v"])))
    if s["op"] == "append":
        q = paged.append(kv, s["k"], s["v"], s["slots"], q=s["q"], q_out=s["q_out"], positions=s["pos"], rope=s["rope"], halves=s["halves"])
        return [q, s["k_cache"], s["v_cache"]]
    return paged.attention(s["q"], kv, s["table"], s["q_start"], s["kv_len"], s["max_new"], scale=s["scale"], causal=s["causal"])


@functools.lru_cache(None)
def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sme-ai-ops_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from smeai_b200 import paged, q2k
    return paged, q2k


def work(case):
    op = case["op"]
    if op == "plan":
        cached, new = _lengths(case)
        page, n, T = case["page"], case["n_req"], sum(new) + case["pad"]
        fresh = sum(-(-(c + m) // page) + -c // page for c, m in zip(cached, new))
        return {"bytes": n * 8 + fresh * 8 + (2 * n + 1) * 4 + T * 12, "flops": 4 * n + 6 * T}
    if op == "append":
        T, H, K, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        rope = case["rope"] != "none"
        return {"bytes": T * (H + 2 * K) * D * 6 + T * 8 + rope * (T * 4 + min(T, 8192) * D * 4), "flops": rope * 3 * T * (H + K) * D}
    if op == "addnorm":
        n, k = case["rows"], case["k"]
        return {"bytes": n * k * 12 + n * k // 256 * 292 + k * 4, "flops": 9 * n * k}
    new, kv = _lengths(case)
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    # keys that the rows see, summed: n rows of a request whose cache holds m keys, the last row seeing all m
    pairs = sum((n * m - n * (n - 1) // 2 if case["causal"] else n * m) if m else 0 for n, m in zip(new, kv))
    pages = sum(-(-m // case["page"]) for m in kv)
    return {"bytes": sum(kv) * K * D * 4 + sum(new) * H * D * 4 + pages * 4 + (2 * len(new) + 1) * 4, "flops": 4 * pairs * H * D}


# ---- exact values ------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "addnorm":
        # the 8-bit values step where a rounding falls on a border: only the sum has a value in 64 bits
        return [s["x"].double() + s["resid"].double(), None, None]
    if case["op"] == "append":
        z = torch.complex(torch.zeros((), dtype=torch.float64), torch.ones((), dtype=torch.float64)).to(s["q"].device)

        def turned(x):
            x = x.double()
            if s["rope"] is None:
                return x
            D = x.shape[-1]
            c = s["rope"].double()[s["pos"].long()]
            w = (c[:, :D // 2] + z * c[:, D // 2:])[:, None]
            pairs = x.unflatten(-1, (2, D // 2)).transpose(-1, -2) if s["halves"] else x.unflatten(-1, (D // 2, 2))
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * w)
            return (y.transpose(-1, -2) if s["halves"] else y).flatten(-2)

        k, v, slots = turned(s["k"]), s["v"].double(), s["slots"]
        out = [turned(s["q"])]
        keep = slots >= 0
        for cache, x in ((s["k_cache"], k), (s["v_cache"], v)):
            flat = cache.double().permute(0, 2, 1, 3).flatten(0, 1)          # [slots, heads, dim]
            flat[slots[keep]] = x[keep]
            out.append(flat.unflatten(0, cache.shape[::2][:2]).permute(0, 2, 1, 3))
        return out
    q, H, K, page = s["q"].double(), case["heads"], case["kv_heads"], case["page"]
    out = torch.zeros_like(q)
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    for b, m in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        if m == 0 or hi == lo:
            continue
        pages = s["table"][b, :-(-m // page)].long()
        k = s["k"][pages].transpose(1, 2).flatten(0, 1)[:m].double()          # [m, K, D]
        v = s["v"][pages].transpose(1, 2).flatten(0, 1)[:m].double()
        for h in range(K):
            heads = slice(h * (H // K), (h + 1) * (H // K))
            w = torch.einsum("ngd,md->gnm", q[lo:hi, heads], k[:, h]) * s["scale"]
            if s["causal"]:
                w += torch.full((hi - lo, m), -math.inf, device=w.device, dtype=w.dtype).triu(m - (hi - lo) + 1)
            out[lo:hi, heads] = torch.einsum("gnm,md->ngd", torch.softmax(w, -1), v[:, h])
    return out
