"""The paged key/value cache on the GPU: plan, append and attention against plain
implementations (Python loops, 64 bits), at the lengths, layouts and masks
where they can go wrong."""
import math

import pytest
import torch

import smeai_b200 as S
from smeai_b200 import paged

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


# ---- plan ------------------------------------------------------------------------

def plan_reference(cached, new, page, free, used, table, n_tokens, max_blocks):
    """The documented rules, request by request."""
    table, start, kv, slots, pos = [row[:] for row in table], [0], [], [-1] * n_tokens, [0] * n_tokens
    asked = row = 0
    taken = 0
    for i, (c, n) in enumerate(zip(cached, new)):
        held, want = -(-c // page), -(-(c + n) // page)
        fits = row + n <= n_tokens and want <= max_blocks
        need = want - held if fits else 0
        asked += need
        ok = fits and (need == 0 or used + asked <= len(free))
        if ok:
            for b in range(need):
                table[i][held + b] = free[used + asked - need + b]
            if need:
                taken = asked
            for t in range(n):
                p = c + t
                slots[row + t], pos[row + t] = table[i][p // page] * page + p % page, p
        kv.append(c + n if ok else 0)
        row += n
        start.append(min(row, n_tokens))
    return table, start, kv, slots, pos, used + taken


def run_plan(dev, cached, new, page, free, used, table, n_tokens):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    t = i32(table)
    plan = paged.PagedPlan(t, page, n_tokens)
    plan.slots.fill_(77)
    n_used = i32([used])
    plan.build(i32(cached), i32(new), i32(free), n_used)
    return plan, n_used


PLANS = {
    "one token": ([0], [1], 16, 4, 0, 0),
    "nothing new": ([5, 0, 16], [0, 0, 0], 16, 2, 0, 3),
    "page edges": ([15, 16, 17, 0, 31], [1, 1, 1, 33, 2], 16, 9, 2, 5),
    "pages of one token": ([3, 0, 9], [2, 7, 1], 1, 30, 1, 0),
    "pool runs out in the middle": ([4, 4, 3, 0, 4], [8, 8, 1, 9, 0], 4, 5, 1, 1),
    "pool empty": ([4, 8, 2], [1, 1, 1], 4, 0, 0, 0),
    "wide pages": ([1000, 65536 * 2], [3, 70000], 65536, 3, 0, 2),
}


@pytest.mark.parametrize("name", PLANS)
def test_plan_small(cuda, name):
    cached, new, page, n_free, used, pad = PLANS[name]
    n_blocks = max(-(-(c + n) // page) for c, n in zip(cached, new)) + 1
    ids = iter(range(100, 10000))
    table = [[next(ids) if b < -(-c // page) else -9 for b in range(n_blocks)] for c in cached]
    free = [next(ids) for _ in range(n_free)]
    T = sum(new) + pad
    ref = plan_reference(cached, new, page, free, used, table, T, n_blocks)
    plan, n_used = run_plan(cuda, cached, new, page, free, used, table, T)
    got = (plan.block_table.tolist(), plan.q_start.tolist(), plan.kv_len.tolist(), plan.slots.tolist(), plan.positions.tolist(), n_used.item())
    assert got == tuple(ref)
    assert S.take_device_error() == 0


@pytest.mark.parametrize("n_req,new_hi,page,short,cut", [(1, 9000, 16, 0, 0), (33, 1, 16, 3, 0), (1023, 3, 8, 0, 5), (1024, 20, 32, 40, 0),
                                                          (1025, 40, 16, 200, 900), (8192, 4, 4, 0, 0), (8192, 1, 128, 1000, 1)])
def test_plan_random(cuda, n_req, new_hi, page, short, cut):
    """Both sides of the one-kernel limit (8192 rows), pools too small by
    `short` pages, row buffers too small by `cut` rows."""
    g = torch.Generator().manual_seed(n_req + new_hi)
    cached = torch.randint(0, 100, (n_req,), generator=g).tolist()
    new = torch.randint(0, new_hi + 1, (n_req,), generator=g).tolist() if n_req > 1 else [new_hi]
    held, want = [-(-c // page) for c in cached], [-(-(c + n) // page) for c, n in zip(cached, new)]
    n_blocks = max(want) if not short else max(1, max(want) - 1)      # some requests pass the table
    n_blocks = max(n_blocks, max(held), 1)
    ids = torch.randperm(sum(held) + sum(want) + 10, generator=g).tolist()
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-3] * (n_blocks - h))
        at += h
    free = ids[at:at + max(0, sum(want) - sum(held) - short) + 2]
    T = max(0, sum(new) - cut + (7 if not cut else 0))
    ref = plan_reference(cached, new, page, free, 2, table, T, n_blocks)
    plan, n_used = run_plan(cuda, cached, new, page, free, 2, table, T)
    assert plan.q_start.tolist() == ref[1] and plan.kv_len.tolist() == ref[2] and n_used.item() == ref[5]
    assert plan.block_table.tolist() == ref[0]
    assert plan.slots.tolist() == ref[3] and plan.positions.tolist() == ref[4]
    assert S.take_device_error() == 0


def test_plan_negative_lengths_are_reported(cuda):
    plan, n_used = run_plan(cuda, [4, -5, 3], [2, 2, -1], 4, [50, 51, 52], 0, [[7, -1], [-1, -1], [8, -1]], 6)
    assert S.take_device_error() == 2
    assert plan.slots.tolist()[:2] == [50 * 4, 50 * 4 + 1] and plan.kv_len.tolist()[0] == 6


@pytest.mark.parametrize("n_req,lo,hi,steps", [(3, 1, 1, 40), (1200, 0, 3, 6), (50, 100, 400, 3), (1, 9000, 9000, 2)])
def test_plan_over_its_own_lengths(cuda, n_req, lo, hi, steps):
    """One step's kv_len is the next one's cached_len, in place; rows on both
    sides of the one-kernel limit.  New lengths lie in q_start every other step."""
    page, g = 16, torch.Generator().manual_seed(n_req)
    news = [torch.randint(lo, hi + 1, (n_req,), generator=g) for _ in range(steps)]
    blocks = -(-hi * steps // page) + 1
    T = n_req * hi + 3
    pages = torch.randperm(n_req * blocks, generator=g).tolist()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    plan = paged.PagedPlan(torch.full((n_req, blocks), -1, dtype=torch.int32, device=cuda), page, T)
    free, used = i32(pages), i32([0])
    cached, table, taken = [0] * n_req, [[-1] * blocks for _ in range(n_req)], 0
    for step, new in enumerate(news):
        new_len = new.to(torch.int32).to(cuda)
        if step % 2:
            plan.q_start[:n_req] = new_len
            new_len = plan.q_start[:n_req]
        plan.build(plan.kv_len, new_len, free, used)
        table, start, cached, slots, pos, taken = plan_reference(cached, new.tolist(), page, pages, taken, table, T, blocks)
        assert plan.kv_len.tolist() == cached and plan.q_start.tolist() == start and used.item() == taken
        assert plan.block_table.tolist() == table
        assert plan.slots.tolist() == slots and plan.positions.tolist() == pos
    assert S.take_device_error() == 0


# ---- append ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rope", ["none", "pairs", "halves"])
@pytest.mark.parametrize("T,H,K,D,page,layout", [(1, 1, 1, 8, 1, "heads"), (3, 4, 2, 64, 16, "heads"), (257, 8, 8, 128, 64, "tokens"),
                                                 (40, 6, 2, 80, 4, "tokens"), (17, 5, 1, 256, 16, "odd")])
def test_append(cuda, dtype, rope, T, H, K, D, page, layout):
    g = torch.Generator(device=cuda).manual_seed(T + D)
    extra = 3 if layout == "odd" else 0         # rows at odd addresses: no wide loads
    x = torch.randn((T, (H + 2 * K) * D + extra), generator=g, device=cuda) * 3
    x = x[:, extra:]
    q, k, v = x[:, :H * D].unflatten(1, (H, D)), x[:, H * D:(H + K) * D].unflatten(1, (K, D)), x[:, (H + K) * D:].unflatten(1, (K, D))
    P = T // page + 3
    if layout == "tokens":                       # page by token by head in memory
        caches = [torch.randn((P, page, K, D), generator=g, device=cuda).to(dtype).transpose(1, 2) for _ in range(2)]
    else:
        caches = [torch.randn((P, K, page, D), generator=g, device=cuda).to(dtype) for _ in range(2)]
    slots = torch.randperm(P * page, generator=g, device=cuda)[:T].contiguous()
    if T > 2:
        slots[1] = -1
    pos = torch.randint(0, 500, (T,), generator=g, device=cuda).to(torch.int32)
    table = paged.rope_table(500, D, device=cuda)
    want = [c.clone() for c in caches]
    kv = paged.PagedKV(*caches)
    got_q = paged.append(kv, k, v, slots, q=q, positions=pos, rope=None if rope == "none" else table, halves=rope == "halves")

    def turned(y):
        y = y.double()
        if rope == "none":
            return y, torch.zeros_like(y)
        cs = table.double()[pos.long()][:, None]
        c, s = cs[..., :D // 2], cs[..., D // 2:]
        a, b = (y[..., :D // 2], y[..., D // 2:]) if rope == "halves" else (y[..., 0::2], y[..., 1::2])
        out, size = [a * c - b * s, a * s + b * c], [(a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()]
        join = (lambda z: torch.cat(z, -1)) if rope == "halves" else (lambda z: torch.stack(z, -1).flatten(-2))
        return join(out), join(size)

    def near(got, y):
        ref, size = turned(y)
        # two products and a sum, each off by 2^-24 of its size at most, then one rounding
        tol = size * 2.0 ** -23 + (ref.abs() + size * 2.0 ** -23) * torch.finfo(dtype).eps / 2 + 2.0 ** -25
        assert ((got.double() - ref).abs() <= tol).all()

    near(got_q, q)
    for cache, w, y in zip(caches, want, (k, None)):
        for t in range(T):
            s = slots[t].item()
            if s < 0:
                continue
            row = cache[s // page, :, s % page]
            if y is not None:
                near_rows = row
                ref, size = turned(y)
                tol = size[t] * 2.0 ** -23 + (ref[t].abs() + size[t] * 2.0 ** -23) * torch.finfo(dtype).eps / 2 + 2.0 ** -25
                assert ((near_rows.double() - ref[t]).abs() <= tol).all()
            else:
                assert torch.equal(row, v[t].to(dtype))
            w[s // page, :, s % page] = row
    assert all(torch.equal(c, w) for c, w in zip(caches, want))   # nothing else was written
    assert S.take_device_error() == 0


def test_append_outside_is_skipped_and_reported(cuda):
    kv = paged.PagedKV(torch.zeros((2, 1, 4, 16), dtype=F16, device=cuda), torch.zeros((2, 1, 4, 16), dtype=F16, device=cuda))
    x = torch.ones((4, 1, 16), device=cuda)
    paged.append(kv, x, x, torch.tensor([8, -2, 1 << 40, 3], device=cuda))
    assert S.take_device_error() == 2
    want = torch.zeros((2, 1, 4, 16), dtype=F16, device=cuda)
    want[0, 0, 3] = 1
    assert torch.equal(kv.k, want) and torch.equal(kv.v, want)
    far = torch.tensor([10, -1, 0, 0], dtype=torch.int32, device=cuda)
    paged.append(kv, x, x, torch.arange(4, device=cuda), positions=far, rope=paged.rope_table(8, 16, device=cuda))
    assert S.take_device_error() == 2


# ---- attention ------------------------------------------------------------------------

class Problem:
    """Requests (new tokens, keys) over a cache whose other slots hold NaN."""

    def __init__(self, dev, lens, H, K, D, page, dtype, layout="heads", pad=0, seed=0, spread=1.0):
        g = torch.Generator(device=dev).manual_seed(seed)
        self.lens, self.page, self.H, self.K, self.D = lens, page, H, K, D
        want = [-(-m // page) for _, m in lens]
        P = sum(want) + 2
        ids = torch.randperm(P, generator=g, device=dev).tolist()
        blocks = max(1, max(want))
        table, at = [], 0
        for w in want:
            table.append(ids[at:at + w] + [-1] * (blocks - w))
            at += w
        shape = (P, page, K, D) if layout == "tokens" else (P, K, page, D)
        self.k, self.v = (torch.full(shape, math.nan, dtype=dtype, device=dev) for _ in range(2))
        if layout == "tokens":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.rows = []
        for (n, m), row in zip(lens, table):
            kr, vr = (torch.randn((m, K, D), generator=g, device=dev).to(dtype) for _ in range(2))
            self.rows.append((kr, vr))
            for b in range(-(-m // page)):
                part = slice(b * page, min(m, (b + 1) * page))
                self.k[row[b], :, :part.stop - part.start] = kr[part].transpose(0, 1)
                self.v[row[b], :, :part.stop - part.start] = vr[part].transpose(0, 1)
        T = sum(n for n, _ in lens)
        self.T = T
        self.q = (torch.randn((T + pad, H, D), generator=g, device=dev) * spread).to(dtype)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        starts = [0]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.table, self.starts, self.q_start, self.kv_len = i32(table), starts, i32(starts), i32([m for _, m in lens])
        self.kv = paged.PagedKV(self.k, self.v)

    def run(self, causal=True, max_new=None, **kw):
        max_new = max(n for n, _ in self.lens) if max_new is None else max_new
        return paged.attention(self.q, self.kv, self.table, self.q_start, self.kv_len, max_new, causal=causal, **kw)

    def check(self, out, causal=True, scale=None):
        """Within: half a step of the output's type; half a step of the cache's
        type for every softmax weight; 1e-4 of the weighted |v| for fp32 scores
        (128 products of size 8: 128 * 2^-24 * 8 = 6e-5), the exponential and sums."""
        scale = self.D ** -0.5 if scale is None else scale
        half = torch.finfo(self.q.dtype).eps / 2
        for i, (n, m) in enumerate(self.lens):
            lo, hi = self.starts[i], self.starts[i + 1]
            if n == 0:
                continue
            got = out[lo:hi].double()
            if m == 0:
                assert (got == 0).all()
                continue
            k, v = (x.double().repeat_interleave(self.H // self.K, 1) for x in self.rows[i])
            s = torch.einsum("nhd,mhd->hnm", self.q[lo:hi].double(), k) * scale
            if causal:
                sees = torch.arange(m, device=s.device)[None] <= m - n + torch.arange(n, device=s.device)[:, None]
                s = s.masked_fill(~sees, -math.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            ref = torch.einsum("hnm,mhd->nhd", p, v)
            size = torch.einsum("hnm,mhd->nhd", p, v.abs())
            tol = 1.01 * (half * ref.abs() + (half + 1e-4) * size) + 2.0 ** -25
            worst = ((got - ref).abs() - tol).max().item()
            assert worst <= 0, (i, n, m, worst)
        assert S.take_device_error() == 0


DECODE = [(1, 1), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (0, 30), (1, 0), (1, 383), (1, 384), (1, 385), (1, 1000), (0, 0)]
CHUNK = [(1, 1), (5, 5), (7, 100), (64, 64), (65, 130), (33, 700), (0, 12), (9, 0), (12, 7), (130, 131)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D,page", [(1, 1, 64, 16), (8, 2, 128, 16), (8, 8, 64, 1), (15, 3, 80, 8), (7, 1, 128, 64), (16, 1, 96, 128),
                                        (4, 2, 256, 16), (2, 2, 8, 2), (34, 2, 128, 32)])
def test_attention_one_token(cuda, dtype, H, K, D, page):
    p = Problem(cuda, DECODE, H, K, D, page, dtype)
    p.check(p.run())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D,page", [(1, 1, 128, 16), (8, 2, 128, 16), (6, 2, 64, 1), (5, 1, 80, 8), (4, 4, 256, 64), (3, 1, 96, 128)])
def test_attention_chunks(cuda, dtype, causal, H, K, D, page):
    p = Problem(cuda, CHUNK, H, K, D, page, dtype, seed=1)
    p.check(p.run(causal=causal), causal=causal)


MANY = [(300, 300), (257, 1000), (128, 2500), (129, 129), (256, 256), (1, 70), (400, 380), (90, 0), (16, 500), (513, 900)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D,page", [(1, 1, 64, 16), (1, 1, 128, 16), (4, 2, 128, 1), (3, 1, 80, 32), (8, 1, 64, 128)])
def test_attention_many_rows(cuda, dtype, causal, H, K, D, page):
    """Tiles of 256 rows, the last one or its lower half partly filled; keys that
    end inside a block; rows that see nothing (fewer keys than new tokens)."""
    p = Problem(cuda, MANY, H, K, D, page, dtype, seed=12)
    p.check(p.run(causal=causal), causal=causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,H,K,D,page", [(F16, 8, 8, 128, 16), (BF16, 8, 8, 64, 32), (F16, 16, 8, 80, 4)])
def test_attention_half_filled_tiles(cuda, dtype, causal, H, K, D, page):
    """Rows for one half of a 256-row tile only, over one to nine blocks of 128
    keys, so many of them that a CTA takes several, whole tiles in between."""
    lens = [(n, m) for m in (1, 128, 129, 256, 300, 384, 385, 520, 1030, 1152) for n in (128 * K // H, 25, 64)]
    lens += [(128 * K // H - 1, 100), (300, 700), (127, 64), (33, 2000), (1, 900), (256, 513), (26, 0), (31, 3000)]
    p = Problem(cuda, lens, H, K, D, page, dtype, seed=20, spread=4.0)
    out = p.run(causal=causal)
    p.check(out, causal=causal)
    assert torch.equal(out, p.run(causal=causal))


@pytest.mark.parametrize("H,K,D,n,m", [(4, 1, 128, 1, 20000), (1, 1, 64, 1, 50001), (32, 8, 128, 3, 3001), (2, 1, 256, 1, 9000),
                                       (8, 8, 128, 300, 2500), (2, 1, 64, 1000, 1000), (1, 1, 128, 2, 30000)])
def test_attention_split_over_ctas(cuda, H, K, D, n, m):
    """Few rows and many keys: tiles shared by many CTAs, then joined."""
    for dtype in (F16, BF16):
        p = Problem(cuda, [(n, m)], H, K, D, 16, dtype, seed=2)
        out = p.run()
        p.check(out)
        assert torch.equal(out, p.run())        # the joining order does not depend on timing


def test_attention_uneven_batch(cuda):
    g = torch.Generator().manual_seed(5)
    lens = [(1, int(m)) for m in torch.randint(1, 3000, (70,), generator=g)] + [(1, 40000)]
    p = Problem(cuda, lens, 8, 2, 128, 16, BF16, seed=3)
    p.check(p.run())
    lens = [(int(n), int(m)) for n, m in zip(torch.randint(0, 9, (40,), generator=g), torch.randint(9, 2000, (40,), generator=g))]
    p = Problem(cuda, lens + [(400, 1500)], 8, 2, 64, 32, F16, seed=4)
    p.check(p.run())
    p.check(p.run(max_new=1))                   # a bound that is too small costs time only


@pytest.mark.parametrize("lens", [DECODE, CHUNK])
def test_attention_layouts_and_rows_left_alone(cuda, lens):
    p = Problem(cuda, lens, 8, 2, 128, 16, F16, layout="tokens", pad=5, seed=6)
    wide = torch.zeros((p.T + 5, 8 * 128 + 24), dtype=F16, device=cuda)
    wide[:, :1024] = p.q.flatten(1)
    p.q = wide[:, :1024].unflatten(1, (8, 128))
    out = torch.full((p.T + 5, 8 * 128 + 8), 7.0, dtype=F16, device=cuda)
    got = p.run(out=out[:, :1024].unflatten(1, (8, 128)))
    p.check(got)
    assert (out[p.T:] == 7).all() and (out[:, 1024:] == 7).all()


def test_attention_large_scores_and_scale(cuda):
    """Score spans of hundreds: weights far below the largest, maxima that move."""
    p = Problem(cuda, [(1, 900), (70, 500)], 4, 2, 128, 16, F16, seed=7, spread=8.0)
    out = p.run(scale=0.5)
    # scores up to ~8 * 11 * 4 * 0.5: their fp32 error is 8 times that of check()'s allowance
    half = torch.finfo(F16).eps / 2
    for i, (n, m) in enumerate(p.lens):
        lo, hi = p.starts[i], p.starts[i + 1]
        k, v = (x.double().repeat_interleave(2, 1) for x in p.rows[i])
        s = torch.einsum("nhd,mhd->hnm", p.q[lo:hi].double(), k) * 0.5
        s = s.masked_fill(~(torch.arange(m, device=cuda)[None] <= m - n + torch.arange(n, device=cuda)[:, None]), -math.inf)
        w = torch.softmax(s, -1)
        ref, size = torch.einsum("hnm,mhd->nhd", w, v), torch.einsum("hnm,mhd->nhd", w, v.abs())
        assert ((out[lo:hi].double() - ref).abs() <= 1.01 * (half * ref.abs() + (half + 8e-4) * size) + 2.0 ** -25).all()


@pytest.mark.parametrize("scale", [2.0 ** -7, 2.0 ** -4])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D,lens", [(4, 1, 128, [(1, 900), (1, 20000), (1, 70)]), (4, 1, 64, [(4, 900), (3, 5000)]),
                                        (4, 2, 128, [(12, 900), (10, 6000)]), (2, 1, 256, [(40, 900), (9, 5000)]),
                                        (4, 2, 128, [(200, 900), (300, 5000), (20, 3000), (1, 600)])])
def test_attention_far_scores(cuda, dtype, scale, H, K, D, lens):
    """Scores of +-2^30 + 128 j, j of 0 to 11, which fp32 holds exactly (2^30 has
    steps of 128): times the scale they are +-2^23 + j and +-2^26 + 8 j, where
    fp32 has steps of one to eight.  The weights are e^j and e^8j all the same."""
    p = Problem(cuda, lens, H, K, D, 16, dtype, seed=21)
    g = torch.Generator(device=cuda).manual_seed(22)
    p.q.zero_()
    p.q[..., 0], p.q[..., 1] = 2.0 ** 15, 8.0
    for i, ((_, m), (kr, _)) in enumerate(zip(p.lens, p.rows)):
        kr[..., 0] = 2.0 ** 15 if i % 2 else -2.0 ** 15
        kr[..., 1] = 16 * torch.randint(0, 12, kr.shape[:2], generator=g, device=cuda).to(dtype)
        at = torch.arange(m, device=cuda)
        p.k[p.table[i, at // 16].long(), :, at % 16] = kr
    out = p.run(scale=scale)
    # the scale is rounded twice on its way: 17 * 8 octaves * 2^-23 = 2e-5 of a weight, inside check()'s 1e-4
    p.check(out, scale=scale)


def test_attention_infinities_stay_in_their_request(cuda):
    p = Problem(cuda, [(1, 100), (3, 80), (1, 70)], 4, 2, 64, 16, F16, seed=8)
    clean = p.run().clone()
    page, place = p.table[1, 79 // 16].item(), 79 % 16
    p.k[page, :, place] = math.inf
    p.v[page, :, place] = math.nan
    out = p.run()
    assert torch.equal(out[0], clean[0]) and torch.equal(out[4], clean[4])
    assert out[3].isnan().all()


def test_attention_bad_lengths_and_pages_are_reported(cuda):
    p = Problem(cuda, [(1, 40), (1, 40)], 2, 1, 64, 16, F16, seed=9)
    want = p.run().clone()
    table = p.table.clone()
    table[1, 1] = p.kv.n_pages
    out = paged.attention(p.q, p.kv, table, p.q_start, p.kv_len, 1)
    assert S.take_device_error() == 2 and torch.equal(out[0], want[0])
    out = paged.attention(p.q, p.kv, p.table, p.q_start, torch.tensor([40, 1000], dtype=torch.int32, device=cuda), 1)
    assert S.take_device_error() == 2 and torch.equal(out[0], want[0])
    out = paged.attention(p.q, p.kv, p.table, torch.tensor([0, 1, 900], dtype=torch.int32, device=cuda), p.kv_len, 1)
    assert S.take_device_error() == 2 and torch.equal(out[0], want[0])


def test_attention_streams_and_graphs(cuda):
    """Two calls in flight on two streams; a captured call replayed with other
    lengths; two captured calls replayed after each other."""
    a = Problem(cuda, [(1, 5000), (1, 3)], 8, 2, 128, 16, F16, seed=10)
    b = Problem(cuda, [(200, 4000)], 8, 2, 128, 16, F16, seed=11)
    ra, rb = a.run().clone(), b.run().clone()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(s1):
            oa = a.run()
        with torch.cuda.stream(s2):
            ob = b.run()
    torch.cuda.synchronize()
    assert torch.equal(oa, ra) and torch.equal(ob, rb)
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        oa = a.run()
    with torch.cuda.graph(gb):
        ob = b.run()
    for _ in range(3):
        ga.replay()
        gb.replay()
    torch.cuda.synchronize()
    assert torch.equal(oa, ra) and torch.equal(ob, rb)
    a.kv_len.copy_(torch.tensor([4100, 1], dtype=torch.int32))
    ga.replay()
    short = Problem(cuda, [(1, 5000), (1, 3)], 8, 2, 128, 16, F16, seed=10)
    short.kv_len.copy_(a.kv_len)
    assert torch.equal(oa, short.run())


@pytest.mark.parametrize("n_req,chunk", [(130, 0), (700, 0), (400, 90)])
def test_attention_many_requests(cuda, n_req, chunk):
    """More requests than a CTA has threads; with a chunk both kernels run."""
    g = torch.Generator().manual_seed(n_req)
    lens = [(int(n), int(m)) for n, m in zip(torch.randint(0, 3, (n_req,), generator=g), torch.randint(0, 200, (n_req,), generator=g))]
    if chunk:
        lens[n_req // 2] = (chunk, 300)
    p = Problem(cuda, lens, 4, 2, 64, 16, BF16, seed=13)
    p.check(p.run())


@pytest.mark.parametrize("n", [1, 90])
def test_attention_rows_before_the_first_request(cuda, n):
    p = Problem(cuda, [(n, 100), (n, 450)], 4, 2, 128, 16, F16, pad=6, seed=14)
    p.q = p.q.roll(4, 0)
    p.q_start += 4
    p.starts = [s + 4 for s in p.starts]
    out = torch.full_like(p.q, 3.0)
    p.check(p.run(out=out))
    assert (out[:4] == 3).all() and (out[4 + 2 * n:] == 3).all()


@pytest.mark.parametrize("n,page", [(1, 16), (200, 16), (200, 4)])
def test_attention_and_append_far_into_a_large_cache(cuda, n, page):
    """Pages that lie more than 2^32 bytes apart."""
    K, D, step = 2, 128, 1 << 27
    blocks, far = -(-300 // page), 18
    base = torch.zeros((far + 1) * step, dtype=F16, device=cuda)
    shape, stride = (far + 1, K, page, D), (step, page * D, D, 1)
    spread = [base.as_strided(shape, stride, o) for o in (0, 1 << 20)]
    order = list(range(far, -1, -1))[:blocks]       # the last page first
    m = min(300, len(order) * page)
    p = Problem(cuda, [(n, m)], 4, K, D, page, F16, seed=16)
    kr, vr = p.rows[0]
    kv = paged.PagedKV(*spread)
    pos = torch.arange(m, device=cuda)
    slots = torch.tensor(order, device=cuda)[pos // page] * page + pos % page
    paged.append(kv, kr.float(), vr.float(), slots)
    table = torch.tensor([order], dtype=torch.int32, device=cuda)
    assert torch.equal(spread[0][order[0], :, 0], kr[0]) and torch.equal(spread[1][order[1], :, 0], vr[page])
    n_new = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    out = paged.attention(p.q, kv, table, n_new, p.kv_len, n)
    p.check(out)


def test_attention_bad_page_of_a_chunk_is_reported(cuda):
    p = Problem(cuda, [(100, 300), (100, 300)], 4, 2, 128, 16, F16, seed=17)
    want = p.run().clone()
    table = p.table.clone()
    table[1, 3], table[1, 7] = -5, 1 << 30
    out = paged.attention(p.q, p.kv, table, p.q_start, p.kv_len, 100)
    assert S.take_device_error() == 2 and torch.equal(out[:100], want[:100])


def test_refused_tensors(cuda):
    p = Problem(cuda, [(1, 40), (1, 40)], 2, 1, 64, 16, F16, seed=18)
    args = (p.q_start, p.kv_len, 1)
    with pytest.raises(AssertionError):      # one row for all requests
        paged.attention(p.q, p.kv, p.table[:1].expand(2, -1), *args)
    with pytest.raises(AssertionError):
        paged.attention(p.q.float(), p.kv, p.table, *args)
    with pytest.raises(AssertionError):
        paged.attention(p.q, p.kv, p.table, p.q_start[:2], p.kv_len, 1)
    with pytest.raises(AssertionError):
        paged.attention(p.q.cpu(), p.kv, p.table, *args)
    with pytest.raises(S.SmeaiError, match="workspace"):
        big = torch.full((2, 100), -1, dtype=torch.int32, device=cuda)
        paged.attention(p.q, p.kv, big, *args, workspace=torch.empty(256, dtype=torch.uint8, device=cuda))
    with pytest.raises(S.SmeaiError, match="scale"):
        paged.attention(p.q, p.kv, p.table, *args, scale=0.0)
    one = p.k.new_empty((1, 1, 1, 64)).expand(3, -1, -1, -1)
    with pytest.raises(S.SmeaiError, match="overlap"):
        paged.append(paged.PagedKV(one, one), torch.zeros((1, 1, 64), device=cuda), torch.zeros((1, 1, 64), device=cuda),
                     torch.zeros(1, dtype=torch.int64, device=cuda))


@pytest.mark.parametrize("H,K,D,page,lens", [(8, 2, 128, 16, [(300, 3000), (40, 5000), (1, 900)]), (8, 8, 64, 32, [(64, 4000)] * 30),
                                             (4, 2, 128, 4, [(300, 3000), (40, 5000)])])
def test_attention_gives_up_when_a_wait_runs_out(cuda, H, K, D, page, lens):
    """With a limit of a nanosecond the first wait of the tensor-core kernel that
    is not over at once runs out.  The call ends, says so, and the next one is
    right: nothing of the first was left in flight, and tensor memory was freed."""
    p = Problem(cuda, lens, H, K, D, page, F16, seed=23)
    want = p.run().clone()
    assert S.take_device_error() == 0
    try:
        S.lib().smeai_set_wait_timeouts(1, 0)
        for _ in range(5):
            p.run()
    finally:
        S.lib().smeai_set_wait_timeouts(0, 0)
    torch.cuda.synchronize()
    assert S.take_device_error() == 1
    for _ in range(3):
        assert torch.equal(p.run(), want)
    p.check(want)


def test_workspace_sizes_are_not_collected(cuda):
    """A server's steps differ in their sizes for ever; a cache keeps a bounded number of answers."""
    kv = paged.PagedKV.empty(4, 2, 16, 64, device=cuda)
    sizes = [paged.attention_workspace(kv, 8, t, 3, 100, t) for t in range(1, 1000)]
    assert len(kv._workspace) <= 64
    assert sizes == [paged.attention_workspace(kv, 8, t, 3, 100, t) for t in range(1, 1000)] and min(sizes) > 0


# ---- every head_dim and tile that the documentation allows ---------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D,page", [(4, 2, 24, 16), (3, 1, 40, 4), (8, 1, 104, 8), (4, 2, 136, 16), (9, 1, 192, 1), (2, 2, 248, 64)])
def test_attention_one_token_odd_head_dims(cuda, dtype, H, K, D, page):
    p = Problem(cuda, DECODE + [(1, 9000)], H, K, D, page, dtype, seed=24)
    p.check(p.run())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,K,D,page", [(4, 2, 136, 16), (3, 1, 192, 4), (2, 2, 216, 32)])
def test_attention_chunks_odd_head_dims(cuda, causal, H, K, D, page):
    """64-row tiles over padded columns, some of them split over CTAs."""
    p = Problem(cuda, CHUNK + [(40, 6000)], H, K, D, page, BF16, seed=25)
    p.check(p.run(causal=causal), causal=causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,H,K,D,page", [(F16, 2, 1, 8, 16), (BF16, 2, 1, 8, 4), (F16, 1, 1, 24, 4), (BF16, 1, 1, 24, 64), (F16, 3, 1, 40, 8),
                                              (F16, 2, 2, 72, 16), (BF16, 1, 1, 88, 128), (F16, 2, 1, 104, 2), (BF16, 2, 1, 120, 32)])
def test_attention_many_rows_odd_head_dims(cuda, causal, dtype, H, K, D, page):
    """The tensor-core kernel's boxes and tiles are wider than the head."""
    p = Problem(cuda, MANY, H, K, D, page, dtype, seed=26)
    p.check(p.run(causal=causal), causal=causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D", [(4, 1, 128), (6, 2, 64), (8, 1, 96), (1, 1, 128)])
def test_attention_drafts(cuda, dtype, causal, H, K, D):
    """Tiles of 24 rows: several tokens a request, so several limits in a tile;
    rows that the tile has too many; long requests split and joined."""
    most = 24 * K // H
    lens = [(1 + i % most, m) for i, m in enumerate((1, 30, 64, 65, 190, 383, 384, 385, 700, 1000, 2500, 3001))]
    lens += [(most, 20000), (most, most), (most, 0), (0, 70), (most - 1, 9000)]
    p = Problem(cuda, lens, H, K, D, 16, dtype, seed=27)
    assert 16 < most * (H // K) <= 24
    out = p.run(causal=causal)
    p.check(out, causal=causal)
    assert torch.equal(out, p.run(causal=causal))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D,n", [(8, 2, 128, 1), (4, 1, 64, 4), (2, 1, 128, 8), (16, 1, 80, 1), (4, 2, 256, 3)])
def test_attention_of_up_to_16_rows_keeps_its_weights(cuda, dtype, H, K, D, n):
    """Up to 16 rows a request the weights keep what their rounding leaves, so
    the result is off by its own rounding and that of fp32 alone."""
    p = Problem(cuda, [(n, m) for m in (n, 40, 100, 500, 3000, 20000)], H, K, D, 16, dtype, seed=28)
    out = p.run()
    half = torch.finfo(dtype).eps / 2
    for i, (n, m) in enumerate(p.lens):
        lo, hi = p.starts[i], p.starts[i + 1]
        k, v = (x.double().repeat_interleave(H // K, 1) for x in p.rows[i])
        s = torch.einsum("nhd,mhd->hnm", p.q[lo:hi].double(), k) * D ** -0.5
        s = s.masked_fill(torch.arange(m, device=cuda)[None] > m - n + torch.arange(n, device=cuda)[:, None], -math.inf)
        w = torch.softmax(s, -1)
        ref, size = torch.einsum("hnm,mhd->nhd", w, v), torch.einsum("hnm,mhd->nhd", w, v.abs())
        # as check(), with the square of half a step for the weights: what one rounding leaves, rounded again
        assert ((out[lo:hi].double() - ref).abs() <= 1.01 * (half * ref.abs() + (half * half + 1e-4) * size) + 2.0 ** -25).all(), (n, m)


@pytest.mark.parametrize("D", [8, 24, 40, 72, 136, 248])
@pytest.mark.parametrize("rope", ["pairs", "halves"])
def test_append_odd_head_dims(cuda, rope, D):
    """Against the same values appended by hand."""
    T, H, K, page = 37, 3, 2, 8
    g = torch.Generator(device=cuda).manual_seed(D)
    q, k, v = (torch.randn((T, n, D), generator=g, device=cuda) for n in (H, K, K))
    kv = paged.PagedKV(*(torch.zeros((8, K, page, D), dtype=F16, device=cuda) for _ in range(2)))
    slots, pos = torch.randperm(8 * page, generator=g, device=cuda)[:T].contiguous(), torch.arange(T, dtype=torch.int32, device=cuda) + 100
    table = paged.rope_table(200, D, device=cuda)
    got = paged.append(kv, k, v, slots, q=q, positions=pos, rope=table, halves=rope == "halves")
    cs = table.double()[pos.long()][:, None]
    c, s = cs[..., :D // 2], cs[..., D // 2:]
    for out, x in ((got, q), (kv.k[slots // page, :, slots % page], k)):
        y = x.double()
        a, b = (y[..., :D // 2], y[..., D // 2:]) if rope == "halves" else (y[..., 0::2], y[..., 1::2])
        ref = [a * c - b * s, a * s + b * c]
        ref = torch.cat(ref, -1) if rope == "halves" else torch.stack(ref, -1).flatten(-2)
        # fp32 products and sum of values below 6 (3 * 6 * 2^-24 < 2^-19), then one rounding
        assert ((out.double() - ref).abs() <= 2.0 ** -11 * ref.abs() + 2.0 ** -19 + 2.0 ** -25).all()
    assert torch.equal(kv.v[slots // page, :, slots % page], v.half())
    assert S.take_device_error() == 0


@pytest.mark.parametrize("H,K,D,lens", [(4, 1, 128, [(1, 900), (1, 20000)]), (4, 2, 128, [(12, 900), (10, 6000)]),
                                        (2, 1, 256, [(40, 900), (9, 5000)]), (4, 2, 128, [(200, 900), (300, 5000), (20, 3000)])])
def test_attention_of_the_largest_values(cuda, H, K, D, lens):
    """A mean of values is no larger than they are: with values of +-65504 the
    rounding of the weights must not carry a row past fp16's range.  An infinite
    value still gives infinities."""
    p = Problem(cuda, lens, H, K, D, 16, F16, seed=29, spread=3.0)
    for i, ((_, m), (_, vr)) in enumerate(zip(p.lens, p.rows)):
        vr.copy_(torch.where(torch.arange(D, device=cuda) % 3 > 0, 65504.0, -65504.0).half().expand_as(vr))
        at = torch.arange(m, device=cuda)
        p.v[p.table[i, at // 16].long(), :, at % 16] = vr
    out = p.run()
    p.check(out)
    p.v[p.table[0, 0].item(), :, 0, :8] = math.inf
    out = p.run()
    n = p.lens[0][0]
    assert not out[:n, :, :8].isfinite().any() and out[:n, :, 8:].isfinite().all() and out[n:].isfinite().all()
    assert S.take_device_error() == 0
