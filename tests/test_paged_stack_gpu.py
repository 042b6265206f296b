"""The paged operators as a serving loop uses them: plan, append, attention and
the residual norm in the decode stack, prompts in chunks beside decoding."""
import math

import pytest
import torch

import smeai_b200 as S
from smeai_b200 import paged
from smeai_b200.stack import Q2KDecodeStack

pytestmark = pytest.mark.gpu


def turned(y, pos, base=10000.0):
    """RoPE of adjacent pairs in 64 bits."""
    D = y.shape[-1]
    angle = pos.double()[:, None, None] * base ** (-torch.arange(0, D, 2, device=y.device, dtype=torch.float64) / D)
    a, b = y.double()[..., 0::2], y.double()[..., 1::2]
    return torch.stack([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1).flatten(-2)


class Checked:
    """paged.append and paged.attention with every result held against 64 bits
    on the values that the step itself produced."""

    def __init__(self, monkeypatch, plan):
        self.plan, self.append, self.attention, self.calls = plan, paged.append, paged.attention, 0
        monkeypatch.setattr(paged, "append", self.check_append)
        monkeypatch.setattr(paged, "attention", self.check_attention)

    def check_append(self, kv, k, v, slots, q=None, positions=None, rope=None):
        out = self.append(kv, k, v, slots, q=q, positions=positions, rope=rope)
        at = (slots >= 0).nonzero()[:, 0]
        s, page = slots[at], kv.page_size
        half = torch.finfo(kv.dtype).eps / 2
        for got, src in ((kv.k[s // page, :, s % page], k[at]), (out[at], q[at])):
            ref, size = turned(src, positions[at]), src.double().abs().amax()
            # cosines, products and the sum are off by 2^-24 of the values at most, five times; then one rounding
            assert ((got.double() - ref).abs() <= half * ref.abs() + 5 * 2.0 ** -24 * size + 2.0 ** -25).all()
        assert torch.equal(kv.v[s // page, :, s % page], v[at].to(kv.dtype))
        return out

    def check_attention(self, q, kv, table, q_start, kv_len, max_new):
        out = self.attention(q, kv, table, q_start, kv_len, max_new)
        half = torch.finfo(kv.dtype).eps / 2
        for i, m in enumerate(kv_len.tolist()):
            lo, hi = q_start[i].item(), q_start[i + 1].item()
            n = hi - lo
            if n == 0:
                continue
            if m == 0:
                assert (out[lo:hi] == 0).all()
                continue
            pages = table[i, :-(-m // kv.page_size)].long()
            k, v = (c[pages].transpose(1, 2).flatten(0, 1)[:m].double() for c in (kv.k, kv.v))
            s = torch.einsum("nhd,mhd->hnm", q[lo:hi].double(), k) * kv.head_dim ** -0.5
            s = s.masked_fill(torch.arange(m, device=s.device)[None] > m - n + torch.arange(n, device=s.device)[:, None], -math.inf)
            p = torch.softmax(s, -1)
            ref, size = torch.einsum("hnm,mhd->nhd", p, v), torch.einsum("hnm,mhd->nhd", p, v.abs())
            # the output's rounding, the weights' rounding, fp32 scores and sums (scores of size 30 at most)
            assert ((out[lo:hi].double() - ref).abs() <= 1.01 * (half * ref.abs() + (half + 1e-4) * size) + 2.0 ** -25).all()
        self.calls += 1
        return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_serving_steps(cuda, monkeypatch, dtype):
    st = Q2KDecodeStack(n_layers=2, hidden=1024, ffn=2816, vocab=2048, device=cuda, seed=21)
    page, blocks, B = 16, 30, 4
    caches = [paged.PagedKV.empty(60, 8, page, 128, dtype=dtype, device=cuda) for _ in range(2)]
    for c in caches:
        c.k.fill_(math.nan)
        c.v.fill_(math.nan)
    rope = paged.rope_table(1024, 128, device=cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    table, used = torch.full((B, blocks), -1, dtype=torch.int32, device=cuda), i32([0])
    pool = torch.randperm(60, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(torch.int32)
    g = torch.Generator(device=cuda).manual_seed(2)
    # a prompt in two chunks, one behind it, decoding, a request without tokens, a late long prompt (its 30 pages are 53 of
    # 60 in all), and at the end a request that passes the table's 30 pages
    cached = [0, 0, 0, 0]
    for new, served in (([200, 7, 0, 0], 4), ([100, 1, 1, 0], 4), ([1, 1, 1, 1], 4), ([3, 2, 16, 1], 4), ([1, 1, 1, 1], 4), ([1, 1, 1, 470], 4),
                        ([2, 1, 1, 40], 3)):
        T = sum(new) + 2                                     # two padded rows
        plan = paged.PagedPlan(table, page, T).build(i32(cached), i32(new), pool, used)
        with monkeypatch.context() as mp:
            checked = Checked(mp, plan)
            logits = st.step_cached(torch.randn((T, 1024), generator=g, device=cuda), plan, caches, max(new), rope=rope)
        assert checked.calls == 2 and logits.shape == (T, 2048)
        assert logits[:sum(new[:served])].isfinite().all()
        cached = [c + (n if i < served else 0) for i, (c, n) in enumerate(zip(cached, new))]
        assert plan.kv_len.tolist() == [c if i < served else 0 for i, c in enumerate(cached)]
    assert used.item() == sum(-(-c // page) for c in cached)
    assert S.take_device_error() == 0
    st.free()


def test_decoding_captured_and_replayed(cuda):
    """A decode step with its plan in one CUDA graph, lengths advanced in the
    graph: the same logits as the eager steps."""
    st = Q2KDecodeStack(n_layers=1, hidden=1024, ffn=2816, vocab=512, device=cuda, seed=22)
    B, page, steps = 3, 16, 20
    x = torch.randn((steps, B, 1024), generator=torch.Generator(device=cuda).manual_seed(3), device=cuda)
    new = torch.ones(B, dtype=torch.int32, device=cuda)
    pool = torch.arange(12, dtype=torch.int32, device=cuda).flip(0).contiguous()

    def fresh():
        caches = [paged.PagedKV.empty(12, 8, page, 128, device=cuda)]
        plan = paged.PagedPlan(torch.full((B, 2), -1, dtype=torch.int32, device=cuda), page, B)
        return caches, plan, torch.zeros(B, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)

    def step(state, xt):
        caches, plan, cached, used = state
        plan.build(cached, new, pool, used)
        logits = st.step_cached(xt, plan, caches, 1)
        cached += new
        return logits

    state = fresh()
    want = [step(state, x[t]) for t in range(steps)]
    state, xt = fresh(), x[0].clone()
    step(state, xt)                                          # set-up outside the capture
    torch.cuda.synchronize()
    state[2].zero_()
    state[3].zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = step(state, xt)
    state[2].zero_()
    state[3].zero_()
    for t in range(steps):
        xt.copy_(x[t])
        graph.replay()
        assert torch.equal(logits, want[t]), t
    assert state[2].tolist() == [steps] * B and S.take_device_error() == 0
    st.free()
