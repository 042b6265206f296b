"""Refusals of the paged-cache entry points: every argument check answers
before any GPU is looked at."""
import ctypes

import pytest

import smeai_b200 as S

BAD, SMALL, NONE = S.SME_AI_BAD_ARGUMENT, S.SME_AI_WORKSPACE_TOO_SMALL, S.SME_AI_UNSUPPORTED
P = 4096          # an aligned address that is never read


def cache(**kw):
    d = dict(k=P, v=P, type=S.KV_F16, page_size=16, n_kv_heads=2, head_dim=128, n_pages=10, page_stride=2 * 16 * 128,
             head_stride=16 * 128, token_stride=128)
    d.update(kw)
    return ctypes.byref(S.KVCache(**d))


def plan(**kw):
    d = dict(cached=P, new=P, n_req=4, page=16, free=P, n_free=8, used=P, used_out=P, table=P, ld=9, blocks=9, q_start=P, kv_len=P, slots=P,
             pos=P, T=5)
    d.update(kw)
    return S.lib().smeai_paged_plan(*d.values(), None)


@pytest.mark.parametrize("kw", [dict(cached=None), dict(new=None), dict(used=None), dict(used_out=None), dict(table=None), dict(free=None),
                                dict(q_start=None), dict(kv_len=None), dict(slots=None), dict(pos=None), dict(n_req=0), dict(n_req=8193),
                                dict(page=0), dict(page=12), dict(page=1 << 17), dict(n_free=-1), dict(T=-1), dict(T=1 << 31), dict(blocks=0),
                                dict(ld=8)])
def test_plan_refuses(kw):
    assert plan(**kw) == BAD and S.last_error().startswith("smeai_paged_plan")


BAD_CACHES = [dict(k=None), dict(v=None), dict(type=0), dict(page_size=0), dict(page_size=24), dict(page_size=1 << 17), dict(head_dim=0),
              dict(head_dim=100), dict(head_dim=264), dict(n_kv_heads=0), dict(n_pages=0), dict(n_pages=1 << 31), dict(k=P + 8), dict(v=P + 2),
              dict(token_stride=132), dict(token_stride=120), dict(head_stride=-128), dict(page_stride=64), dict(page_stride=1 << 41)]


def append(c=None, **kw):
    d = dict(k=P, ld_k=256, v=P, ld_v=256, q=P, ld_q=1024, heads=8, qo=P, ld_qo=1024, T=3, slots=P, pos=P, rope=P, n_rope=10, halves=0)
    d.update(kw)
    return S.lib().smeai_paged_append(c or cache(), *d.values(), None)


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_append_refuses_caches(kw):
    assert append(cache(**kw)) == BAD and S.last_error().startswith("smeai_paged_append")


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(slots=None), dict(T=-1), dict(ld_k=255), dict(ld_v=255), dict(q=None),
                                dict(qo=None), dict(heads=0), dict(ld_q=1023), dict(ld_qo=1016), dict(ld_qo=1028), dict(qo=P + 8),
                                dict(pos=None), dict(n_rope=0), dict(heads=1 << 16, ld_q=1 << 23, ld_qo=1 << 23)])
def test_append_refuses(kw):
    assert append(**kw) == BAD and S.last_error().startswith("smeai_paged_append")


def attention(c=None, **kw):
    d = dict(q=P, ld_q=1024, heads=8, T=3, q_start=P, kv_len=P, n_req=2, table=P, ld_table=7, blocks=7, max_new=2, scale=0.1, causal=1, out=P,
             ld_out=1024, ws=P, ws_bytes=1 << 40)
    d.update(kw)
    return S.lib().smeai_paged_attention(c or cache(), *d.values(), None)


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_attention_refuses_caches(kw):
    assert attention(cache(**kw)) == BAD and S.last_error().startswith("smeai_paged_attention")


@pytest.mark.parametrize("kw", [dict(q=None), dict(out=None), dict(q_start=None), dict(kv_len=None), dict(table=None), dict(heads=0),
                                dict(heads=7), dict(T=-1), dict(T=1 << 30), dict(n_req=0), dict(blocks=-1), dict(max_new=-1), dict(ld_q=1016),
                                dict(ld_q=1028), dict(ld_out=1000), dict(q=P + 8), dict(out=P + 4), dict(ld_table=6), dict(scale=0.0),
                                dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))])
def test_attention_refuses(kw):
    assert attention(**kw) == BAD and S.last_error().startswith("smeai_paged_attention")


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_attention_refuses_scales_that_overflow(scale):
    """Finite, but times log2(e), as the kernels use it, they are not."""
    assert attention(scale=scale) == BAD and "scale" in S.last_error()


def test_empty_calls_do_nothing():
    assert append(T=0, k=None) == 0 and attention(T=0, q=None) == 0


def add_rms(**kw):
    d = dict(x=P, ld_x=512, r=2 * P, ld_r=512, n=3, k=512, w=None, eps=1e-5, h=3 * P, ld_h=512, y=P)
    d.update(kw)
    return S.lib().smeai_add_rms_q8k_quantize(*d.values(), None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(r=None), dict(h=None), dict(y=None), dict(k=0), dict(k=300), dict(k=65536 + 256, ld_x=1 << 20, ld_r=1 << 20, ld_h=1 << 20),
                                dict(n=0), dict(n=1 << 31), dict(ld_x=511), dict(ld_r=256), dict(ld_h=500), dict(h=P, ld_h=1024), dict(h=2 * P, ld_h=513)])
def test_add_rms_refuses(kw):
    assert add_rms(**kw) == BAD and "add_rms_q8k_quantize" in S.last_error()


@pytest.mark.parametrize("off", [1, 2, 3])
def test_add_rms_refuses_blocks_off_their_words(off):
    """A byte view of any offset is a legal tensor; the blocks are written in words."""
    assert add_rms(y=P + off) == BAD and "aligned" in S.last_error()


def test_register_hand_over_is_one_instruction_a_warpgroup():
    """All warps of a warpgroup have to meet at the same setmaxnreg; the roles
    of the tensor-core kernel's last four warps differ, so it stands before them."""
    import os
    source = os.path.join(os.path.dirname(__file__), "..", "sme-ai-ops_b200", "csrc", "paged_attn_tc.cu")
    with open(source) as f:
        text = f.read()
    assert text.count("setmaxnreg.dec") == 1 and text.count("setmaxnreg.inc") == 1


@pytest.mark.skipif(__import__("torch").cuda.is_available(), reason="only meaningful on a host without a GPU")
def test_without_a_device():
    assert plan() == NONE and append() == NONE and attention() == NONE


def step_cached(caches, **plan):
    """Q2KDecodeStack.step_cached on a host without tensors on a GPU: its checks come first."""
    import types
    import torch
    from smeai_b200.stack import Q2KDecodeStack
    stack = types.SimpleNamespace(world=1, L=len(caches), H=256, eps=1e-5, V=32)
    plan = types.SimpleNamespace(**{**dict(n_tokens=3, page_size=16), **plan})
    return Q2KDecodeStack.step_cached(stack, torch.zeros((plan.n_tokens, 256)), plan, caches, 1)


@pytest.mark.parametrize("second,match", [(dict(page_size=32), "page size"), (dict(n_kv_heads=4), "alike"), (dict(head_dim=64), "alike")])
def test_step_refuses_caches_that_do_not_fit_the_plan(second, match):
    import types
    kv = lambda **kw: types.SimpleNamespace(**{**dict(page_size=16, n_kv_heads=2, head_dim=128), **kw})  # noqa: E731
    with pytest.raises(AssertionError, match=match):
        step_cached([kv(), kv(**second)])
    with pytest.raises(AssertionError, match="page size"):
        step_cached([kv(), kv()], page_size=8)


def test_step_without_tokens_does_nothing():
    import types
    kv = types.SimpleNamespace(page_size=16, n_kv_heads=2, head_dim=128)
    assert step_cached([kv, kv], n_tokens=0).shape == (0, 32)
