"""Residual addition + RMSNorm + Q8_K in one kernel: bit-identical to the
addition followed by the stand-alone kernel, and near the formula in 64 bits."""
import pytest
import torch

from smeai_b200 import q2k as Q

pytestmark = pytest.mark.gpu


def case(dev, n, k, stride, off, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x, r = (torch.randn((n, stride + off), generator=g, device=dev)[:, off:off + k] for _ in range(2))
    return x, r * 3, 1 + 0.2 * torch.randn(k, generator=g, device=dev)


@pytest.mark.parametrize("weight", [True, False])
@pytest.mark.parametrize("n,k,extra,off", [(1, 256, 0, 0), (1, 4096, 0, 0), (3, 512, 4, 0), (5, 4096, 1, 1), (300, 2048, 0, 0), (2, 8192, 256, 0),
                                           (7, 11008, 0, 0), (1, 65536, 0, 0), (1000, 768, 3, 2)])
def test_equals_the_separate_kernels(cuda, n, k, extra, off, weight):
    x, r, w = case(cuda, n, k, k + extra, off)
    w = w if weight else None
    h, blocks = Q.add_rms_quantize_q8k(x, r, 1e-5, norm_w=w)
    want = (x + r).contiguous()
    assert torch.equal(h, want) and torch.equal(blocks, Q.rms_quantize_q8k(want, 1e-5, norm_w=w))


@pytest.mark.parametrize("k", [1024, 11008])
def test_sum_in_place(cuda, k):
    x, r, w = case(cuda, 9, k, k + 8, 0)
    h, blocks = Q.add_rms_quantize_q8k(x, r, 1e-5, norm_w=w)
    x2 = x.clone()
    h2, b2 = Q.add_rms_quantize_q8k(x2, r, 1e-5, norm_w=w, sum_out=x2)
    assert torch.equal(x2, h) and torch.equal(b2, blocks)
    r2 = torch.empty((9, k + 8), device=cuda)[:, :k].copy_(r)
    Q.add_rms_quantize_q8k(x, r2, 1e-5, norm_w=w, sum_out=r2, out=b2)
    assert torch.equal(r2, h) and torch.equal(b2, blocks)


def test_against_64_bits(cuda):
    n, k = 64, 4096
    x, r, w = case(cuda, n, k, k, 0, seed=3)
    x[0], r[0] = 0.0, 0.0                                   # a row of zeros
    x[1, 256:512], r[1, 256:512] = 2.0, -2.0                # a block of zeros
    h, blocks = Q.add_rms_quantize_q8k(x, r, 1e-5, norm_w=w)
    b = blocks.view(n, k // 256, 292)
    d, q = b[:, :, :4].view(torch.float32).double(), b[:, :, 4:260].view(torch.int8).double()
    sums = b[:, :, 260:].view(torch.int16)
    ref = h.double()
    y = (ref / torch.sqrt((ref * ref).mean(1, keepdim=True) + 1e-5) * w.double()).view(n, k // 256, 256)
    # half a step of the block, and the roundings of the norm, the scale and the product (2^-21 covers their sum)
    step = y.abs().amax(2, keepdim=True) / 127
    assert ((q * d - y).abs() <= step * (0.5 + 127 * 2.0 ** -21)).all()
    assert torch.equal(q.view(n, k // 256, 16, 16).sum(3).to(torch.int16), sums)
    assert (blocks[0] == 0).all() and (b[1, 1] == 0).all()


def test_captured_and_replayed(cuda):
    x, r, w = case(cuda, 4, 2048, 2048, 0)
    out, h = torch.empty((4, 8 * 292), dtype=torch.uint8, device=cuda), torch.empty((4, 2048), device=cuda)
    Q.add_rms_quantize_q8k(x, r, 1e-5, norm_w=w, out=out, sum_out=h)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        Q.add_rms_quantize_q8k(x, r, 1e-5, norm_w=w, out=out, sum_out=h)
    x.mul_(-2)
    g.replay()
    want, blocks = Q.add_rms_quantize_q8k(x, r, 1e-5, norm_w=w)
    assert torch.equal(h, want) and torch.equal(out, blocks)
