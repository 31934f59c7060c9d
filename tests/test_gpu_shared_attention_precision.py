"""What the shared-prefix attention's matrix-core kernel keeps of a key's share, whatever the output's type
and the other keys' value scales and weights.

Bound of an output value against 64 bits, first order in each error: half a step of the output's type at
the exact value; a score is a sum of head_dim exact products with fp32 additions and scalings, off by
delta_j = (head_dim + 16) * 2^-24 * sum_d |q_d k_jd| log2(e)/sqrt(D), and its weight by ln(2) delta_j and
the exponential's 2^-22, which moves the output by at most w_j (|v_j| + |out|) of that; weight x value
scale is rounded to fp32 (2^-24) and held in bf16 terms that each round what the terms before leave (a
relative 2^-8): two of them, 2^-16, for bf16 outputs, three, 2^-24, for the others; fp32 sums over the
keys, the waves and the splits: (keys + 32) * 2^-24 of sum_j w_j |v_j|, and the same of the weights' sum."""
import math

import pytest
import torch

from helpers import require_env
from layer_quant_amd import _abi
from oracle import int4_kv as oik
from test_gpu_shared_attention import BF16, FP16, FP32, cache_of

pytestmark = pytest.mark.gpu
LOG2E = 1.4426950408889634


def attend(q, own, lp, lo, nrep, g, dtype, mask=None):
    pre = own.prefix
    out = torch.empty(q.shape[0], q.shape[1], q.shape[-1], device=q.device, dtype=dtype)
    with require_env("LQ_ATTN_REQUIRE_FAST", True):
        _abi.int4_shared_decode_attention(
            q, None, None, (pre.k_packed, pre.v_packed, pre.k_scale, pre.v_scale),
            (own.k_packed, own.v_packed, own.k_scale, own.v_scale), mask, out, lp, lp + lo, nrep, g)
    return out


def half_step(x, dtype):
    """Half the distance between the values of `dtype` around x (64 bits, not 0)."""
    bits = {BF16: 8, FP16: 11, FP32: 24}[dtype]
    e = torch.floor(torch.log2(x.abs().clamp_min(1e-300)))
    if dtype == FP16:
        e = e.clamp_min(-14)
    return torch.exp2(e - bits)


def worst(out, q, own, lp, lo, nrep, g, dtype):
    """The largest |out - exact| / bound."""
    pre, d = own.prefix, q.shape[-1]
    N = q.shape[0] // pre.k_packed.shape[0]
    top = 0.0
    for b in range(q.shape[0]):
        k, v = (torch.cat([oik.dequantize(getattr(c, n + "_packed")[i:i + 1, :, :m].cpu(),
                                          getattr(c, n + "_scale")[i:i + 1, :, :m].cpu(), g)[0].double()
                           for c, i, m in ((pre, b // N, lp), (own, b, lo))], 1).to(q.device) for n in "kv")
        k, v = k.repeat_interleave(nrep, 0), v.repeat_interleave(nrep, 0)
        x = q[b, :, 0, :, None].double()
        s = (k @ x)[..., 0] * (LOG2E / math.sqrt(d))
        delta = (k.abs() @ x.abs())[..., 0] * (LOG2E / math.sqrt(d)) * (d + 16) * 2.0 ** -24
        w = torch.exp2(s - s.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        want = (w[:, None] @ v)[:, 0]
        eps = w * (math.log(2) * delta + 2.0 ** -22)
        mag = (w[:, None] @ v.abs())[:, 0]
        bound = half_step(want, dtype) + (eps[:, None] @ v.abs())[:, 0] + eps.sum(-1, keepdim=True) * want.abs()
        bound += ((2.0 ** -16 if dtype == BF16 else 2.0 ** -23) + 2.0 ** -24) * mag
        bound += (lp + lo + 32) * 2.0 ** -24 * (mag + want.abs()) + 1e-300
        top = max(top, ((out[b].double() - want).abs() / bound).max().item())
    print(f"[close] {dtype} lp{lp} lo{lo} g{g}: max err/bound {top:.3g}")
    return top


@pytest.mark.parametrize("g", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("N,lp,lo", [(8, 3, 1), (3, 7, 0), (64, 40, 9)])
def test_every_output_is_its_rounding(gpu, dtype, g, N, lp, lo):
    """Few keys with weights near each other: an output is off by its own rounding and little else."""
    own = cache_of(gpu, N, 8, lo, max(lo, 1), 128, g, 2)
    own.prefix = cache_of(gpu, 1, 8, lp, lp, 128, g, 1)
    q = (0.1 * torch.randn(N, 32, 1, 128, device=gpu)).to(BF16)
    assert worst(attend(q, own, lp, lo, 4, g, dtype), q, own, lp, lo, 4, g, dtype) <= 1.0


@pytest.mark.parametrize("g", [32, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("N", [2, 8])
@pytest.mark.parametrize("span", [24, 60])
def test_a_large_scale_of_little_weight(gpu, dtype, g, N, span):
    """One key with value scales 2^span times the others' and next to no weight: the others' shares keep
    their precision."""
    lp, lo, nrep = 70, 5, 4
    own = cache_of(gpu, N, 2, lo, lo, 128, g, 2)
    own.prefix = pre = cache_of(gpu, 1, 2, lp, lp, 128, g, 1)
    pre.k_packed[:, :, 10] = 0x99  # level -7 in every dim, under a positive query
    pre.k_scale[:, :, 10] = 0.75 if span == 24 else 1.25
    pre.v_scale[:, :, 10] *= 2.0 ** span
    q = (0.7 + 0.3 * torch.rand(N, 2 * nrep, 1, 128, device=gpu)).to(BF16)
    out = attend(q, own, lp, lo, nrep, g, dtype)
    assert worst(out, q, own, lp, lo, nrep, g, dtype) <= 1.0


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_scales_of_every_size(gpu, dtype):
    """Value scales spread over 2^48 from key to key: each share has its own precision."""
    N, lp, lo, nrep, g = 4, 90, 20, 4, 32
    own = cache_of(gpu, N, 2, lo, lo, 128, g, 2)
    own.prefix = pre = cache_of(gpu, 1, 2, lp, lp, 128, g, 1)
    gen = torch.Generator(device=gpu).manual_seed(3)
    for c, n in ((pre, lp), (own, lo)):
        e = torch.randint(-38, 10, c.v_scale.shape[:3], device=gpu, generator=gen)
        c.v_scale *= torch.exp2(e.float())[..., None]
    q = (0.3 * torch.randn(N, 2 * nrep, 1, 128, device=gpu, generator=gen)).to(BF16)
    assert worst(attend(q, own, lp, lo, nrep, g, dtype), q, own, lp, lo, nrep, g, dtype) <= 1.0
