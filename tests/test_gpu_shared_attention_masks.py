"""Masked calls of the shared-prefix attention in every instance that the matrix-core kernel has: query and
output types, groups, one and two column tiles of query rows, own units of one, two and four waves."""
import math

import pytest
import torch

from layer_quant_amd import int4_8b_attention as ia
from test_gpu_shared_attention import BF16, FP16, FP32, assert_near, cache_of, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("g", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("N", [3, 6])  # 12 and 24 query rows per KV head
@pytest.mark.parametrize("lp,lo", [(100, 30), (1500, 3)])
def test_masks(gpu, dtype, g, N, lp, lo):
    """Padded prompts, rows without a key, short masks, biases of every kind, -inf and the lowest."""
    P, hkv, nrep = 2, 2, 4
    B, S = P * N, lp + lo
    keep = torch.ones(B, S, dtype=torch.int64, device=gpu)
    keep[:N, : lp // 2] = 0
    keep[N] = 0
    keep[N + 1, :-1] = 0
    keep[N + 2, -lo:] = 0
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 1, keep)
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 1, (keep != 0)[:, None, None])
    torch.manual_seed(lp + N)
    bias = torch.randn(B, 1, 1, S, device=gpu)
    bias[:, :, :, ::3] = -torch.inf
    bias[0] = torch.finfo(torch.float32).min
    bias[1, :, :, : S // 2] = torch.finfo(torch.float32).min
    bias[2, :, :, :lp] = -torch.inf
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 2, bias)
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 2, bias[..., :lp], token=False)


@pytest.mark.parametrize("g", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("N", [2, 6])
@pytest.mark.parametrize("additive", [False, True])
def test_masked_rows_may_hold_anything(gpu, dtype, g, N, additive):
    """Infinities and NaN in cache rows that no row attends to, in whole tiles and inside them."""
    P, hkv, nrep, lp, lo = 2, 1, 4, 200, 40
    pre = cache_of(gpu, P, hkv, lp, lp + 8, 128, g, 1)
    own = cache_of(gpu, P * N, hkv, lo, lo + 8, 128, g, 2)
    own.prefix = pre
    keep = torch.ones(P * N, lp + lo, dtype=torch.int64, device=gpu)
    for c, at in ((pre, 0), (own, lp)):
        for j in (0, 5, 17, 31, 33):
            keep[:, at + j] = 0
            c.k_scale[:, :, j], c.v_scale[:, :, j] = torch.nan, torch.inf
    pre.v_scale[:, :, 64:100] = torch.nan
    keep[:, 64:100] = 0
    q = torch.randn(P * N, hkv * nrep, 1, 128, device=gpu).to(dtype)
    bias = torch.where(keep != 0, 0.0, -math.inf)
    mask = bias[:, None, None] if additive else keep
    out = ia.shared_prefix_decode_attention(q, own, lp + lo, nrep, g, mask)
    for c in (pre, own):
        c.k_scale.nan_to_num_(0, 0, 0)
        c.v_scale.nan_to_num_(0, 0, 0)
    ref = reference(q, own, lp + lo, nrep, g, bias.double())
    assert_near(out, ref, dtype, 128, lp + lo, dtype != FP32)


@pytest.mark.parametrize("g", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lo", [40, 100, 250, 300])
@pytest.mark.parametrize("mask", ["none", "keep", "bias"])
def test_many_own_rows(gpu, lo, dtype, g, mask):
    """Own units behind a prefix that fills the GPU: one, two or four waves each, odd numbers of them."""
    P, N, hkv, nrep, lp = 5, 13, 8, 4, 2500
    gen = torch.Generator(device=gpu).manual_seed(lo)
    keep = (torch.rand(P * N, lp + lo, device=gpu, generator=gen) < 0.8).long()
    m = {"none": None, "keep": keep}.get(mask)
    if mask == "bias":
        m = torch.where(keep != 0, torch.randn(keep.shape, device=gpu, generator=gen), -torch.inf)[:, None, None]
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, lo, m)
