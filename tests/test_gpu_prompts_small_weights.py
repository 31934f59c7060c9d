"""Attention with one key of almost all the weight and no value, and many of little weight that make the result."""
import math

import pytest
import torch

from layer_quant_amd import prompts

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("below", [9.0, 11.5, 13.25, 14.25])
def test_many_small_weights(gpu, dtype, d, below):
    """Key 0 has score 0 and value 0, the others -below (weights down to 2^-20.6) and values about 1. Half a
    step for the output, and for each weight; fp32 scores, exponentials and sums 2^-17."""
    rows = 3000
    gen = torch.Generator(device=gpu).manual_seed(0)
    v = 1 + 0.25 * torch.rand(rows, 1, d, device=gpu, generator=gen)
    v[0] = 0
    q, k = torch.zeros(rows, 2, d, device=gpu), torch.zeros(rows, 1, d, device=gpu)
    q[..., 0], k[1:, :, 0] = 1.0, -below
    q, k, v = (t.to(dtype) for t in (q, k, v))
    got = prompts.prompt_attention(q, k, v, torch.tensor([0, rows], device=gpu), scale=1.0)
    w = math.exp(-below)
    total = v[:, 0].double().cumsum(0) * w
    count = torch.arange(rows, device=gpu, dtype=torch.float64)[:, None]
    want = (total / (1 + w * count))[:, None].expand(-1, 2, -1)
    assert ((got.double() - want).abs() <= (torch.finfo(dtype).eps + 2.0 ** -17) * want
            + torch.finfo(dtype).tiny * torch.finfo(dtype).eps).all()
