"""Attention whose scores are so large that one key has all the weight."""
import pytest
import torch

from layer_quant_amd import prompts

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("d", [64, 128, 96])
@pytest.mark.parametrize("scale", [2.0 ** -10, 1.0, 1000.0, 2.0 ** 35, 3e18])
@pytest.mark.parametrize("largest", ["last", "first", "middle"])
def test_one_key_has_all_the_weight(gpu, dtype, d, scale, largest):
    """Scores 2^24 j scale, exact before they are scaled, so that the next key is 2^14 and more behind: the
    value of the largest key so far, off by its weight's rounding and the output's (half a step each) and the
    sums' 2^-18."""
    rows = 127
    gen = torch.Generator(device=gpu).manual_seed(0)
    v = torch.randn(rows, 2, d, device=gpu, generator=gen).to(dtype)
    at = torch.arange(rows, device=gpu)
    rank = {"last": at, "first": rows - 1 - at, "middle": rows - 1 - (at - 70).abs() * 2 + (at < 70)}[largest]
    q = torch.zeros(rows, 4, d, device=gpu, dtype=dtype)
    k = torch.zeros(rows, 2, d, device=gpu, dtype=dtype)
    q[..., 0], k[..., 0] = 2.0 ** 15, (rank * 2.0 ** 9).to(dtype)[:, None]
    k[..., 1] = 1.0  # of weight 0 in q
    got = prompts.prompt_attention(q, k, v, torch.tensor([0, rows], device=gpu), scale=scale)
    best = torch.cummax(k[:, 0, 0].float(), 0).indices
    want = v[best].double().repeat_interleave(2, 1)
    assert ((got.double() - want).abs() <= (torch.finfo(dtype).eps + 2.0 ** -18) * want.abs()).all()
