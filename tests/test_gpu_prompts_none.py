"""Packed rows of no prompt: zeros, whatever their number and the kernel that writes them."""
import pytest
import torch

from layer_quant_amd import prompts

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("rows", [1, 16, 63, 64, 65, 3000])
@pytest.mark.parametrize("starts", [[0], [5], [1 << 20], [2, 2]], ids=str)
def test_rows_of_no_prompt(gpu, dtype, rows, starts):
    """One start (no prompt), or one prompt without rows, which hands its state on."""
    gen = torch.Generator(device=gpu).manual_seed(rows)
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen)  # noqa: E731
    x, dt, A = randn(rows, 8, 64).to(dtype), randn(rows, 8), -torch.rand(8, device=gpu, generator=gen)
    B, C = randn(rows, 2, 128).to(dtype), randn(rows, 2, 128).to(dtype)
    at = torch.tensor(starts, device=gpu)
    initial = randn(len(starts) - 1, 8, 64, 128)
    y, states = prompts.prompt_scan(x, dt, A, B, C, at, dt_softplus=True, initial_states=initial)
    assert y.shape == x.shape and not y.any()
    assert torch.equal(states, initial)
    q, k = randn(rows, 4, 64).to(dtype), randn(rows, 2, 64).to(dtype)
    assert not prompts.prompt_attention(q, k, k, at).any()
