"""Outputs in the same tensor as the inputs, without overlapping them: fused rows, states in halves."""
import pytest
import torch

from layer_quant_amd import _abi, prompts

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_attention_into_fused_rows(gpu, dtype):
    gen = torch.Generator(device=gpu).manual_seed(0)
    fused = torch.randn(300, 12, 64, device=gpu, generator=gen).to(dtype)
    starts = torch.tensor([0, 190, 300], device=gpu)
    q, k, v, more = fused[:, :4], fused[:, 4:6], fused[:, 6:8], fused[:, 8:]
    want = prompts.prompt_attention(*(t.clone() for t in (q, k, v)), starts)
    before = fused.clone()
    assert torch.equal(prompts.prompt_attention(q, k, v, starts, out=more), want)
    assert torch.equal(fused[:, :8], before[:, :8])
    for wrong in (fused[:, 5:9], fused[:, 1:5], fused[:1, 8:].expand(300, 4, 64)):
        with pytest.raises(_abi.LQError, match="overlap"):
            prompts.prompt_attention(q, k, v, starts, out=wrong)
    assert torch.equal(prompts.prompt_attention(q, k, v, starts, out=q), want)
    assert torch.equal(fused[:, 4:8], before[:, 4:8])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_states_in_halves_of_a_tensor(gpu, dtype):
    gen = torch.Generator(device=gpu).manual_seed(1)
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen)  # noqa: E731
    x, dt, A = randn(1500, 4, 64).to(dtype), randn(1500, 4), -torch.rand(4, device=gpu, generator=gen)
    B, C = randn(1500, 1, 128).to(dtype), randn(1500, 1, 128).to(dtype)
    starts, both = torch.tensor([0, 1200, 1500], device=gpu), randn(2, 2, 4, 64, 128)
    for first, last in ((both[:, 0], both[:, 1]), (both[0], both[1])):
        y, st = prompts.prompt_scan(x, dt, A, B, C, starts, dt_softplus=True, initial_states=first.clone())
        again, _ = prompts.prompt_scan(x, dt, A, B, C, starts, dt_softplus=True, initial_states=first, states=last)
        assert torch.equal(again, y) and torch.equal(last, st)
        with pytest.raises(_abi.LQError, match="overlap"):
            prompts.prompt_scan(x, dt, A, B, C, starts, dt_softplus=True, initial_states=first,
                                states=first[:1].expand(2, 4, 64, 128))
