"""Decode steps that would leave unwritten rows between a shared prefix and the step's token."""
import pytest
import torch

import fake_nemotron as fk
from layer_quant_amd import beam_decode as bd
from layer_quant_amd import int4_8b_attention as ia
from test_gpu_beam_search import build, prefill

pytestmark = pytest.mark.gpu


def test_forward_refuses_a_gap_behind_the_prefix(gpu):
    model = build(gpu)
    try:
        _, cache = prefill(model, gpu, 2, 16, False)
        bd.share_prompt(model, cache, 3)
        token = torch.zeros(6, 1, dtype=torch.int64, device=gpu)

        def step(at):
            return model(token, cache_params=cache, cache_position=torch.tensor([at], device=gpu))

        for at in (17, 18, 40):
            with pytest.raises(ValueError, match="unwritten"):
                step(at)
        step(16)
        step(17)
        with pytest.raises(ValueError, match="unwritten"):
            step(19)
        step(17)  # the last row again
        assert [layer.length for layer in ia._cache_dict(cache).values()] == [2, 2]
    finally:
        fk.reset_module()
