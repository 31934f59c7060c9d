"""The patched model's prompts: SDPA unless the prompt kernel was asked for."""
import pytest
import torch

import fake_nemotron as fake
from layer_quant_amd import int4_8b_attention as ia
from layer_quant_amd import nemotron_8b_decode_eval as de
from layer_quant_amd import prompts

pytestmark = pytest.mark.gpu


@pytest.fixture
def model(gpu):
    fake.reset_module()
    torch.manual_seed(0)
    model = fake.FakeNemotronHForCausalLM(fake.make_config(hybrid_override_pattern="*-*")).to(
        gpu, torch.bfloat16).eval()
    de.patch_attention_cache_in_blocks(model)
    yield model
    fake.reset_module()


@pytest.fixture
def calls(monkeypatch):
    """How many times the prompt kernel was called."""
    count = [0]
    kernel = prompts.prompt_attention

    def counted(*args, **kwargs):
        count[0] += 1
        return kernel(*args, **kwargs)

    monkeypatch.setattr(prompts, "prompt_attention", counted)
    return count


def logits_of(model, gpu):
    cache = fake.HybridMambaAttentionDynamicCache(model.config, 2, torch.bfloat16, gpu)
    ids = torch.arange(2 * 45, device=gpu).reshape(2, 45) % 64
    with torch.no_grad():
        return model(ids, cache_params=cache, cache_position=torch.arange(45, device=gpu)).float()


def test_a_model_patched_without_the_switch(gpu, model, calls):
    """Mixers that lack the switch's attribute (patched by hand, or before there was one) run SDPA."""
    ia.patch_nemotron_h_attention_int4_kv(model, group_size=64)
    want = logits_of(model, gpu)
    for layer in model.backbone.layers:
        if hasattr(layer.mixer, "_int4_kv_prompt_kernel"):
            del layer.mixer._int4_kv_prompt_kernel
    assert torch.equal(logits_of(model, gpu), want) and calls[0] == 0


def test_the_switch_of_a_patched_model(gpu, model, calls):
    """Patching again with prompt_kernel switches it on and off, and without leaves it."""
    layers = sum(layer.block_type == "attention" for layer in model.backbone.layers)
    ia.patch_nemotron_h_attention_int4_kv(model, group_size=64)
    plain = logits_of(model, gpu)
    assert calls[0] == 0
    for given, used in ((True, 1), (None, 1), (False, 0), (None, 0), (True, 1)):
        calls[0] = 0
        ia.patch_nemotron_h_attention_int4_kv(model, prompt_kernel=given)
        got = logits_of(model, gpu)
        assert calls[0] == used * layers, given
        assert torch.equal(got, plain) if not used else (got - plain).norm() <= 2e-2 * plain.norm()
