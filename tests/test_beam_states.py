"""share_prompt and beam_search on the CPU: what they do to a hybrid cache and the MX registries, and what
they refuse, with the selection and the model replaced."""
from types import SimpleNamespace

import pytest
import torch

import fake_nemotron as fk
from layer_quant_amd import beam_decode as bd
from layer_quant_amd import int4_8b_attention as ia
from layer_quant_amd import mamba_state_8b_kernel as ms


def mx_cache(state):
    shape = state.shape
    return ms.MambaStateKernelCache(q_state=torch.ones(shape, dtype=torch.int8),
                                    shared_exp=torch.ones(*shape[:-1], shape[-1] // 16, dtype=torch.uint8),
                                    micro_exp=torch.ones(*shape[:-1], shape[-1] // 2, dtype=torch.uint8),
                                    format_bits=8)


@pytest.fixture
def model():
    fk.reset_module()
    torch.manual_seed(0)
    yield fk.FakeNemotronHForCausalLM(fk.make_config(num_attention_heads=2, num_key_value_heads=1))
    fk.reset_module()


def hybrid(model, batch):
    return fk.HybridMambaAttentionDynamicCache(model.config, batch, torch.float32)


def register(model, *states):
    model._mamba_decode_state_kernel_caches = {id(s): mx_cache(s) for s in states}
    fk._mamba_decode_state_kernel_caches = dict(model._mamba_decode_state_kernel_caches)


def test_share_prompt_keeps_other_caches_registered(model):
    """A registered cache goes on with its MX states where another cache's prompt is shared."""
    a, b = hybrid(model, 2), hybrid(model, 3)
    register(model, a.ssm_states[0], a.ssm_states[2])
    held = [model._mamba_decode_state_kernel_caches[id(a.ssm_states[i])] for i in (0, 2)]
    bd.share_prompt(model, b, 4)
    for registry in (model._mamba_decode_state_kernel_caches, fk._mamba_decode_state_kernel_caches):
        assert [registry.get(id(a.ssm_states[i])) for i in (0, 2)] == held
        assert len(registry) == 2
    assert b.ssm_states[0].shape[0] == 12


def test_share_prompt_renews_its_own_entries(model):
    a, b = hybrid(model, 2), hybrid(model, 3)
    register(model, a.ssm_states[0], b.ssm_states[0], b.ssm_states[2])
    of_a = model._mamba_decode_state_kernel_caches[id(a.ssm_states[0])]
    for i in (0, 2):
        model._mamba_decode_state_kernel_caches[id(b.ssm_states[i])].q_state *= torch.arange(3)[:, None, None, None]
    old = [b.ssm_states[i] for i in (0, 2)]
    bd.share_prompt(model, b, 4)
    for registry in (model._mamba_decode_state_kernel_caches, fk._mamba_decode_state_kernel_caches):
        assert registry[id(a.ssm_states[0])] is of_a
        assert not any(id(s) in registry for s in old)
        assert len(registry) == 3
        for i in (0, 2):
            mx = registry[id(b.ssm_states[i])]
            assert torch.equal(mx.q_state[:, 0, 0, 0], torch.arange(3, dtype=torch.int8).repeat_interleave(4))
            assert mx.shared_exp.shape[0] == mx.micro_exp.shape[0] == 12


def test_share_prompt_drops_entries_of_freed_states(model):
    """An entry whose state is gone must not become that of a new tensor with its id."""
    b = hybrid(model, 2)
    stale = {n: mx_cache(torch.zeros(1, 1, 1, 16)) for n in range(8)}
    model._mamba_decode_state_kernel_caches = dict(stale)
    fk._mamba_decode_state_kernel_caches = dict(stale)
    real = torch.Tensor.repeat_interleave

    def repeat(self, *args, **kw):
        out = real(self, *args, **kw)
        for registry in (model._mamba_decode_state_kernel_caches, fk._mamba_decode_state_kernel_caches):
            registry[id(out)] = registry.pop(min(registry), None)  # as if the id had been a freed state's
        return out

    with pytest.MonkeyPatch.context() as patch:
        patch.setattr(torch.Tensor, "repeat_interleave", repeat)
        bd.share_prompt(model, b, 2)
    for registry in (model._mamba_decode_state_kernel_caches, fk._mamba_decode_state_kernel_caches):
        assert not any(id(s) in registry for s in b.ssm_states)


def int4_layer(batch, length):
    layer = ia._allocate_layer_cache(batch, 1, 16, 128, 2, torch.device("cpu"))
    layer.length = length
    return layer


@pytest.mark.parametrize("start", [0, 8, 10, 11])
def test_beam_search_refuses_a_start_off_its_caches(model, start):
    """The first new token stands right behind the prompts' rows: rows in between would be attended
    without having been written."""
    cache = hybrid(model, 2)
    ia._cache_dict(cache).update({1: int4_layer(2, 9), 4: int4_layer(2, 9)})
    before = list(cache.ssm_states)
    with pytest.raises(ValueError, match="start"):
        bd.beam_search(model, torch.zeros(2, 64), cache, 4, 3, start=start)
    assert all(a is b for a, b in zip(cache.ssm_states, before))
    assert all(layer.prefix is None for layer in ia._cache_dict(cache).values())


def test_beam_search_refuses_caches_of_different_lengths(model):
    cache = hybrid(model, 2)
    ia._cache_dict(cache).update({1: int4_layer(2, 9), 4: int4_layer(2, 8)})
    for start in (8, 9):
        with pytest.raises(ValueError, match="start"):
            bd.beam_search(model, torch.zeros(2, 64), cache, 4, 3, start=start)


@pytest.fixture
def on_cpu(monkeypatch):
    """beam_search with the selection in torch, no reordering, and a model that makes the same logits."""
    seen = SimpleNamespace(scores=[], grad=[])

    def select(logits, scores, num=None, *, finished=None, pad_token=0, keep_slots=False):
        seen.scores.append(scores)
        P, N = scores.shape
        total = scores[..., None] + logits.reshape(P, N, -1).float().log_softmax(-1)
        best = total.reshape(P, -1).topk(N if num is None else num)
        V = logits.shape[-1]
        return best.values, best.indices // V, best.indices % V

    def model(tokens, **kw):
        seen.grad.append(torch.is_grad_enabled())
        return SimpleNamespace(logits=torch.arange(64.0).expand(tokens.shape[0], 1, 64))

    monkeypatch.setattr(bd, "beam_select", select)
    monkeypatch.setattr(bd, "reorder_states", lambda *a: None)
    seen.run = lambda: bd.beam_search(model, torch.randn(2, 64), SimpleNamespace(), 4, 3, start=5)
    return seen


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_running_scores_are_fp32_whatever_the_default_dtype(on_cpu, dtype):
    default = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        tokens, scores = on_cpu.run()
    finally:
        torch.set_default_dtype(default)
    assert tokens.shape == (2, 4, 3) and scores.dtype == torch.float32
    assert all(s.dtype == torch.float32 for s in on_cpu.scores)


def test_a_search_records_no_gradients(on_cpu):
    """States are written in place, step after step: with gradients on, a graph over all steps stayed alive."""
    assert torch.is_grad_enabled()
    on_cpu.run()
    assert on_cpu.grad == [False, False] and torch.is_grad_enabled()
