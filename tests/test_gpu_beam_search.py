"""The beam-decoding operators together, on the patched stand-in model: every call that beam_search
makes is checked on its own inputs -- the selection against a sort in 64 bits, the reordering of every
state byte for byte, the attention over the shared prompt against 64 bits with the tolerance derived in
test_gpu_shared_attention.py -- and the result against the calls' own record."""
import numpy as np
import pytest
import torch

import fake_nemotron as fk
from layer_quant_amd import beam_decode as bd
from layer_quant_amd import int4_8b_attention as ia
from layer_quant_amd import mamba_state_8b_kernel as ms
from layer_quant_amd import nemotron_8b_decode_eval as de
from test_gpu_beam_select import reference as select_reference
from test_gpu_reorder_beams import expected, same_bytes
from test_gpu_shared_attention import assert_near, pack_token, reference

pytestmark = pytest.mark.gpu
GROUP = 64


def build(gpu, seed=0):
    fk.reset_module()
    torch.manual_seed(seed)
    cfg = fk.make_config(hybrid_override_pattern="M*M-M*", num_attention_heads=8, num_key_value_heads=2,
                         head_dim=128, mamba_num_heads=16, mamba_head_dim=64, ssm_state_size=128,
                         n_groups=2, vocab_size=211)
    model = fk.FakeNemotronHForCausalLM(cfg).to(torch.bfloat16).to(gpu).eval()
    model.lm_head.weight.data *= 6
    de.patch_attention_cache_in_blocks(model)
    ia.patch_nemotron_h_attention_int4_kv(model, group_size=GROUP)
    ms.patch_nemotron_h_mamba_decode_state_kernel(model, stochastic=False)
    return model


def prefill(model, gpu, P, L, registered):
    ids = torch.randint(0, 211, (P, L), device=gpu, generator=torch.Generator(device=gpu).manual_seed(L))
    cache = de.make_hybrid_cache(model, P)
    logits = model(ids, cache_params=cache, cache_position=torch.arange(L, device=gpu), use_cache=True)
    if registered:
        ms.register_mamba_state_kernel_caches(model, cache, {0: "mx8", 2: "mx4"})
    return logits[:, -1], cache


@pytest.mark.parametrize("registered", [False, True])
@pytest.mark.parametrize("P,N,L,steps", [(1, 4, 40, 24), (3, 5, 33, 12)])
def test_every_call_of_a_search(gpu, registered, P, N, L, steps, monkeypatch):
    model = build(gpu)
    try:
        logits, cache = prefill(model, gpu, P, L, registered)
        scores_seen, calls = [], dict(attention=0, reorder=0)
        select, reorder, attend = bd.beam_select, bd.reorder_beams, ia.shared_prefix_decode_attention

        def checked_select(logits, scores, num=None, **kw):
            out = select(logits, scores, num, **kw)
            num = scores.shape[1] if num is None else num
            want = select_reference(logits, scores, num, slots=kw.get("keep_slots", False))
            assert np.array_equal(out[1].cpu().numpy(), want[1])
            assert np.array_equal(out[2].cpu().numpy(), want[2])
            scores_seen.append(out)
            return out

        def checked_reorder(tensors, beams, rows=None):
            want = [expected(t, beams, r) for t, r in zip(tensors, rows)]
            # two attention layers, three Mamba2 layers of which two are registered
            assert len(tensors) == 2 * 4 + (2 * 3 + 1 if registered else 3)
            reorder(tensors, beams, rows)
            assert all(same_bytes(t, w) for t, w in zip(tensors, want))
            calls["reorder"] += 1

        def checked_attention(q, own, seq_len, nrep, g, mask, k, v):
            assert q.shape[0] == P * N and own.prefix.k_packed.shape[0] == P
            out = attend(q, own, seq_len, nrep, g, mask, k, v)
            lo = seq_len - own.prefix.length
            row = ia._allocate_layer_cache(P * N, 2, 16, 128, 128 // g, gpu)
            pack_token(k, row.k_packed, row.k_scale, 0, g)
            assert torch.equal(own.k_packed[:, :, lo - 1], row.k_packed[:, :, 0])
            assert torch.equal(own.k_scale[:, :, lo - 1], row.k_scale[:, :, 0])
            assert_near(out, reference(q, own, seq_len, nrep, g), torch.bfloat16, 128, seq_len, True)
            calls["attention"] += 1
            return out

        monkeypatch.setattr(bd, "beam_select", checked_select)
        monkeypatch.setattr(bd, "reorder_beams", checked_reorder)
        monkeypatch.setattr(ia, "shared_prefix_decode_attention", checked_attention)
        tokens, scores = bd.beam_search(model, logits, cache, N, steps, start=L)
        assert calls == dict(attention=2 * (steps - 1), reorder=steps - 1)
        for layer in ia._cache_dict(cache).values():
            assert layer.length == steps - 1 and layer.prefix.length == L
        # the sequences, followed back through the calls' beams
        order = torch.sort(scores_seen[-1][0], dim=1, descending=True, stable=True)
        assert torch.equal(scores, order.values)
        row = order.indices
        for step in range(steps - 1, -1, -1):
            assert torch.equal(tokens[:, :, step], scores_seen[step][2].gather(1, row))
            row = scores_seen[step][1].gather(1, row)
    finally:
        fk.reset_module()


def test_finished_beams_and_padding(gpu):
    """A beam that chose the end token goes on with the pad token at its score; left-padded prompts."""
    model = build(gpu, 1)
    try:
        P, N, L, eos, pad = 2, 4, 20, 7, 3
        model.lm_head.weight.data[eos] = model.lm_head.weight.data[11]  # a token that is chosen now and then
        logits, cache = prefill(model, gpu, P, L, False)
        mask = torch.ones(P, L, dtype=torch.int64, device=gpu)
        mask[1, :6] = 0
        logits[:, eos] = logits.max() - 1
        tokens, scores = bd.beam_search(model, logits, cache, N, 10, start=L, eos_token_id=eos,
                                        pad_token=pad, attention_mask=mask)
        ended = tokens == eos
        assert ended.any(), "no beam has ended: nothing is tested"
        behind = ended.cumsum(-1) - ended.long() > 0
        assert (tokens[behind] == pad).all()
        assert torch.isfinite(scores).all()
    finally:
        fk.reset_module()


def test_forward_refuses_what_a_shared_prefix_cannot_take(gpu):
    model = build(gpu)
    try:
        logits, cache = prefill(model, gpu, 2, 16, False)
        with pytest.raises(ValueError, match="num_beams"):
            bd.share_prompt(model, cache, 0)
        bd.share_prompt(model, cache, 3)
        with pytest.raises(ValueError, match="already"):
            bd.share_prompt(model, cache, 3)
        two = torch.zeros(6, 2, dtype=torch.int64, device=gpu)
        with pytest.raises(ValueError, match="one later token"):
            model(two, cache_params=cache, cache_position=torch.tensor([16, 17], device=gpu))
        with pytest.raises(ValueError, match="one later token"):
            model(two[:, :1], cache_params=cache, cache_position=torch.tensor([3], device=gpu))
        model(two[:, :1], cache_params=cache, cache_position=torch.tensor([16], device=gpu))
    finally:
        fk.reset_module()
