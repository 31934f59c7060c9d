"""A prompt's keys and values into the INT4 cache, and a decode step over them."""
import pytest
import torch

from helpers import assert_close_rel
from layer_quant_amd import int4_8b_attention as ia
from layer_quant_amd import prompts
from oracle import int4_kv as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [32, 64])
def test_decode_attention_over_a_packed_prompt(gpu, group):
    """Two packed prompts of different lengths: each one's rows are packed as the oracle packs them, and the next
    token attends to them and to itself as in the oracle, and, where the cache's rounding allows, as the same
    token at the prompt's end. bf16 results: their rounding (2^-8), with the oracle's tests' tolerance."""
    gen = torch.Generator(device=gpu).manual_seed(0)
    lengths, hq, hkv, d = [65, 130], 8, 2, 128
    starts = torch.tensor([0, 66, 66 + 131], device=gpu)  # with the next tokens
    q, k, v = (torch.randn(197, h, d, device=gpu, generator=gen).bfloat16() for h in (hq, hkv, hkv))
    whole = prompts.prompt_attention(q, k, v, starts)
    for first, n in zip(starts.tolist(), lengths):
        rows = [t[first:first + n].transpose(0, 1)[None] for t in (k, v)]
        new = [t[first + n][None, :, None] for t in (q, k, v)]
        cache = ia._ensure_layer_cache(type("Cache", (), {})(), 0, 1, hkv, n + 1, d, group, gpu)
        ia._pack_kv_into_cache(cache, *rows, torch.arange(n, device=gpu), group)
        got = ia._pack_and_decode_attention(*new, cache, n + 1, hq // hkv, group)
        want = oracle.allocate_cache(1, hkv, n + 1, d, group)
        oracle.pack_kv_into_cache(want, *(t[first:first + n + 1].transpose(0, 1)[None].cpu() for t in (k, v)),
                                  torch.arange(n + 1), group)
        for name in ("k_packed", "v_packed", "k_scale", "v_scale"):
            assert torch.equal(getattr(cache, name)[:, :, :n + 1].cpu(), want[name]), name
        exact = oracle.decode_attention(new[0].cpu(), want["k_packed"], want["v_packed"], want["k_scale"],
                                        want["v_scale"], n + 1, hq // hkv, group)
        assert_close_rel(got.float().cpu(), exact, rtol=8e-3)
        assert cache.length == n + 1
        # an INT4 value is off by a 14th of its group's largest at most, about a tenth of its size on average, so
        # that scores and values move the result by some fifth of its length: the same direction as without it
        a, b = got.float().flatten(), whole[first + n].float().flatten()
        assert torch.dot(a, b) > 0.9 * a.norm() * b.norm()
