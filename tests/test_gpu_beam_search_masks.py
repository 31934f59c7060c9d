"""A beam search over left-padded prompts with an end token, call by call: the mask that reaches the
attention and what it attends to, the flags of finished beams and their scores, against the plain forms."""
import math

import numpy as np
import pytest
import torch

import fake_nemotron as fk
from layer_quant_amd import beam_decode as bd
from layer_quant_amd import int4_8b_attention as ia
from test_gpu_beam_search import build, prefill
from test_gpu_beam_select import reference as select_reference
from test_gpu_shared_attention import assert_near, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int64, torch.bool])
@pytest.mark.parametrize("P,N,L,pads,registered", [(2, 4, 20, (0, 6), False), (3, 5, 33, (32, 0, 9), True)])
def test_padded_prompts_and_end_tokens(gpu, P, N, L, pads, registered, dtype, monkeypatch):
    model = build(gpu, 1)
    try:
        eos, pad, steps = 7, 3, 10
        model.lm_head.weight.data[eos] = model.lm_head.weight.data[11]  # a token that is chosen now and then
        logits, cache = prefill(model, gpu, P, L, registered)
        logits[:, eos] = logits.max() - 1
        mask = torch.ones(P, L, dtype=torch.int64, device=gpu)
        for p, n in enumerate(pads):
            mask[p, :n] = 0
        select, attend = bd.beam_select, ia.shared_prefix_decode_attention
        flags, ended, calls = [None], [], [0]

        def checked_select(logits, scores, num=None, *, finished=None, pad_token=0, keep_slots=False):
            out = select(logits, scores, num, finished=finished, pad_token=pad_token, keep_slots=keep_slots)
            want = select_reference(logits, scores, scores.shape[1] if num is None else num,
                                    None if finished is None else finished.cpu(), pad_token, keep_slots)
            assert np.array_equal(out[1].cpu().numpy(), want[1])
            assert np.array_equal(out[2].cpu().numpy(), want[2])
            if flags[0] is None:
                assert finished is None
                flags[0] = out[2] == eos
                return out
            # the flags follow the beams, and a finished beam goes on with the pad token at its score
            assert pad_token == pad and torch.equal(finished, flags[0])
            of_finished = finished.gather(1, out[1])
            old = scores.gather(1, out[1])
            assert torch.equal(out[2][of_finished], torch.full_like(out[2][of_finished], pad))
            assert torch.equal(out[0][of_finished].view(torch.int32), old[of_finished].view(torch.int32))
            ended.append(int(of_finished.sum()))
            flags[0] = of_finished | (out[2] == eos)
            return out

        def checked_attention(q, own, seq_len, nrep, g, m, k, v):
            out = attend(q, own, seq_len, nrep, g, m, k, v)
            behind = torch.ones(P * N, seq_len - L, dtype=torch.int64, device=gpu)
            keep = torch.cat((mask.repeat_interleave(N, 0), behind), 1)
            assert m.dtype == dtype and torch.equal(m.long(), keep)
            bias = torch.where(keep != 0, 0.0, -math.inf).double()
            assert_near(out, reference(q, own, seq_len, nrep, g, bias), torch.bfloat16, 128, seq_len, True)
            calls[0] += 1
            return out

        monkeypatch.setattr(bd, "beam_select", checked_select)
        monkeypatch.setattr(ia, "shared_prefix_decode_attention", checked_attention)
        bd.beam_search(model, logits, cache, N, steps, start=L, eos_token_id=eos, pad_token=pad,
                       attention_mask=mask.to(dtype))
        assert calls[0] == 2 * (steps - 1)
        assert sum(ended), "no finished beam was selected again: nothing is tested"
    finally:
        fk.reset_module()
