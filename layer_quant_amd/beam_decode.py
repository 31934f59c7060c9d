"""Beam decoding over the quantized decode states (no reference counterpart: its driver scores given
text, one row per sequence).

Several beams of a prompt share the prompt's INT4 cache, and after every step the states of each row
follow the beam that was selected for it:

    beam_select     the best continuations of each prompt's beams         -> lq_beam_select
    reorder_beams   state tensors follow the selected beams, in place     -> lq_reorder_beams
    int4_8b_attention.shared_prefix_decode_attention (called by the patched attention forward)
                                                             -> lq_int4_shared_decode_attention

share_prompt and reorder_states apply them to a patched model's hybrid cache, and beam_search runs the
whole loop. Rows are prompt-major: row p*N + n is beam n of prompt p.
"""
from __future__ import annotations

from dataclasses import replace

import torch

from . import _abi
from . import int4_8b_attention as ia


def beam_select(logits: torch.Tensor, scores: torch.Tensor, num: int | None = None, *,
                finished: torch.Tensor | None = None, pad_token: int = 0,
                keep_slots: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The `num` (default: N) best continuations of each prompt's N beams: (scores [P, num] fp32,
    beams [P, num] int64, tokens [P, num] int64).

    logits [P*N, V] or [P, N, V] in fp32, fp16 or bf16, any strides; scores [P, N] fp32, the beams'
    running scores. The total of beam n and token t is scores[n] + log_softmax(logits[n])[t], its
    log-sum-exp off by less than 2^-18 (fp32 sums); totals are compared in 64 bits, equal ones by the
    lower n * V + t. `finished` (bool [P, N]): such a beam has one continuation, pad_token at its own
    score. Continuations of a beam whose score or log-sum-exp is not finite count as -inf.

    In descending order, or with keep_slots (num == N) by place: the best continuation selected of a
    beam stands at that beam's place, the others at the free places in order, so that reorder_beams
    moves no state of a beam that goes on. At most 64 beams and 64 continuations.
    """
    if scores.dim() != 2:
        raise ValueError(f"Expected scores [prompts, beams], got {tuple(scores.shape)}")
    prompts, beams = scores.shape
    if logits.dim() == 2:
        if logits.shape[0] != prompts * beams:
            raise ValueError(f"Expected logits of {prompts} x {beams} rows, got {logits.shape[0]}")
    elif logits.dim() != 3 or logits.shape[:2] != scores.shape:
        raise ValueError(f"Expected logits [{prompts}, {beams}, vocab], got {tuple(logits.shape)}")
    if finished is not None:
        if finished.dtype != torch.bool or finished.shape != scores.shape:
            raise ValueError(f"Expected finished bool {tuple(scores.shape)}, got {finished.dtype} "
                             f"{tuple(finished.shape)}")
        finished = finished.view(torch.uint8)
    num = beams if num is None else num
    if num < 0:
        raise ValueError(f"num must not be negative, got {num}")
    shape = (prompts, num)
    out_scores = torch.empty(shape, device=scores.device, dtype=torch.float32)
    out_beams = torch.empty(shape, device=scores.device, dtype=torch.int64)
    out_tokens = torch.empty(shape, device=scores.device, dtype=torch.int64)
    _abi.beam_select(logits, scores, finished, out_scores, out_beams, out_tokens, pad_token,
                     keep_slots)
    return out_scores, out_beams, out_tokens


def reorder_beams(tensors, beams: torch.Tensor, rows=None) -> None:
    """In place, for every tensor [P*N, ...]: row p*N + n takes the contents that row
    p*N + beams[p, n] had before the call. Entries outside [0, N) leave their row as it is.

    beams int64 [P, N] (N <= 64); the tensors of any dtype the ABI knows and any strides, up to 512,
    none overlapping itself, another or the beams. rows[i]: how many entries of dim 2 of tensor i are
    moved (the live rows of an INT4 cache), None for all. One launch for a model's states, in any
    permutation.
    """
    if rows is not None and len(rows) != len(tensors):
        raise ValueError(f"{len(rows)} row counts for {len(tensors)} tensors")
    _abi.reorder_beams(list(tensors), None if rows is None else list(rows), beams)


def _mx_registry(model) -> dict:
    return getattr(model, "_mamba_decode_state_kernel_caches", None) or {}


def _float_states(cache_params):
    """(list, index) of every state tensor with rows in the hybrid cache: the convolution and SSM
    states, and unquantized K/V of attention layers that are not patched."""
    for name in ("conv_states", "ssm_states", "key_cache", "value_cache"):
        held = getattr(cache_params, name, None)
        if held is None:
            continue
        for i in (held if isinstance(held, dict) else range(len(held))):
            if isinstance(held[i], torch.Tensor) and held[i].dim() > 0 and held[i].numel() > 0:
                yield held, i


def share_prompt(model, cache_params, num_beams: int) -> None:
    """After the prompts' forward pass: `num_beams` rows per prompt in place of one.

    Every INT4 layer cache becomes the shared prefix of a new, empty cache of P * num_beams rows; the
    convolution and SSM states are repeated per row, and so are their MX caches where
    register_mamba_state_kernel_caches has been called (their rounding stream is that of the larger
    batch from then on).
    """
    if num_beams < 1:
        raise ValueError(f"num_beams must be >= 1, got {num_beams}")
    caches = ia._cache_dict(cache_params)
    for layer_idx, layer in caches.items():
        if layer.prefix is not None:
            raise ValueError(f"Layer {layer_idx} already has a shared prefix")
    for layer_idx, layer in list(caches.items()):
        prompts, kv_heads, _, half = layer.k_packed.shape
        own = ia._allocate_layer_cache(prompts * num_beams, kv_heads, 16, 2 * half,
                                       layer.k_scale.shape[-1], layer.k_packed.device)
        own.prefix = layer
        caches[layer_idx] = own
    module = __import__(model.__class__.__module__, fromlist=["selective_state_update"])
    registries = [_mx_registry(model)]
    held_by_module = getattr(module, "_mamba_decode_state_kernel_caches", None)
    if held_by_module is not None and held_by_module is not registries[0]:
        registries.append(held_by_module)
    for held, i in _float_states(cache_params):
        old = held[i]
        held[i] = old.repeat_interleave(num_beams, dim=0)
        # this state's entries alone: other hybrid caches stay registered (an entry under the new
        # tensor's id can only be that of a state that is gone)
        renewed = {}
        for entries in registries:
            mx = entries.pop(id(old), None)
            entries.pop(id(held[i]), None)
            if mx is None:
                continue
            if id(mx) not in renewed:
                renewed[id(mx)] = replace(
                    mx, q_state=mx.q_state.repeat_interleave(num_beams, dim=0),
                    shared_exp=mx.shared_exp.repeat_interleave(num_beams, dim=0),
                    micro_exp=mx.micro_exp.repeat_interleave(num_beams, dim=0))
            entries[id(held[i])] = renewed[id(mx)]


def reorder_states(model, cache_params, beams: torch.Tensor) -> None:
    """reorder_beams of a hybrid cache: the live own rows of the INT4 caches, the MX caches of the
    registered SSM states and the other states themselves."""
    tensors, rows = [], []
    for layer in ia._cache_dict(cache_params).values():
        tensors += [layer.k_packed, layer.v_packed, layer.k_scale, layer.v_scale]
        rows += [layer.length] * 4
    registry = _mx_registry(model)
    for held, i in _float_states(cache_params):
        mx = registry.get(id(held[i]))
        parts = [held[i]] if mx is None else [mx.q_state, mx.shared_exp, mx.micro_exp]
        tensors += parts
        rows += [None] * len(parts)
    reorder_beams(tensors, beams, rows)


@torch.no_grad()
def beam_search(model, logits: torch.Tensor, cache_params, num_beams: int, max_new_tokens: int, *,
                start: int, eos_token_id: int | None = None, pad_token: int = 0,
                attention_mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Beam search of a patched model behind its prompts: (tokens [P, N, max_new_tokens] int64,
    scores [P, N] fp32), the beams of a prompt in descending order of their summed log-probabilities.

    logits [P, V] are the prompts' last ones and cache_params their hybrid cache, `start` the
    position of the first new token (right behind the INT4 caches' rows), attention_mask the prompts'
    2-D keep-mask, if any. A beam that has chosen eos_token_id goes on with pad_token at its score.
    """
    if max_new_tokens < 1:
        raise ValueError(f"max_new_tokens must be >= 1, got {max_new_tokens}")
    for layer_idx, layer in ia._cache_dict(cache_params).items():
        if layer.length != start:
            raise ValueError(f"start={start} is not behind the {layer.length} rows of layer {layer_idx}")
    prompts = logits.shape[0]
    device = logits.device
    scores = torch.zeros(prompts, 1, device=device, dtype=torch.float32)
    scores, _, tokens = beam_select(logits[:, None], scores, num_beams)
    finished = None if eos_token_id is None else tokens == eos_token_id
    share_prompt(model, cache_params, num_beams)
    if attention_mask is not None:
        attention_mask = attention_mask.repeat_interleave(num_beams, dim=0)
    sequences = tokens[:, :, None]
    for step in range(1, max_new_tokens):
        if attention_mask is not None:
            attention_mask = torch.nn.functional.pad(attention_mask, (0, 1), value=1)
        at = torch.tensor([start + step - 1], device=device)
        out = model(tokens.reshape(-1, 1), cache_params=cache_params, cache_position=at,
                    attention_mask=attention_mask, use_cache=True, return_dict=True)
        scores, beams, tokens = beam_select(out.logits[:, -1], scores, finished=finished,
                                            pad_token=pad_token, keep_slots=True)
        reorder_states(model, cache_params, beams)
        sequences = torch.cat((sequences.gather(1, beams[:, :, None].expand_as(sequences)),
                               tokens[:, :, None]), dim=2)
        if finished is not None:
            finished = finished.gather(1, beams) | (tokens == eos_token_id)
    order = torch.sort(scores, dim=1, descending=True, stable=True).indices
    return (sequences.gather(1, order[:, :, None].expand_as(sequences)), scores.gather(1, order))
