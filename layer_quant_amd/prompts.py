"""Whole prompts through the hybrid model's two mixers, and the scores of given tokens (no reference
counterpart: its driver walks a text token by token, and leaves prompts to the remote module).

    prompt_attention  causal attention of prompts over their own keys      -> lq_prompt_attention
    prompt_scan       the Mamba2 recurrence over prompts, with its states  -> lq_prompt_scan
    token_logprobs    log-probabilities of given tokens, entropy, the likeliest alternatives
                                                                           -> lq_token_logprobs

Prompts are a batch of equal lengths [B, L, ...], or packed one behind another [T, ...] with `starts`, an
int32 or int64 tensor [S + 1] on the GPU: prompt s has rows [starts[s], starts[s + 1]), so that texts of
different lengths run without padding. Nothing waits for the GPU: the starts are read by the kernels, and
a captured call takes the starts that stand there at replay. They must ascend within [0, T]. Rows of no
prompt (in front of starts[0], behind starts[-1]) give zeros. The pad tokens of a padded batch can stand
behind each text (nothing behind a row reaches it), or be prompts of their own between packed texts.

Forward only, like every operator here: inputs that require gradients are refused while gradients are
enabled.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _abi


def _no_gradients(*tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("the prompt operators have no backward: call them under torch.no_grad()")


def _check_prompts(name: str, t: torch.Tensor, starts: torch.Tensor | None) -> None:
    if starts is None:
        if t.dim() != 4:
            raise ValueError(f"Expected {name} [batch, length, heads, dim] without starts, got "
                             f"{tuple(t.shape)}")
    elif t.dim() != 3:
        raise ValueError(f"Expected {name} [rows, heads, dim] with starts, got {tuple(t.shape)}")
    elif starts.dim() != 1 or starts.numel() < 1 or starts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"Expected starts int32 or int64 [prompts + 1], got {starts.dtype} "
                         f"{tuple(starts.shape)}")


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                     starts: torch.Tensor | None = None, *, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of whole prompts: query [T, Hq, D], key and value [T, Hkv, D] with `starts`, or
    [B, L, heads, D] without, in fp32, fp16 or bf16 with any strides; Hq a multiple of Hkv, D <= 256.
    Row t of a prompt attends to the prompt's rows up to t; scale is 1 / sqrt(D) unless given.
    -> query's shape and dtype, in `out` where given (which may be query, and overlaps no key or value).

    Scores, softmax and sums are fp32 (16-bit inputs: the weights are rounded to that type before
    they multiply the values). What stands behind a row in its prompt never reaches its result, be it NaN. A
    value of inf or NaN that it sees does, as that infinity (NaN where its weight is below 2^-80) or as NaN.
    """
    _check_prompts("query", query, starts)
    _no_gradients(query, key, value)
    if out is None:
        out = torch.empty(query.shape, device=query.device, dtype=query.dtype)
    if scale is None:
        scale = 1.0 / math.sqrt(max(query.shape[-1], 1))
    return _abi.prompt_attention(query, key, value, starts, out, float(scale))


def prompt_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                starts: torch.Tensor | None = None, *, D: torch.Tensor | None = None,
                z: torch.Tensor | None = None, dt_bias: torch.Tensor | None = None,
                dt_softplus: bool = False, dt_limit: tuple[float, float] = (0.0, math.inf),
                initial_states: torch.Tensor | None = None,
                states: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The Mamba2 recurrence over whole prompts (mamba_state_8b_kernel.selective_state_update over each
    prompt's tokens in one call): (y in x's shape and dtype, states [S, H, P, N]).

    x [T, H, P], dt [T, H], B, C [T, G, N] with `starts`, or [B, L, ...] without (S = B then); A, D,
    dt_bias [H]; z like x. Per head: dt = clamp(softplus(dt + dt_bias), *dt_limit);
    S = exp(A dt) S + dt x B^T from initial_states [S, H, P, N] or zero; y = S C + D x, times silu(z).
    Any strides; x, B and C of one dtype, the rest fp32, fp16 or bf16; N <= 256.

    The states behind the prompts go to `states`, of any float dtype (the cache's own tensor, and the
    same as initial_states to go on in place; they overlap in no other way), or to a new fp32 tensor; a
    prompt without rows hands its initial state on.

    States and sums are fp32. bf16 prompts of heads of 64 and states of 128 run on matrix instructions: there
    the state in front of each 64 rows and the weights of x within them are rounded to bf16 before they make y
    (half a step of each term, beside y's own rounding), and what a row adds to the state is off by 2^-16 of
    itself, or 2^-24 where `states` are fp32. The other prompts round what they return and nothing else.

    What stands behind a row in its prompt never reaches it. An x of inf or NaN leaves every y and state
    that it reaches not finite, inf or NaN (the sign of an infinity is not followed through the products).
    """
    _check_prompts("x", x, starts)
    _no_gradients(x, dt, A, B, C, D, z, dt_bias, initial_states)
    if B.dim() != x.dim():
        raise ValueError(f"Expected B and C of x's rank {x.dim()}, got {tuple(B.shape)}")
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    if states is None:
        prompts = x.shape[0] if starts is None else starts.numel() - 1
        states = torch.empty((prompts, *x.shape[-2:], B.shape[-1]), device=x.device,
                             dtype=torch.float32)
    low, high = dt_limit
    _abi.prompt_scan(x, dt, A, B, C, starts, D, z, dt_bias, initial_states, states, out, dt_softplus,
                     float(low), float(high))
    return out, states


class TokenLogprobs(NamedTuple):
    """Of each row: the given token's log-probability, the entropy (nats), and the `top` likeliest
    tokens with their log-probabilities (None where top is 0)."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor | None
    top_tokens: torch.Tensor | None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Scores of tokens [...] (int64) under logits [..., V] (fp32, fp16 or bf16, any strides, one or two
    leading dims): log_softmax(logits)[token] in fp32, without the log-softmax of the other tokens in
    memory. A token outside [0, V), such as -100, gives 0.

    `top` (<= 32): the largest logits in descending order, equal ones by the lower token. A row with a
    NaN or +inf logit, or without one above -inf, gives NaN. To score a text: logits[:, :-1] and
    ids[:, 1:]."""
    if logits.dim() not in (2, 3) or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"Expected logits [rows, vocab] or [batch, length, vocab] and a token for each "
                         f"row, got {tuple(logits.shape)} and {tuple(tokens.shape)}")
    if top < 0:
        raise ValueError(f"top must not be negative, got {top}")
    _no_gradients(logits)
    lead, device = tokens.shape, logits.device
    logprobs = torch.empty(lead, device=device, dtype=torch.float32)
    entropy = torch.empty(lead, device=device, dtype=torch.float32)
    top_logprobs = top_tokens = None
    if top:
        top_logprobs = torch.empty((*lead, top), device=device, dtype=torch.float32)
        top_tokens = torch.empty((*lead, top), device=device, dtype=torch.int64)
    _abi.token_logprobs(logits, tokens, logprobs, entropy, top_logprobs, top_tokens)
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_tokens)
