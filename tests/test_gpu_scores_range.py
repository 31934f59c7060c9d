"""Log-probabilities over the whole range of the logits' types: the type's lowest value as a mask, rows of it
alone, logits in the millions and far beyond, against the definition in 64 bits."""
import math

import pytest
import torch

import prompt_reference as ref
from layer_quant_amd import prompts

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
LARGEST = torch.finfo(F32).max


def check(logits, tokens, top, what):
    """NaN and infinities where they are expected (a value below fp32's range is -inf) and nowhere else. The
    rest: fp32 sums of V terms in runs of less than 64 (2^-18 of the sum), exponentials' arguments and values
    (2^-21 of them), a logarithm of up to 32 (2^-18), the result's own rounding: 2^-16 and 2^-21 of itself."""
    got = prompts.token_logprobs(logits, tokens, top)
    want, entropy, lp = ref.logprobs(logits, tokens)
    best = torch.sort(logits.float().cpu() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    known = ~torch.isnan(entropy)
    assert torch.equal(got.top_tokens.cpu()[known], best[known]), what
    pairs = [(got.logprobs, want), (got.entropy, entropy), (got.top_logprobs[known.to(logits.device)],
                                                           lp.gather(1, best)[known])]
    for g, w in pairs:
        g, w = g.double().cpu(), torch.where(w < -LARGEST, -math.inf, w)
        assert torch.equal(torch.isnan(g), torch.isnan(w)), what
        assert torch.equal(torch.isinf(g), torch.isinf(w)) and (g[torch.isinf(g)] < 0).all(), what
        fine = torch.isfinite(w)
        assert ((g - w).abs()[fine] <= 2.0 ** -16 + 2.0 ** -21 * w[fine].abs()).all(), what


def inputs(gpu, rows, vocab, seed):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    return (3 * torch.randn(rows, vocab, device=gpu, generator=gen),
            torch.randint(0, vocab, (rows,), device=gpu, generator=gen))


FORMS = [(6, 1000), (600, 1000), (5, 40000), (3, 131072)]  # a workgroup per row, wide and narrow, and parts


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("scale", [1e3, 1e5, 1e7, 1.5e8, 3e8, 1e9, 1e12, 1e25, 1e30, 1e36, 5e37])
def test_large_logits(gpu, dtype, rows, vocab, scale):
    logits, tokens = inputs(gpu, rows, vocab, 0)
    logits = logits.clamp(-6, 6) * scale
    logits[::2] = logits[::2] - logits[::2].amax(-1, keepdim=True)  # the largest 0, or small
    logits = logits.clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype)
    tokens[: rows // 2] = logits[: rows // 2].argmax(-1)
    check(logits, tokens, 7, f"{dtype} {rows} x {vocab} {scale}")


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("rows,vocab", FORMS)
def test_the_lowest_value_as_a_mask(gpu, dtype, rows, vocab):
    """All but a few tokens masked, scores of masked ones among the likeliest, rows that are masked whole, and
    rows that hold -inf, too."""
    logits, tokens = inputs(gpu, rows, vocab, 1)
    logits = logits.to(dtype)
    low = torch.finfo(dtype).min
    keep = logits[:, 500:505].clone()
    logits[:] = low
    logits[:, 500:505] = keep
    logits[0] = low
    logits[1, ::2] = -math.inf
    logits[1, 500:505] = low
    logits[2, 3:] = -math.inf
    tokens[: rows // 2] = 501
    check(logits, tokens, 32, f"{dtype} {rows} x {vocab}")


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("rows,vocab", FORMS)
def test_the_largest_value(gpu, dtype, rows, vocab):
    logits, tokens = inputs(gpu, rows, vocab, 2)
    logits = logits.to(dtype)
    logits[:, 7::13] = torch.finfo(dtype).max
    logits[0, 9] = torch.finfo(dtype).min
    tokens[0], tokens[1], tokens[2] = 9, 7, 8
    check(logits, tokens, 32, f"{dtype} {rows} x {vocab}")


def test_neighbours_where_the_sums_change_their_scale(gpu):
    """fp32 logits one and two steps apart around 2^28, 2^29 and 2^30, of both signs, in many lanes."""
    for power in (24, 28, 29, 30):
        for sign in (1, -1):
            at = torch.tensor([sign * 2.0 ** power], device=gpu)
            steps = [at]
            for direction in (math.inf, -math.inf):
                near = at
                for _ in range(2):
                    near = torch.nextafter(near, torch.full_like(near, direction))
                    steps.append(near)
            values = torch.cat(steps)
            logits = values[torch.arange(40000, device=gpu) % 5].repeat(5, 1)
            for r in range(5):
                logits[r][logits[r] == values[r]] = -math.inf
            check(logits, torch.arange(5, device=gpu), 9, f"{sign} 2^{power}")
