"""Values of inf and NaN that attention sees, and values so large that unnormalised sums of them would leave
fp32, against the definition in 64 bits, element by element."""
import math

import pytest
import torch

import prompt_reference as ref
from layer_quant_amd import prompts

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def agree(got, want, bound, what):
    """NaN and infinities (with their signs) where they are expected and nowhere else, the rest within bound."""
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN places"
    assert torch.equal(got == math.inf, want == math.inf), f"{what}: inf places"
    assert torch.equal(got == -math.inf, want == -math.inf), f"{what}: -inf places"
    fine = torch.isfinite(want)
    err = (got - want).abs()[fine] / bound[fine].clamp_min(1e-300)
    assert not err.numel() or err.amax() <= 1, f"{what}: {err.amax():.3g}"


def inputs(gpu, rows, d, dtype, hq=4, hkv=2, seed=0):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    return [torch.randn(rows, h, d, device=gpu, generator=gen).to(dtype) for h in (hq, hkv, hkv)]


def check(q, k, v, starts, what):
    got = prompts.prompt_attention(q, k, v, torch.tensor(starts, device=q.device))
    want, weight, score = ref.attention(q, k, v, starts)
    agree(got, want, ref.attention_bound(want, weight, score, q.dtype, q.shape[-1]), what)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("d", [64, 72, 128, 256])
@pytest.mark.parametrize("at", [0, 31, 40, 63, 64, 100, 199])
def test_infinite_values_that_rows_see(gpu, dtype, d, at):
    """In a prompt's first tile, a later one, its last row; the rows behind get the infinity, and NaN where
    both signs, or a NaN, are seen."""
    q, k, v = inputs(gpu, 260, d, dtype)
    v[at, 0, 3], v[at, 0, 60], v[at, 1, 5] = math.inf, -math.inf, math.nan
    v[at, 1, 63] = math.inf
    v[min(at + 20, 199), 1, 63] = -math.inf if at < 199 else math.inf
    check(q, k, v, [0, 200, 260], f"{dtype} {d} {at}")


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_an_infinite_value_of_little_weight(gpu, dtype, d):
    """Keys whose weight 2^-1000 is no fp32 number: the rows that see their infinite values are not finite
    there, and finite elsewhere."""
    q, k, v = inputs(gpu, 150, d, dtype, seed=1)
    q[:], k[:] = 1.0, 0.0
    k[:70] = -700.0 / d
    v[5, :, 7], v[90, :, 9] = math.inf, -math.inf
    got = prompts.prompt_attention(q, k, v, torch.tensor([0, 150], device=gpu), scale=1.0).cpu()
    assert not torch.isfinite(got[5:, :, 7]).any() and (got[90:, :, 9] == -math.inf).all()
    got[5:, :, 7] = got[90:, :, 9] = 0
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("general", [False, True])
def test_values_next_to_the_largest(gpu, dtype, d, general, diag):
    """3000 values of up to 3e38, whose plain sum is beyond fp32 and whose mean is not; the next prompt's
    ordinary ones."""
    if general:
        diag.set("LQ_PROMPT_FORCE_GENERIC")
    q, k, v = inputs(gpu, 3100, d, dtype, 2, 1, seed=2)
    v[:3000] = (v[:3000].float().abs().clamp(0.1, 1) * 3e38).to(dtype)
    rows = torch.tensor([0, 1, 7, 63, 64, 500, 2999, 3000, 3050, 3099])
    got = prompts.prompt_attention(q, k, v, torch.tensor([0, 3000, 3100], device=gpu)).cpu()
    for t in rows.tolist():
        first = 0 if t < 3000 else 3000
        kk, vv = (x[first:t + 1, 0].double().cpu() for x in (k, v))
        qt = q[t].double().cpu()
        p = torch.softmax(qt @ kk.T / math.sqrt(d), -1)
        score = (qt.abs() @ kk.abs().T / math.sqrt(d)).amax(-1)
        want, weight = p @ vv, p @ vv.abs()
        agree(got[t], want, ref.attention_bound(want, weight, score, dtype, d), f"row {t}")
