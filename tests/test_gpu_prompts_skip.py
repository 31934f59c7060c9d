"""The D x term of the recurrence: D is an fp32 parameter, and what is rounded is the result."""
import math

import pytest
import torch

import prompt_reference as ref
from layer_quant_amd import prompts

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("rows", [1, 63, 64, 65, 200, 3000])
def test_d_is_not_rounded_to_the_inputs_type(gpu, dtype, rows):
    """C = 0: y = D x. Half a step of the type, and 2^-16 for D as the sum of two bf16 values (2^-8 of each
    one's rest, less than 2^-17 of D) and the products' fp32 sum."""
    gen = torch.Generator(device=gpu).manual_seed(rows)
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen)  # noqa: E731
    x, dt, A, D = randn(rows, 6, 64).to(dtype), randn(rows, 6), -torch.rand(6, device=gpu, generator=gen), randn(6)
    B = randn(rows, 1, 128).to(dtype)
    y, _ = prompts.prompt_scan(x[None], dt[None], A, B[None], torch.zeros_like(B)[None], D=D, dt_softplus=True)
    want = x.double() * D.double()[:, None]
    bound = (torch.finfo(dtype).eps / 2 + 2.0 ** -16) * want.abs() + torch.finfo(dtype).tiny
    assert ((y[0].double() - want).abs() <= bound).all()


def test_infinite_d(gpu):
    """An infinite D makes its head's rows infinite, with the sign of D x, and leaves the other heads (their
    bounds: the result's rounding; in bf16 half a step of the mixing weights and the state, 2^-8 of the terms'
    sum, else 2^-16 for fp32 sums, steps and decays)."""
    gen = torch.Generator(device=gpu).manual_seed(0)
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen)  # noqa: E731
    for dtype in (BF, F16, F32):
        x, dt, A = randn(100, 4, 64).to(dtype), randn(100, 4), -torch.ones(4, device=gpu)
        x[x == 0] = 1
        B, C, D = randn(100, 1, 128).to(dtype), randn(100, 1, 128).to(dtype), randn(4)
        want, _, terms, _ = ref.scan(x, dt, A, B, C, [0, 100], D=D, dt_softplus=True)
        bound = torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -8 * (dtype == BF) + 2.0 ** -16) * terms
        D[1], D[2] = math.inf, -math.inf
        y = prompts.prompt_scan(x[None], dt[None], A, B[None], C[None], D=D, dt_softplus=True)[0][0].cpu()
        for h, sign in ((1, 1), (2, -1)):
            assert (y[:, h] == sign * math.inf * x[:, h].cpu().sign()).all()
        for h in (0, 3):
            assert ((y[:, h].double() - want[:, h]).abs() <= bound[:, h] + torch.finfo(dtype).tiny).all()
