"""Packed calls of many prompts, most of them short or empty: every row belongs to its own."""
import math
import random

import pytest
import torch

import prompt_reference as ref
from layer_quant_amd import prompts

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def starts_of(lengths, gpu, first=0):
    return first + torch.tensor([0, *lengths], device=gpu).cumsum(0)


def check_rows_by_length(got, call, lengths, starts):
    """got [T, ...] against call(rows [n, L]) of all prompts of a length as a batch, bit for bit."""
    lengths = torch.tensor(lengths, device=got.device)
    for n in lengths.unique().tolist():
        if n == 0:
            continue
        rows = starts[:-1][lengths == n][:, None] + torch.arange(n, device=got.device)
        assert torch.equal(got[rows], call(rows)), f"prompts of {n}"


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("count", [1, 61, 62, 63, 64, 65, 126, 127, 129, 400, 509, 510, 511, 4000, 4094, 4095, 4097])
def test_attention_of_many_prompts(gpu, dtype, count):
    """As many spans as a wave's lanes, eight for each, a power of them, and one more or less; empty prompts in
    runs."""
    rng = random.Random(count)
    lengths = [rng.choice([0, 0, 0, 1, 2, 33, 130 if count < 200 else 5]) for _ in range(count)]
    lengths[rng.randrange(count)] = 300
    first, total = 7, sum(lengths) + 12
    gen = torch.Generator(device=gpu).manual_seed(count)
    q, k, v = (torch.randn(total, h, 64, device=gpu, generator=gen).to(dtype) for h in (6, 2, 2))
    starts = starts_of(lengths, gpu, first)
    got = prompts.prompt_attention(q, k, v, starts.to(torch.int32 if count % 2 else torch.int64))
    check_rows_by_length(got, lambda rows: prompts.prompt_attention(q[rows], k[rows], v[rows]), lengths, starts)
    assert not got[:first].any() and not got[total - 5:].any()


def test_attention_of_a_million_prompts(gpu):
    """Single tokens, pairs and empty ones: v itself, and the mean of two values by their scores."""
    gen = torch.Generator(device=gpu).manual_seed(0)
    lengths = torch.randint(0, 3, (1_000_000,), device=gpu, generator=gen)
    starts = torch.cat((lengths.new_zeros(1), lengths.cumsum(0)))
    total = int(starts[-1])
    q, k, v = (torch.randn(total, 1, 64, device=gpu, generator=gen).to(BF) for _ in range(3))
    got = prompts.prompt_attention(q, k, v, starts)[:, 0].double()
    want = v[:, 0].double()
    second = starts[:-1][lengths == 2] + 1
    first = second - 1
    s = torch.stack([(q[second, 0].double() * k[r, 0].double()).sum(-1) / 8 for r in (first, second)], -1)
    p = torch.softmax(s, -1)
    want[second] = p[:, :1] * v[first, 0].double() + p[:, 1:] * v[second, 0].double()
    # half a step of the output and of each weight, 2^-12 for scores of up to 2^7 in fp32
    weight = torch.maximum(v[:, 0].double().abs(), v[:, 0].double().abs().roll(1, 0))
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * weight).all()


@pytest.mark.parametrize("geometry,dtype", [((2, 64, 128), BF), ((4, 16, 32), F16), ((4, 16, 32), F32)], ids=str)
@pytest.mark.parametrize("many", [0, 3, 57, 58, 100, 505, 506, 700])
def test_scan_segments_among_many_prompts(gpu, geometry, dtype, many):
    """Prompts of several segments among few and many others (their first segments' places go by the
    prompts' number, or by the rows alone), empty ones in runs, the states in place."""
    h, p, n = geometry
    rng = random.Random(many)
    lengths = [rng.choice([0, 0, 1, 2]) for _ in range(many)] + [1100, 0, 300, 1025, 64]
    rng.shuffle(lengths)
    first, total = 5, sum(lengths) + 9
    gen = torch.Generator(device=gpu).manual_seed(many)
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen)  # noqa: E731
    x, dt, A = randn(total, h, p).to(dtype), randn(total, h) - 3, -0.2 * torch.rand(h, device=gpu, generator=gen)
    B, C = randn(total, 1, n).to(dtype), randn(total, 1, n).to(dtype)
    initial = randn(len(lengths), h, p, n)
    starts = starts_of(lengths, gpu, first)
    want, ws, wy, size = ref.scan(x, dt, A, B, C, starts.tolist(), dt_softplus=True, initial=initial)
    y, st = prompts.prompt_scan(x, dt, A, B, C, starts, dt_softplus=True, initial_states=initial, states=initial)
    # fp32 sums, steps and decays over 1100 rows 2^-16 of the terms' sum; in bf16 the factors of C half a step
    # and a state's terms 2^-24
    half = torch.finfo(dtype).eps / 2
    by = half * want.abs() + (2.0 ** -8 * (dtype == BF) + 2.0 ** -16) * wy + torch.finfo(dtype).tiny
    assert ((y.double().cpu() - want).abs() <= by).all()
    assert ((st.double().cpu() - ws).abs() <= 2.0 ** -16 * size + 1e-30).all()
    assert not y[:first].any() and not y[total - 4:].any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_of_the_most_prompts(gpu, dtype):
    """65535 prompts of a token or none: y = dt (B . C) x and the state dt x B^T."""
    gen = torch.Generator(device=gpu).manual_seed(1)
    count = 65535
    lengths = torch.randint(0, 2, (count,), device=gpu, generator=gen)
    starts = torch.cat((lengths.new_zeros(1), lengths.cumsum(0)))
    total = int(starts[-1])
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen)  # noqa: E731
    x, dt, A = randn(total, 2, 8).to(dtype), torch.rand(total, 2, device=gpu, generator=gen), -torch.ones(2, device=gpu)
    B, C = randn(total, 1, 16).to(dtype), randn(total, 1, 16).to(dtype)
    y, st = prompts.prompt_scan(x, dt, A, B, C, starts)
    xd, dd, Bd, Cd = (t.double() for t in (x, dt, B, C))
    terms = (dd * (Bd.abs() * Cd.abs()).sum(-1))[..., None] * xd.abs()
    want = (dd * (Bd * Cd).sum(-1))[..., None] * xd
    assert ((y.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -18 * terms).all()
    state = (dd[..., None] * xd)[..., None] * Bd[:, :, None]
    assert ((st[lengths == 1].double() - state).abs() <= 2.0 ** -20 * state.abs()).all()
    assert not st[lengths == 0].any()
    assert math.isfinite(y.float().abs().max())
