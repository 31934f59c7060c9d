"""The scores of beam_select against 64 bits, where the log-sum-exp's roundings add up: many terms of one
size whose low bits every addition drops, long rows, rows of a slope.

Bound: the score's own rounding, 2^-24 of it, and the sum's relative error, which its logarithm has
absolutely: fewer than 2^5 additions in a row and 7 exponentials with 6 products, 2^-24 each (an
exponential 2^-23), and the exponents' roundings, at most 2^-24 ln 2 log2(V): 61 * 2^-24 < 2^-18."""
import pytest
import torch

from layer_quant_amd import beam_decode as bd

pytestmark = pytest.mark.gpu


def check_scores(logits, num=4):
    rows = logits.shape[0]
    scores = torch.zeros(rows, 1, device=logits.device)
    got, _, tokens = bd.beam_select(logits, scores, num)
    x = logits.double()
    want = x.gather(1, tokens) - torch.logsumexp(x, 1, keepdim=True)
    assert torch.equal(x.gather(1, tokens)[:, 0], x.amax(1))
    err = (got.double() - want).abs() - 2.0 ** -24 * want.abs()
    print(f"[close] V {logits.shape[1]}: max err {err.max().item():.3g}")
    assert err.max().item() <= 2.0 ** -18


@pytest.mark.parametrize("V", [4096, 16384, 131072, 300001, 1 << 22])
@pytest.mark.parametrize("low", [3, 7, 11, 15, 31])
def test_terms_below_one(gpu, V, low):
    """Every lane has a term of 1 and others of about 1 - low * 2^-24."""
    for rows in (1, 64) if V <= 131072 else (1,):
        x = torch.full((rows, V), -low * 2.0 ** -24, device=gpu)
        x[:, ::4] = 0
        check_scores(x)
        x[:, ::4] = -low * 2.0 ** -24
        x[:, ::16] = 0
        check_scores(x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [9000, 131072, 1 << 20, 1 << 22])
def test_slopes(gpu, V, dtype):
    """Rising and falling rows: every run, wave and part rescales the sum before it."""
    up = torch.linspace(-30, 5, V, device=gpu)
    for x in (up, up.flip(0), 0.05 * up, (40 * up).clamp(-80, 80)):
        check_scores(x[None].to(dtype))


@pytest.mark.parametrize("V", [1 << 20, 1 << 24])
def test_random_long_rows(gpu, V):
    gen = torch.Generator(device=gpu).manual_seed(V)
    x = torch.randn(1, V, device=gpu, generator=gen)
    check_scores(x, 64)
    check_scores((3 * x).to(torch.bfloat16), 64)
