"""The order of equal and nearly equal totals in beam_select: totals are compared in all 64 bits, equal
ones by the lower n * V + t."""
import math

import pytest
import torch

from layer_quant_amd import beam_decode as bd
from test_gpu_beam_select import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("parts", [16, 64])
def test_totals_that_differ_in_the_last_bit(gpu, first, parts):
    """One beam whose totals lie between 512 and 1024, where 64-bit numbers are 2^-43 apart: every logit
    is `first` steps, those of the 63 last tokens one more (and one token 4, so that the log-sum-exp does
    not depend on `first`). For one of the two `first` the totals differ in their lowest bit alone."""
    V, step = 4096 * parts, 2.0 ** -43
    logits = torch.full((1, V), first * step, device=gpu)
    logits[:, -63:] = (first + 1) * step
    logits[:, 5] = 4 * step
    out = bd.beam_select(logits, torch.full((1, 1), 1000.0, device=gpu), 64)
    assert out[2][0].tolist() == [5] + list(range(V - 63, V))
    assert abs(out[0][0, 0].item() - (1000 - math.log(V))) < 1e-3


@pytest.mark.parametrize("V,num", [(64, 8), (5, 5), (1000, 64), (9001, 33)])
@pytest.mark.parametrize("score", [-math.inf, math.nan, math.inf])
def test_finished_beams_without_a_score(gpu, V, num, score):
    """Every continuation of a finished beam at -inf is equal: the lowest indices, wherever the pad token is."""
    logits = torch.randn(3 * 2, V, device=gpu)
    scores = torch.full((3, 2), score, device=gpu)
    fin = torch.ones(3, 2, dtype=torch.bool, device=gpu)
    for pad in (0, V // 2, V - 1):
        check(logits, scores, num, finished=fin, pad=pad)
    fin[1, 0] = False  # beside beams that go on, with and without a score
    check(logits, scores, num, finished=fin, pad=V - 1)
    scores[1, 0], scores[2, 1] = -3.0, -1.0
    check(logits, scores, num, finished=fin, pad=V - 1)
