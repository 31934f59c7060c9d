"""beam_select where a wave holds four runs of a row (64 logits per lane, rows * ceil(V / 1024) >= 32 times
the GPU's CUs), and rows of more than 64 parts, against the 64-bit sort of test_gpu_beam_select.py."""
import numpy as np
import pytest
import torch

from test_gpu_beam_select import check, random, reference

from layer_quant_amd import beam_decode as bd

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def four_runs(gpu, rows, V):
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count
    return rows * ((V + 1023) // 1024) >= 32 * cus


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("P,N,V,num", [(8, 8, 131072, 8), (16, 8, 100003, 64)])
def test_four_runs(gpu, dtype, P, N, V, num):
    assert four_runs(gpu, P * N, V)
    logits, scores = random(gpu, P, N, V, dtype, V)
    before = logits.clone()
    check(logits, scores, num)
    torch.manual_seed(V)
    check(logits, scores, slots=True, finished=torch.rand(P, N, device=gpu) < 0.4, pad=V - 1)
    assert torch.equal(logits, before)


@pytest.mark.parametrize("dtype", DTYPES)
def test_four_runs_of_strided_rows(gpu, dtype):
    P, N, V = 2, 64, 66001
    assert four_runs(gpu, P * N, V)
    wide, scores = random(gpu, P, N, 2 * V, dtype, 7)
    check(wide[:, 1::2], scores, 33)
    check(wide[:, :V].flip(1).t().contiguous().t(), scores, 33)
    check(wide[:, 1:V + 1], scores, 33)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("num", [5, 64])
@pytest.mark.parametrize("kind", ["equal", "few", "sorted", "falling", "banned", "mostly -inf", "-inf"])
def test_four_runs_of_ties_and_slopes(gpu, dtype, num, kind):
    """Lists that overflow are cut on the way; parts and whole rows without a logit above -inf."""
    P, N, V = 2, 64, 65537
    assert four_runs(gpu, P * N, V)
    gen = torch.Generator(device=gpu).manual_seed(V)
    few = torch.randint(0, 3, (1, V), device=gpu, generator=gen).float()
    rand = torch.rand(N * P, V, device=gpu, generator=gen)
    at = torch.arange(V, device=gpu)
    x = {"equal": torch.zeros(1, V, device=gpu), "few": few,
         "sorted": torch.linspace(-20, 20, V, device=gpu)[None],
         "falling": torch.linspace(20, -20, V, device=gpu)[None],
         "banned": torch.where(rand < 0.99, -torch.inf, few),
         "mostly -inf": torch.where((at < 16000) | (at % 5000 == 3), -torch.inf, few),
         "-inf": torch.full((1, V), -torch.inf, device=gpu)}[kind].to(dtype).expand(P * N, V)
    scores = torch.zeros(P, N, device=gpu)
    check(x, scores, num)
    check(x.contiguous(), scores, slots=True)
    torch.manual_seed(num)
    check(x, -torch.rand(P, N, device=gpu), num, finished=torch.arange(P * N, device=gpu).reshape(P, N) % 3 == 0,
          pad=V - 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("P,N,V", [(1, 2, 300001), (1, 2, 1 << 22), (2, 1, 1048577)])
def test_rows_of_many_parts(gpu, dtype, P, N, V):
    """More parts than a wave has lanes, and more than the final workgroup has threads."""
    logits, scores = random(gpu, P, N, V, dtype, V)
    check(logits, 0 * scores, 64)
    check(logits, 0 * scores, N, slots=True)
    check((logits * 2).round().clamp(-6, 6), 0 * scores, 64)
    check(logits, scores, 16, finished=torch.arange(P * N, device=gpu).reshape(P, N) == 1, pad=V - 1)


def test_capture_with_a_large_eager_call_in_between(gpu):
    """The eager call that grows the scratch between replays gives its own right result."""
    small, scores = random(gpu, 2, 4, 40001, torch.bfloat16, 5)
    big, bs = random(gpu, 16, 8, 100003, torch.bfloat16, 6)
    want, want_big = reference(small, scores, 8), reference(big, bs, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            out = bd.beam_select(small, scores, 8)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        got = bd.beam_select(big, bs, 64)
        g.replay()
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(got[1:], want_big[1:]))
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(out[1:], want[1:]))
