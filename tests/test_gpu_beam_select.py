"""beam_select against a sort of the totals in 64 bits.

The beams and tokens have to be equal. A score is the total rounded to fp32 (half a step, 2^-24
relative) and is off by the log-sum-exp's error: sums of fp32 terms whose roundings add up to less than
2^-19 relative (at most 2^5 additions in a row, each 2^-24, and the exponential's 2^-22), which is the
error of its logarithm."""
import numpy as np
import pytest
import torch

from layer_quant_amd import beam_decode as bd

pytestmark = pytest.mark.gpu


def reference(logits, scores, num, finished=None, pad=0, slots=False):
    """(scores, beams, tokens) in 64 bits on the CPU."""
    P, N = scores.shape
    x = logits.detach().cpu().double().reshape(P, N, -1).numpy()
    s = scores.cpu().double().numpy()
    V = x.shape[-1]
    outs = np.zeros((P, num)), np.zeros((P, num), np.int64), np.zeros((P, num), np.int64)
    for p in range(P):
        total = np.full((N, V), -np.inf)
        for n in range(N):
            if finished is not None and bool(finished[p, n]):
                total[n, pad] = s[p, n] if np.isfinite(s[p, n]) else -np.inf
                continue
            with np.errstate(all="ignore"):
                m = x[p, n].max()
                base = s[p, n] - (m + np.log(np.exp(x[p, n] - m).sum()))
                if np.isfinite(base):
                    total[n] = base + x[p, n]
        flat = total.reshape(-1)
        best = [int(i) for i in np.argsort(-flat, kind="stable")[:num]]
        if slots:
            place, rest = [None] * N, []
            for i in best:
                if place[i // V] is None:
                    place[i // V] = i
                else:
                    rest.append(i)
            best = [i if i is not None else rest.pop(0) for i in place]
        for k, i in enumerate(best):
            outs[0][p, k], outs[1][p, k], outs[2][p, k] = flat[i], i // V, i % V
    return outs


def check(logits, scores, num=None, **kw):
    got = bd.beam_select(logits, scores, num, finished=kw.get("finished"), pad_token=kw.get("pad", 0),
                         keep_slots=kw.get("slots", False))
    fin = kw.get("finished")
    want = reference(logits, scores, num or scores.shape[1], None if fin is None else fin.cpu(),
                     kw.get("pad", 0), kw.get("slots", False))
    assert np.array_equal(got[1].cpu().numpy(), want[1]), (got[1].cpu(), want[1])
    assert np.array_equal(got[2].cpu().numpy(), want[2]), (got[2].cpu(), want[2])
    s, w = got[0].cpu().double().numpy(), want[0]
    live = np.isfinite(w)
    assert np.array_equal(live, np.isfinite(s)) and np.array_equal(s[~live], w[~live])
    assert np.all(np.abs(s[live] - w[live]) <= 2.0 ** -24 * np.abs(w[live]) + 2.0 ** -19)
    return got


def random(gpu, P, N, V, dtype, seed, std=3.0):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    logits = (std * torch.randn(P * N, V, device=gpu, generator=gen)).to(dtype)
    return logits, -30 * torch.rand(P, N, device=gpu, generator=gen)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P,N,V,num", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 21), (1, 64, 100, 64),
                                       (3, 5, 4095, 10), (1, 2, 4096, 64), (2, 4, 4097, 8),
                                       (1, 1, 50257, 33), (5, 7, 32001, 14), (2, 16, 131072, 32)])
def test_random(gpu, dtype, P, N, V, num):
    logits, scores = random(gpu, P, N, V, dtype, seed=V + num)
    check(logits, scores, num)
    if num >= N:
        check(logits, scores, slots=True)
    torch.manual_seed(V)
    fin = torch.rand(P, N, device=gpu) < 0.5
    check(logits, scores, num, finished=fin, pad=V // 2)


@pytest.mark.parametrize("V", [3, 64, 1000, 9001])
def test_ties_and_borders(gpu, V):
    """Equal logits within a beam and between equal beams, banned tokens, rows without a score."""
    P, N, num = 2, 4, 8
    gen = torch.Generator(device=gpu).manual_seed(V)
    same = torch.zeros(P * N, V, device=gpu)
    scores = torch.zeros(P, N, device=gpu)
    check(same, scores, num)
    check(torch.full_like(same, -0.0) * (torch.arange(V, device=gpu) % 2), scores, num)
    few = torch.randint(0, 3, (1, V), device=gpu, generator=gen).float().expand(P * N, V)
    check(few, scores, num)
    check(few.to(torch.bfloat16), scores, num, slots=False)
    check(few, scores, slots=True)
    banned = torch.where(torch.rand(P * N, V, device=gpu, generator=gen) < 0.9, -torch.inf, few)
    banned[1] = -torch.inf
    check(banned, scores, num)
    banned[2, V // 2] = torch.nan
    banned[3, V - 1] = torch.inf
    check(banned, scores, num)
    scores[0] = torch.tensor([-torch.inf, 0.0, torch.nan, torch.inf])
    check(few, scores, num)
    check(few, scores, num, finished=torch.tensor([[True, True, True, False]] * P, device=gpu), pad=V - 1)
    check(few, scores, num, finished=torch.ones(P, N, dtype=torch.bool, device=gpu), pad=1)
    # the first step of beams that are all the same but the first
    scores = torch.full((P, N), -1e9, device=gpu)
    scores[:, 0] = 0
    logits, _ = random(gpu, P, N, V, torch.float32, 3)
    check(logits, scores)


@pytest.mark.parametrize("N,num", [(8, 32), (16, 32), (64, 64)])
@pytest.mark.parametrize("V", [700, 9001, 40000])
def test_many_equal_totals(gpu, N, num, V):
    """More candidates at the border than the final list holds, and lists that overflow."""
    gen = torch.Generator(device=gpu).manual_seed(V + N)
    scores = torch.zeros(2, N, device=gpu)
    row = torch.randint(0, 2, (1, V), device=gpu, generator=gen).float()
    for logits in (torch.zeros(2 * N, V, device=gpu), row.expand(2 * N, V),
                   torch.where(row > 0, 0.0, -torch.inf).expand(2 * N, V).to(torch.bfloat16),
                   torch.full((2 * N, V), -torch.inf, device=gpu)):
        check(logits, scores, num)
        check(logits, scores, slots=True)
        check(logits, scores, num, finished=torch.arange(2 * N, device=gpu).reshape(2, N) % 3 == 0, pad=V - 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sorted_rows(gpu, dtype):
    """The largest logits all next to each other, at the row's start, end or middle."""
    x = torch.linspace(0, 40, 9000, device=gpu).to(dtype)
    rows = torch.stack((x, x.flip(0), x.roll(4500), torch.where(x > 39, x, -torch.inf)))
    check(rows, torch.zeros(1, 4, device=gpu), 64)
    check(rows, torch.zeros(4, 1, device=gpu), 64)


def test_layouts(gpu):
    """Strided logits, scores and flags, rows at odd addresses, three dimensions."""
    P, N, V = 3, 4, 5001
    base, scores = random(gpu, P, N, 2 * V + 3, torch.bfloat16, 1)
    for x in (base[:, 1:V + 1], base[:, 3:2 * V + 3:2], base[:, :V].flip(1),
              base[:, :V].t().contiguous().t(), base[:1, :V].expand(P * N, V),
              base[:, :V].reshape(P, N, V), base.reshape(P, N, -1)[:, :, 7:V + 7]):
        check(x, scores)
        assert torch.equal(x, x.clone())
    wide = torch.empty(N, 2 * P, device=gpu).t()[::2]
    wide.copy_(scores)
    torch.manual_seed(6)
    fin = torch.rand(P, 2 * N, device=gpu)[:, ::2] < 0.4
    check(base[:, :V], wide, 2 * N, finished=fin, pad=17)


def test_stream_and_capture(gpu):
    """On a side stream, and captured: replays follow the inputs, with eager calls of larger shapes
    in between (which grow the eager scratch)."""
    logits, scores = random(gpu, 2, 4, 40001, torch.bfloat16, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(logits, scores)
        graphs = []
        for num in (4, 8):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = bd.beam_select(logits, scores, num)
            graphs.append((g, num, out))
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        new, s = random(gpu, 2, 4, 40001, torch.bfloat16, 50 + seed)
        logits.copy_(new)
        scores.copy_(s)
        big, bs = random(gpu, 16, 8, 100003, torch.bfloat16, seed)
        bd.beam_select(big, bs, 64)
        for g, num, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, num, out in graphs:
            want = reference(logits, scores, num)
            assert np.array_equal(out[1].cpu().numpy(), want[1])
            assert np.array_equal(out[2].cpu().numpy(), want[2])
