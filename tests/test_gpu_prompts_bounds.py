"""Starts that do not ascend: no defined values, and nothing written outside the outputs and the workspace."""
import random

import pytest
import torch

from layer_quant_amd import _abi, prompts

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROWS, SENTINEL = 1500, 7.0


def wild_starts():
    rng = random.Random(0)
    yield from ([0, 1500, 0, 1500, 0, 1500], [1500, 0], [-5, 3000, 7, -1, 1500], [900, 900, 100, 1500], [0, 0, 0])
    for count in (3, 64, 65, 66, 200):
        yield [rng.randrange(-100, 1600) for _ in range(count)]
    yield [0, 1500] * 100
    yield sorted(rng.randrange(0, 1500) for _ in range(130))[::-1]


def inside(shape, gpu, dtype):
    """A tensor between two stretches of sentinels, all of them, and where it lies."""
    n = 1
    for s in shape:
        n *= s
    whole = torch.full((n + 8192,), SENTINEL, device=gpu, dtype=dtype)
    return whole, whole[4096:4096 + n].view(shape)


def untouched(whole, n):
    return (whole[:4096] == SENTINEL).all() and (whole[4096 + n:] == SENTINEL).all()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_scan_writes_nothing_outside(gpu, dtype, index):
    gen = torch.Generator(device=gpu).manual_seed(0)
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen)  # noqa: E731
    h, p, n = 4, 64, 128
    x, dt, A = randn(ROWS, h, p).to(dtype), randn(ROWS, h), -torch.rand(h, device=gpu, generator=gen)
    B, C = randn(ROWS, 1, n).to(dtype), randn(ROWS, 1, n).to(dtype)
    for s in wild_starts():
        starts, prompts_ = torch.tensor(s, device=gpu, dtype=index), len(s) - 1
        initial = randn(prompts_, h, p, n)
        outs, out = inside((ROWS, h, p), gpu, dtype)
        held, states = inside((prompts_, h, p, n), gpu, F32)
        need = _abi.lib().lq_prompt_scan_workspace(_abi.DTYPE_CODES[dtype], prompts_, ROWS, 1, h, p, n)
        work = torch.full((need + 8192,), 7, device=gpu, dtype=torch.uint8)
        stream = torch.cuda.current_stream().cuda_stream
        args = map(_abi.desc, (x, dt, A, B, C, starts, None, None, None, initial, states, out))
        rc = _abi.lib().lq_prompt_scan(*args, 1, 0.0, 10.0, work.data_ptr() if need else None, need, stream)
        assert rc == 0, _abi.last_error()
        torch.cuda.synchronize()
        assert untouched(outs, out.numel()) and untouched(held, states.numel()), s
        assert (work[need:] == 7).all(), s


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_writes_nothing_outside(gpu, dtype):
    gen = torch.Generator(device=gpu).manual_seed(1)
    q, k, v = (torch.randn(ROWS, h, 64, device=gpu, generator=gen).to(dtype) for h in (6, 2, 2))
    for s in wild_starts():
        outs, out = inside((ROWS, 6, 64), gpu, dtype)
        prompts.prompt_attention(q, k, v, torch.tensor(s, device=gpu), out=out)
        torch.cuda.synchronize()
        assert untouched(outs, out.numel()), s
