"""Outputs that share memory with what a call reads, or with themselves, are refused; views that take turns
in one tensor are not. Made-up addresses, never read: an accepted call ends at the next refusal (fp32 never
takes the matrix kernel, which the diagnostic switch requires)."""
import ctypes
import itertools
import random

import pytest
import torch

from layer_quant_amd import _abi

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32
BASE = 1 << 20


def fake(shape, stride, at=0, dtype=F32):
    t = _abi.LQTensor()
    t.data, t.dtype, t.ndim = BASE + at, _abi.DTYPE_CODES[dtype], len(shape)
    for i, (n, s) in enumerate(zip(shape, stride)):
        t.shape[i], t.stride[i] = n, s
    return t


def dense(shape, at=0, dtype=F32):
    stride = [1] * len(shape)
    for i in range(len(shape) - 2, -1, -1):
        stride[i] = stride[i + 1] * shape[i + 1]
    return fake(shape, stride, at, dtype)


def refused(call):
    with _abi.diagnostic("LQ_PROMPT_REQUIRE_MFMA"):
        assert call() == -1
    error = _abi.last_error()
    assert "overlap" in error or "general kernel" in error, error
    return "overlap" in error


def attention(q, k, v, out, starts=None):
    p = lambda t: None if t is None else ctypes.pointer(t)  # noqa: E731
    return refused(lambda: _abi.lib().lq_prompt_attention(p(q), p(k), p(v), p(starts), p(out), 0.1, None))


def bytes_of(t):
    size = 2 if t.dtype == _abi.DTYPE_CODES[BF] else 4
    at = [t.data + size * sum(i * s for i, s in zip(index, t.stride))
          for index in itertools.product(*(range(t.shape[d]) for d in range(t.ndim)))]
    return at, {a + b for a in at for b in range(size)}


FAR = 1 << 18


def test_attention_over_its_own_inputs():
    starts = dense((3,), 3 * FAR, I32)
    q, k, v = dense((10, 4, 8)), dense((10, 2, 8), FAR), dense((10, 2, 8), 2 * FAR)
    assert not attention(q, k, v, dense((10, 4, 8), 4 * FAR), starts)
    assert not attention(q, k, v, q, starts)
    assert attention(q, k, v, dense((10, 4, 8), 4), starts), "q, but not in its places"
    assert attention(q, k, v, fake((10, 4, 8), (8, 80, 1)), starts), "q in other strides"
    for at in (FAR, FAR + 10 * 2 * 8 * 4 - 4, 2 * FAR - 10 * 4 * 8 * 4 + 4, 2 * FAR, 3 * FAR + 8):
        assert attention(q, k, v, dense((10, 4, 8), at), starts), at
    for at in (FAR + 10 * 2 * 8 * 4, 2 * FAR - 10 * 4 * 8 * 4, 3 * FAR + 12):
        assert not attention(q, k, v, dense((10, 4, 8), at), starts), at


@pytest.mark.parametrize("stride", [(0, 8, 1), (32, 0, 1), (32, 8, 0), (31, 8, 1), (32, 7, 1), (4, 1, 1)])
def test_attention_out_over_itself(stride):
    q, k = dense((10, 4, 8)), dense((10, 2, 8), FAR)
    starts = dense((3,), 3 * FAR, I32)
    assert attention(q, k, k, fake((10, 4, 8), stride, 4 * FAR), starts)
    assert not attention(q, k, k, fake((10, 4, 8), (1, 80, 10), 4 * FAR), starts)


def test_attention_in_fused_rows():
    """q, k and v of one tensor, out in q's place or in one more, in the layouts of projections."""
    starts = dense((3,), 3 * FAR, I32)
    row = (4 + 2 + 2 + 4) * 8
    part = lambda heads, at: fake((10, heads, 8), (row, 8, 1), 4 * at)  # noqa: E731
    q, k, v, more = part(4, 0), part(2, 32), part(2, 48), part(4, 64)
    assert not attention(q, k, v, q, starts) and not attention(q, k, v, more, starts)
    assert attention(q, k, v, part(4, 40), starts) and attention(q, k, v, part(4, 33), starts)
    # rows one further: out's last ones lie behind the tensor
    assert not attention(q, k, v, part(4, 64 + row), starts)
    assert attention(q, k, v, part(4, 32 + 3 * row), starts)
    # [B, heads, L, D], a batch
    one = 10 * 8
    block = lambda heads, at: fake((3, 10, heads, 8), (12 * one, 8, one, 1), 4 * at)  # noqa: E731
    q, k, v, more = block(4, 0), block(2, 4 * one), block(2, 6 * one), block(4, 8 * one)
    assert not attention(q, k, v, q) and not attention(q, k, v, more)
    assert attention(q, k, v, block(4, 7 * one)) and attention(q, k, v, block(4, 3 * one + 1))


def test_overlap_is_found_among_random_layouts():
    """Every call whose bytes overlap is refused, and none that shares its rows' stride without overlapping."""
    rng = random.Random(0)
    seen = [0, 0]
    for _ in range(1500):
        rows, hq, d = rng.randint(1, 4), rng.choice([1, 2, 4]), rng.randint(1, 4)
        hkv = rng.choice([h for h in (1, 2, 4) if hq % h == 0])
        shared = rng.random() < 0.5
        row = rng.randint(hq * d, 4 * hq * d)

        def layout(heads):
            head, dim = (d, 1) if rng.random() < 0.7 else (1, heads)
            return fake((rows, heads, d), (row if shared else rng.randint(1, 40), head, dim),
                        4 * rng.randint(0, 60))

        out, k = layout(hq), layout(hkv)
        far = dense((rows, hq, d), FAR), dense((rows, hkv, d), 2 * FAR), dense((2,), 3 * FAR, I32)
        out_at, out_bytes = bytes_of(out)
        overlap = len(set(out_at)) < len(out_at) or bool(out_bytes & bytes_of(k)[1])
        said = attention(far[0], k, far[1], out, far[2])
        assert said or not overlap
        if shared and not overlap:
            seen[1] += 1
            # (within a row, k and out may interleave, which counts as overlapping)
            lo = [(t.data - BASE) % (4 * row) for t in (out, k)]
            ends = [o + 4 * (1 + (t.shape[1] - 1) * t.stride[1] + (t.shape[2] - 1) * t.stride[2])
                    for o, t in zip(lo, (out, k))]
            if max(ends) <= 4 * row and (ends[0] <= lo[1] or ends[1] <= lo[0]):
                assert not said
        seen[0] += overlap
    assert min(seen) > 100


def scan(**change):
    t = dict(x=dense((30, 4, 8)), dt=dense((30, 4), FAR), A=dense((4,), 2 * FAR), B=dense((30, 2, 16), 3 * FAR),
             C=dense((30, 2, 16), 4 * FAR), starts=dense((3,), 5 * FAR, I32), D=dense((4,), 6 * FAR),
             z=dense((30, 4, 8), 7 * FAR), bias=dense((4,), 8 * FAR), initial=dense((2, 4, 8, 16), 9 * FAR),
             states=dense((2, 4, 8, 16), 10 * FAR), out=dense((30, 4, 8), 11 * FAR))
    t.update(change)
    args = [None if v is None else ctypes.pointer(v) for v in t.values()]
    return refused(lambda: _abi.lib().lq_prompt_scan(*args, 1, 0.0, 1.0, 1 << 30, 1 << 28, None))


def test_scan_over_its_own_inputs():
    state = (2, 4, 8, 16)
    assert not scan() and not scan(states=None) and not scan(initial=None)
    assert not scan(states=dense(state, 9 * FAR)), "states in place"
    assert scan(states=dense(state, 9 * FAR + 4)) and scan(states=fake(state, (512, 128, 1, 8), 9 * FAR))
    assert scan(states=dense(state, 9 * FAR, BF)), "in place in another type"
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 8, 11):
        assert scan(states=dense(state, i * FAR)), i
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10):
        assert scan(out=dense((30, 4, 8), i * FAR)), i
    assert scan(states=fake(state, (0, 128, 16, 1), 10 * FAR)) and scan(out=fake((30, 4, 8), (32, 0, 1), 11 * FAR))
    # both halves of one tensor
    assert not scan(initial=fake(state, (1024, 128, 16, 1), 9 * FAR),
                    states=fake(state, (1024, 128, 16, 1), 9 * FAR + 4 * 512))
