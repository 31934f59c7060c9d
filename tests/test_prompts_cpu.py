"""The prompt operators without a GPU: what the C ABI and the Python functions refuse (made-up
addresses, never read), and the reference against the recurrence's closed form."""
import ctypes

import pytest
import torch

import prompt_reference as ref
from layer_quant_amd import _abi, prompts

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I32, I64 = torch.int32, torch.int64


def fake(shape, dtype, stride=None, data=0x1000):
    t = _abi.LQTensor()
    t.data, t.dtype, t.ndim = data, _abi.DTYPE_CODES[dtype], len(shape)
    step = 1
    for i in reversed(range(len(shape))):
        t.shape[i] = shape[i]
        t.stride[i] = step if stride is None else stride[i]
        step *= shape[i]
    return ctypes.pointer(t)


def attention(q=((9, 8, 128), BF), k=((9, 2, 128), BF), v=None, starts=((3,), I32), out=None, scale=0.1):
    v = k if v is None else v
    out = q if out is None else out
    return _abi.lib().lq_prompt_attention(fake(*q), fake(*k), fake(*v), starts and fake(*starts),
                                          fake(*out), scale, None)


@pytest.mark.parametrize("rc,change", [
    (-1, dict(q=((9, 8, 128), I32))),
    (-1, dict(q=((1, 9, 8, 128), BF))),
    (-1, dict(starts=None)),
    (-1, dict(k=((9, 2, 128), F16))),
    (-1, dict(k=((8, 2, 128), BF))),
    (-1, dict(k=((9, 3, 128), BF))),
    (-1, dict(k=((9, 0, 128), BF))),
    (-1, dict(k=((9, 2, 64), BF))),
    (-1, dict(v=((9, 4, 128), BF))),
    (-1, dict(out=((9, 8, 128), F32))),
    (-1, dict(out=((8, 8, 128), BF))),
    (-1, dict(starts=((3,), F32))),
    (-1, dict(starts=((0,), I32))),
    (-1, dict(starts=((3, 1), I32))),
    (-1, dict(starts=((3,), I32, (2,)))),
    (-2, dict(q=((9, 8, 264), BF), k=((9, 2, 264), BF))),
    (-2, dict(q=((9, 8, 0), BF), k=((9, 2, 0), BF))),
    (-1, dict(scale=float("nan"))),
    (-1, dict(scale=float("inf"))),
    (-2, dict(q=((1 << 31, 1, 8), BF), k=((1 << 31, 1, 8), BF))),
    (-2, dict(q=((1 << 29, 8, 8), BF), k=((1 << 29, 2, 8), BF))),
    (-2, dict(starts=((1 << 25,), I32)))])
def test_attention_refusals(rc, change):
    assert attention(**change) == rc, _abi.last_error()


def test_attention_of_nothing():
    assert attention(q=((0, 8, 128), BF), k=((0, 2, 128), BF)) == 0
    assert attention(q=((0, 5, 8, 128), BF), k=((0, 5, 2, 128), BF), starts=None) == 0
    assert attention(q=((2, 0, 8, 128), BF), k=((2, 0, 2, 128), BF), starts=None) == 0


def scan(ws=0x10000, nbytes=None, softplus=1, lo=0.0, hi=float("inf"), **change):
    a = dict(x=((600, 8, 64), BF), dt=((600, 8), BF), A=((8,), F32), B=((600, 2, 128), BF),
             C=((600, 2, 128), BF), starts=((3,), I32), D=None, z=None, bias=None, initial=None,
             states=((2, 8, 64, 128), F32), out=((600, 8, 64), BF))
    a.update(change)
    t = {k: None if v is None else fake(*v) for k, v in a.items()}
    need = _abi.lib().lq_prompt_scan_workspace(3, 2, a["x"][0][0], 1, 8, 64, 128)
    return _abi.lib().lq_prompt_scan(*(t[k] for k in a), softplus, lo, hi, ws,
                                     need if nbytes is None else nbytes, None)


@pytest.mark.parametrize("rc,change", [
    (-1, dict(x=((600, 8, 64), I32))),
    (-1, dict(starts=None)),
    (-1, dict(dt=((600, 4), BF))),
    (-1, dict(dt=((600, 8, 64), BF))),
    (-1, dict(B=((600, 2, 128), F32))),
    (-1, dict(B=((599, 2, 128), BF), C=((599, 2, 128), BF))),
    (-1, dict(C=((600, 4, 128), BF))),
    (-1, dict(B=((600, 3, 128), BF), C=((600, 3, 128), BF))),
    (-1, dict(A=((4,), F32))),
    (-1, dict(A=((8, 64), F32))),
    (-1, dict(D=((4,), F32))),
    (-1, dict(bias=((16,), F32))),
    (-1, dict(z=((600, 8, 32), BF))),
    (-1, dict(states=((3, 8, 64, 128), F32))),
    (-1, dict(states=((2, 8, 128, 64), F32))),
    (-1, dict(initial=((1, 8, 64, 128), F32))),
    (-1, dict(out=((600, 8, 32), BF))),
    (-1, dict(lo=1.0, hi=0.5)),
    (-1, dict(lo=float("nan"))),
    (-2, dict(B=((600, 2, 257), BF), C=((600, 2, 257), BF), states=((2, 8, 64, 257), F32))),
    (-2, dict(starts=((70001,), I32), states=((70000, 8, 64, 128), F32))),
    (-3, dict(ws=None)),
    (-3, dict(nbytes=16)),
    (-3, dict(ws=0x10010))])
def test_scan_refusals(rc, change):
    assert scan(**change) == rc, _abi.last_error()


def test_scan_of_nothing():
    none = dict(x=((0, 8, 64), BF), dt=((0, 8), BF), B=((0, 2, 128), BF), C=((0, 2, 128), BF),
                out=((0, 8, 64), BF), starts=((1,), I32), states=((0, 8, 64, 128), F32))
    assert scan(**none) == 0
    lib = _abi.lib()
    f32, bf = _abi.DTYPE_CODES[F32], _abi.DTYPE_CODES[BF]
    assert lib.lq_prompt_scan_workspace(bf, 1, 0, 1, 8, 64, 128) == 0
    assert lib.lq_prompt_scan_workspace(bf, 0, 5, 0, 8, 64, 128) == 0
    # prompts of one segment carry nothing
    assert lib.lq_prompt_scan_workspace(f32, 4, 200, 0, 64, 64, 128) == 0
    assert lib.lq_prompt_scan_workspace(f32, 1, 16384, 1, 128, 64, 128) > 0
    assert lib.lq_prompt_scan_workspace(bf, 4, 200, 0, 8, 64, 128) == 4 * 200 * 8 * 16


def scores(logits=((4, 100), BF), tokens=((4,), I64), lp=((4,), F32), entropy=((4,), F32),
           tl=((4, 3), F32), tt=((4, 3), I64), ws=0x10000, nbytes=1 << 20):
    t = [None if v is None else fake(*v) for v in (logits, tokens, lp, entropy, tl, tt)]
    return _abi.lib().lq_token_logprobs(*t, ws, nbytes, None)


@pytest.mark.parametrize("rc,change", [
    (-1, dict(logits=((4, 100), I32))),
    (-1, dict(logits=((100,), BF))),
    (-1, dict(logits=((2, 2, 5, 5), BF))),
    (-1, dict(tokens=((4,), I32))),
    (-1, dict(tokens=((5,), I64))),
    (-1, dict(logits=((2, 2, 100), BF))),
    (-1, dict(lp=((4,), BF))),
    (-1, dict(lp=((5,), F32))),
    (-1, dict(lp=((4,), F32, (2,)))),
    (-1, dict(entropy=((3,), F32))),
    (-1, dict(tl=None)),
    (-1, dict(tl=((4, 2), F32))),
    (-1, dict(tl=((4, 3), F32, (4, 1)))),
    (-1, dict(logits=((4, 2), BF))),
    (-1, dict(logits=((4, 0), BF))),
    (-2, dict(tl=((4, 33), F32), tt=((4, 33), I64))),
    (-2, dict(logits=((1 << 24, 100), BF), tokens=((1 << 24,), I64), lp=((1 << 24,), F32),
              entropy=((1 << 24,), F32), tl=None, tt=None)),
    (-3, dict(logits=((4, 40000), BF), ws=None)),
    (-3, dict(logits=((4, 40000), BF), nbytes=8)),
    (-3, dict(logits=((4, 40000), BF), ws=0x10010))])
def test_scores_refusals(rc, change):
    assert scores(**change) == rc, _abi.last_error()


def test_python_refusals():
    t = torch.zeros(6, 4, 16)
    starts = torch.tensor([0, 6])
    with pytest.raises(ValueError, match="without starts"):
        prompts.prompt_attention(t, t, t)
    with pytest.raises(ValueError, match="with starts"):
        prompts.prompt_attention(t[None], t[None], t[None], starts)
    with pytest.raises(ValueError, match="int32 or int64"):
        prompts.prompt_attention(t, t, t, starts.float())
    with pytest.raises(ValueError, match="int32 or int64"):
        prompts.prompt_attention(t, t, t, starts[None])
    with pytest.raises(RuntimeError, match="GPU only"):
        prompts.prompt_attention(t, t, t, starts)
    with pytest.raises(RuntimeError, match="no backward"):
        prompts.prompt_attention(t.requires_grad_(), t, t, starts)
    t = t.detach()
    with pytest.raises(ValueError, match="rank"):
        prompts.prompt_scan(t, t[..., 0], t[0, :, 0], t[0], t[0], starts)
    with pytest.raises(RuntimeError, match="GPU only"):
        prompts.prompt_scan(t, t[..., 0], t[0, :, 0], t, t, starts)
    with pytest.raises(RuntimeError, match="no backward"):
        prompts.prompt_scan(t, t[..., 0], t[0, :, 0].requires_grad_(), t, t, starts)
    with pytest.raises(ValueError, match="a token for each row"):
        prompts.token_logprobs(t[0], torch.zeros(3, dtype=I64))
    with pytest.raises(ValueError, match="negative"):
        prompts.token_logprobs(t[0], torch.zeros(4, dtype=I64), -1)
    with pytest.raises(RuntimeError, match="GPU only"):
        prompts.token_logprobs(t[0], torch.zeros(4, dtype=I64))


def test_binding_declines_tensors_off_the_gpu():
    host = _abi.host_binding()
    t = torch.zeros(2, 2, 2, 2)
    assert host.prompt_attention(t, t, t, None, t, 1.0) is None
    assert host.prompt_scan(*[t] * 5, *[None] * 6, t, True, 0.0, 1.0, _abi._scratch.get) is None
    assert host.token_logprobs(t[0], t[0, 0], *[None] * 4, _abi._scratch.get) is None


def test_reference_scan_is_attention_without_a_softmax():
    """y_t = sum_s exp(A (c_t - c_s)) dt_s (C_t . B_s) x_s, c the steps' running sum."""
    gen = torch.Generator().manual_seed(0)
    x, B, C = (torch.randn(7, 2, n, generator=gen) for n in (3, 4, 4))
    dt, A = torch.rand(7, 2, generator=gen), -torch.rand(2, generator=gen)
    y = ref.scan(x, dt, A, B, C, [0, 7])[0]
    c = dt.double().cumsum(0)
    for h in range(2):
        w = torch.exp(A[h].double() * (c[:, None, h] - c[None, :, h])).tril() * dt[None, :, h].double()
        w = w * (C[:, h].double() @ B[:, h].double().T)
        assert torch.allclose(y[:, h], w @ x[:, h].double(), atol=1e-12)
