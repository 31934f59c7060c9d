"""Refusals of the beam-decoding operators, before any GPU call (made-up addresses, never read), and
of their Python entry points."""
import ctypes

import pytest
import torch

from layer_quant_amd import _abi
from layer_quant_amd import beam_decode as bd
from layer_quant_amd import int4_8b_attention as ia


def fake(shape, dtype, stride=None, data=0x10000):
    t = _abi.LQTensor()
    t.data, t.dtype, t.ndim = data, _abi.DTYPE_CODES[dtype], len(shape)
    step = 1
    for i in reversed(range(len(shape))):
        t.shape[i], t.stride[i] = shape[i], step
        step *= max(shape[i], 1)
    for i, s in enumerate(stride or ()):
        t.stride[i] = s
    return t


F32, I64, U8, BF16 = torch.float32, torch.int64, torch.uint8, torch.bfloat16


def select(P=2, N=4, V=100, num=4, pad=0, slots=0, ws=None, wsb=1 << 30, **over):
    t = dict(logits=fake((P, N, V), BF16), scores=fake((P, N), F32), finished=fake((P, N), U8),
             s=fake((P, num), F32), b=fake((P, num), I64), t=fake((P, num), I64))
    t.update(over)
    return _abi.lib().lq_beam_select(*(None if x is None else ctypes.byref(x) for x in t.values()),
                                     pad, slots, 0x1000 if ws is None else ws, wsb, None)


@pytest.mark.parametrize("kw,code", [
    (dict(logits=fake((2, 400), BF16)), -1), (dict(logits=fake((2, 4, 100), I64)), -1),
    (dict(logits=None), -1), (dict(scores=fake((2, 3), F32)), -1), (dict(scores=fake((2, 4), BF16)), -1),
    (dict(finished=fake((4, 2), U8)), -1), (dict(finished=fake((2, 4), I64)), -1),
    (dict(b=fake((2, 3), I64)), -1), (dict(t=fake((2, 4), F32)), -1), (dict(s=fake((1, 4), F32)), -1),
    (dict(N=65, num=4), -2), (dict(num=65), -2), (dict(V=(1 << 24) + 1), -2), (dict(P=65536), -2),
    (dict(V=1, num=5), -1), (dict(num=3, slots=1), -1), (dict(pad=100), -1), (dict(pad=-1), -1),
    (dict(wsb=8), -3), (dict(ws=0x1004), -3), (dict(logits=fake((2, 4, 100), BF16, data=None)), -1)])
def test_select_refuses(kw, code):
    assert select(**kw) == code, _abi.last_error()
    assert _abi.last_error()


def test_select_of_nothing():
    assert select(P=0) == 0
    assert select(num=0) == 0
    lib = _abi.lib()
    assert lib.lq_beam_select_workspace(0, 4, 100, 4) == 0
    assert lib.lq_beam_select_workspace(1, 4, 100, 4) > 0


def reorder(tensors, beams, rows=None):
    table = (_abi.LQTensor * max(len(tensors), 1))(*tensors)
    live = None if rows is None else (ctypes.c_int64 * len(rows))(*rows)
    return _abi.lib().lq_reorder_beams(table, live, len(tensors), ctypes.byref(beams), None)


def test_reorder_refuses():
    b = fake((2, 4), I64)
    ok = fake((8, 3, 5, 16), U8)
    assert reorder([], b) == 0
    assert reorder([ok], fake((2, 4), torch.int32)) == -1
    assert reorder([ok], fake((8,), I64)) == -1
    assert reorder([ok], fake((1, 65), I64)) == -2
    assert reorder([fake((7, 3), U8)], b) == -1
    assert reorder([ok], b, [6]) == -1
    assert reorder([ok], b, [-2]) == -1
    assert reorder([fake((8, 3), U8)], b, [1]) == -1
    assert reorder([fake((8, 3, 5), U8, (0, 5, 1))], b) == -1
    assert reorder([fake((8, 3, 5), U8, (5, 0, 1))], b) == -1
    assert reorder([ok, fake((8, 3, 5, 16), U8)], b) == -1 and "twice" in _abi.last_error()
    assert reorder([fake((8, 1 << 31, 16), U8, (1 << 40, 32, 2))], b) == -2
    assert reorder([fake((8, 3), U8, data=None)], b) == -1
    assert reorder([ok], fake((8, 1), I64)) == 0  # one beam per prompt: nothing moves
    assert reorder([ok], b, [0]) == 0
    assert reorder([fake((8, 0, 5), U8, data=None)], b) == 0
    assert _abi.lib().lq_reorder_beams(None, None, 1, ctypes.byref(b), None) == -1
    assert reorder([fake((8,), U8, data=0x10000 + 64 * i) for i in range(513)], b) == -2


def test_reorder_refuses_its_beams():
    """Entries that a workgroup reads while another moves them: the tensor itself and any overlap."""
    b = fake((2, 4), I64, data=0x20000)
    for data in (0x20000, 0x20000 - 8 * 15, 0x20000 + 63):
        assert reorder([fake((8, 16), U8, data=data)], b) == -1
        assert "overlaps the beams" in _abi.last_error()
    assert reorder([fake((8,), I64, data=0x20000)], fake((2, 4), I64, (1, 2), data=0x20000)) == -1


def shared(B=6, P=2, hq=8, hkv=2, d=128, g=32, cap=100, ocap=20, lp=50, S=60, nrep=4, mask=None,
           token=True, ws=0x10000, wsb=1 << 40, **over):
    new = fake((B, hkv, 1, d), BF16) if token else None
    t = dict(q=fake((B, hq, 1, d), BF16), k=new, v=new,
             pkp=fake((P, hkv, cap, d // 2), U8), pvp=fake((P, hkv, cap, d // 2), U8),
             pks=fake((P, hkv, cap, d // g), F32), pvs=fake((P, hkv, cap, d // g), F32),
             kp=fake((B, hkv, ocap, d // 2), U8), vp=fake((B, hkv, ocap, d // 2), U8),
             ks=fake((B, hkv, ocap, d // g), F32), vs=fake((B, hkv, ocap, d // g), F32),
             mask=mask, out=fake((B, hq, d), BF16))
    t.update(over)
    return _abi.lib().lq_int4_shared_decode_attention(
        *(None if x is None else ctypes.byref(x) for x in t.values()), lp, S, nrep, g, ws, wsb, None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(q=fake((6, 8, 2, 128), BF16)), -1), (dict(q=fake((6, 8, 1, 128), I64)), -1),
    (dict(B=7), -1), (dict(P=0), -1), (dict(nrep=3), -1), (dict(nrep=0), -1), (dict(hkv=3), -1),
    (dict(d=120), -1), (dict(d=640, g=64), -2), (dict(lp=101, S=102), -1), (dict(lp=-1), -1),
    (dict(S=49), -1), (dict(S=71), -1), (dict(S=50), -1), (dict(lp=0, S=0, token=False), -1),
    (dict(k=None), -1), (dict(v=fake((6, 2, 2, 128), BF16)), -1), (dict(k=fake((6, 3, 1, 128), BF16)), -1),
    (dict(pkp=fake((2, 2, 100, 63), U8)), -1), (dict(pvp=fake((2, 2, 90, 64), U8)), -1),
    (dict(pvs=fake((2, 2, 100, 2), F32)), -1), (dict(kp=fake((5, 2, 20, 64), U8)), -1),
    (dict(ks=fake((6, 2, 20, 4), BF16)), -1), (dict(vs=None), -1),
    (dict(mask=fake((6, 60), F32)), -1), (dict(mask=fake((2, 60), I64)), -1),
    (dict(mask=fake((6, 1, 1, 60), BF16)), -1), (dict(mask=fake((2, 1, 1, 60), F32)), -1),
    (dict(out=fake((6, 8, 64), BF16)), -1), (dict(wsb=16), -3), (dict(ws=0x10010), -3), (dict(ws=0), -3)])
def test_shared_attention_refuses(kw, code):
    assert shared(**kw) == code, _abi.last_error()
    assert _abi.last_error()


def test_shared_attention_of_nothing():
    lib = _abi.lib()
    assert lib.lq_int4_shared_decode_attention_workspace(0, 1, 8, 2, 128, 10, 20, 32) == 0
    assert lib.lq_int4_shared_decode_attention_workspace(1, 4, 8, 2, 128, 20, 10, 32) == 0
    assert lib.lq_int4_shared_decode_attention_workspace(1, 4, 8, 2, 128, 5000, 5010, 32) > 0
    empty = dict(B=0, P=2, token=False)
    assert shared(**empty) == 0


def test_entry_points_refuse():
    logits, scores = torch.zeros(8, 10), torch.zeros(2, 4)
    beams = torch.zeros(2, 4, dtype=torch.int64)
    for bad in (dict(logits=torch.zeros(7, 10)), dict(logits=torch.zeros(4, 2, 10)),
                dict(logits=torch.zeros(10)), dict(scores=torch.zeros(8)), dict(num=-1),
                dict(finished=torch.zeros(2, 4)), dict(finished=torch.zeros(4, 2, dtype=torch.bool))):
        with pytest.raises(ValueError):
            bd.beam_select(**{**dict(logits=logits, scores=scores), **bad})
    with pytest.raises(RuntimeError, match="GPU only"):
        bd.beam_select(logits, scores)
    with pytest.raises(RuntimeError, match="GPU only"):
        bd.reorder_beams([logits], beams)
    with pytest.raises(ValueError, match="row counts"):
        bd.reorder_beams([logits], beams, [1, 2])
    cache = ia._allocate_layer_cache(8, 2, 16, 128, 4, torch.device("cpu"))
    q = torch.zeros(8, 8, 1, 128)
    with pytest.raises(ValueError, match="no shared prefix"):
        ia.shared_prefix_decode_attention(q, cache, 5, 4, 32)
    cache.prefix = ia._allocate_layer_cache(2, 2, 16, 128, 4, torch.device("cpu"))
    with pytest.raises(ValueError, match="q_len=1"):
        ia.shared_prefix_decode_attention(q.transpose(1, 2), cache, 5, 4, 32)
    with pytest.raises(ValueError, match="both or neither"):
        ia.shared_prefix_decode_attention(q, cache, 5, 4, 32, None, q)
    with pytest.raises(ValueError, match="2D or 4D"):
        ia.shared_prefix_decode_attention(q, cache, 5, 4, 32, torch.zeros(8))
    with pytest.raises(RuntimeError, match="GPU only"):
        ia.shared_prefix_decode_attention(q, cache, 5, 4, 32)


def test_host_binding_declines_tensors_off_the_gpu():
    host = _abi.host_binding()
    t = torch.zeros(2, 2, 2, 16)
    assert host.int4_shared_decode_attention(*[t] * 11, None, t, 1, 2, 1, 32, _abi._scratch.get) is None
    assert host.beam_select(*[t] * 6, 0, False, _abi._scratch.get) is None
    assert host.reorder_beams([t], None, t) is None
    assert host.reorder_beams([t], [None, None], t) is None
    with pytest.raises(TypeError):
        host.reorder_beams([t], None)


def test_growth_keeps_the_prefix():
    holder = type("Cache", (), {})()
    cpu = torch.device("cpu")
    own = ia._ensure_layer_cache(holder, 3, 4, 2, 5, 128, 32, cpu)
    own.prefix = prefix = ia._allocate_layer_cache(2, 2, 16, 128, 4, cpu)
    grown = ia._ensure_layer_cache(holder, 3, 4, 2, 40, 128, 32, cpu)
    assert grown is not own and grown.prefix is prefix
