"""Decode attention over a shared prefix against a softmax in 64 bits.

Tolerance of an output value: the rounding of the output's type (half a step, eps / 2 of |out|), and of
the sums' weights and values against A = sum_j w_j |v_j| / sum_j w_j:
  * a score is a sum of head_dim exact products with fp32 additions and scalings, off by at most
    (head_dim + 16) * 2^-24 * sum_d |q_d k_d| log2(e)/sqrt(D), which its weight has relatively (ln 2 of
    it); both the sum of the weights and the weighted values have it: 2 ln 2 delta;
  * the matrix-core kernel rounds weight, value scale and their product to fp16 for bf16 outputs:
    3 * 2^-11; for other outputs it keeps 2^-20 of them;
  * fp16 has steps of 2^-24 below 2^-14: a weighted scale P' = w vs 2^(7-e), 2^e at most twice the
    largest value scale, is off by half a step at most, which with levels of at most 8 is
    8 * 2^-25 * 2^(e-7) <= 2^-28 times the largest value scale per key, whatever the weight (where one
    key has all the weight and level 0, the others' weights can be far below that). A weight below
    2^-126 of the largest is 0 in fp32: 8 * 2^-126 of the largest scale per key;
  * fp32 sums over the keys of a split and the merge: 2^-24 per addition in a row, fewer than 2^8 of
    them in the matrix-core kernel's lanes per rescale step, linear in the keys else: keys * 2^-23.
"""
import math
import threading

import pytest
import torch

from helpers import require_env
from layer_quant_amd import _abi
from layer_quant_amd import int4_8b_attention as ia
from oracle import int4_kv as oik

pytestmark = pytest.mark.gpu
LOG2E = 1.4426950408889634
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def cache_of(gpu, rows, hkv, length, cap, d, g, seed, scale=1.0, fill=0):
    """A filled INT4 cache; what lies behind `length` is `fill` (bytes) and NaN (scales)."""
    gen = torch.Generator(device=gpu).manual_seed(seed)
    c = ia.Int4KVLayerCache(
        torch.full((rows, hkv, cap, d // 2), fill, dtype=torch.uint8, device=gpu),
        torch.full((rows, hkv, cap, d // 2), fill, dtype=torch.uint8, device=gpu),
        torch.full((rows, hkv, cap, d // g), torch.nan, device=gpu),
        torch.full((rows, hkv, cap, d // g), torch.nan, device=gpu))
    if length:
        k = torch.randn(rows, hkv, length, d, device=gpu, generator=gen)
        k *= 1 + 4 * (torch.rand(d, device=gpu, generator=gen) < 0.05)
        v = scale * torch.randn(rows, hkv, length, d, device=gpu, generator=gen)
        _abi.int4_pack_kv_pair(k, v, c.k_packed, c.v_packed, c.k_scale, c.v_scale,
                               torch.arange(length, device=gpu), g)
    c.length = length
    return c


def pack_token(x, packed, scale, row, g):
    """The token's levels and scales: absmax * fl(1/7), levels by IEEE quotients, half to even."""
    xg = x.float().reshape(*x.shape[:-1], -1, g)
    sc = (xg.abs().amax(-1, keepdim=True) * torch.tensor(1 / 7, device=x.device)).clamp_min(1e-8)
    n = (xg / sc).round().clamp(-8, 7).to(torch.int32).reshape(x.shape) & 15
    packed[:, :, row:row + 1] = (n[..., 0::2] | n[..., 1::2] << 4).to(torch.uint8)
    scale[:, :, row:row + 1] = sc[..., 0]


def reference(q, cache, seq_len, nrep, g, bias=None):
    """(out, A, delta, vs) in 64 bits: out [B, Hq, D], the weighted |v|, the scores' error unit, and the
    largest value scale (a group's largest level is 7)."""
    pre, lp = cache.prefix, cache.prefix.length
    B, hq, d = q.shape[0], q.shape[1], q.shape[-1]
    N = B // pre.k_packed.shape[0]
    q = q.reshape(B, hq, d).double()
    outs, mags, deltas, top = [], [], [], 0.0
    for b in range(B):
        rows = [(pre, b // N, lp), (cache, b, seq_len - lp)]
        k, v = (torch.cat([oik.dequantize(getattr(c, n + "_packed")[i:i + 1, :, :m].cpu(),
                                          getattr(c, n + "_scale")[i:i + 1, :, :m].cpu(), g)[0].double()
                           for c, i, m in rows], 1).to(q.device) for n in "kv")
        k, v = k.repeat_interleave(nrep, 0), v.repeat_interleave(nrep, 0)
        s = (k @ q[b, :, :, None])[..., 0] * (LOG2E / math.sqrt(d))
        mag = (k.abs() @ q[b, :, :, None].abs())[..., 0] * (LOG2E / math.sqrt(d))
        if bias is not None:
            gone = bias[b] == -math.inf
            v = torch.where(gone[None, :, None], 0.0, v)
            s = torch.where(gone, -math.inf, s + bias[b])
            mag = torch.where(gone, 0.0, mag)
        top = max(top, v.abs().max().item() / 7)
        w = torch.exp2(s - s.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        outs.append((w[:, None] @ v)[:, 0])
        mags.append((w[:, None] @ v.abs())[:, 0])
        deltas.append(mag.amax(-1, keepdim=True))
    return torch.stack(outs), torch.stack(mags), torch.stack(deltas), top


def fast_expected(dtype, d, g):
    return dtype in (BF16, FP16) and d == 128 and g in (32, 64, 128)


def assert_near(out, ref, dtype, d, keys, fast, what=""):
    want, mag, delta, top = ref
    out = out.double()
    empty = torch.isnan(want)
    assert torch.equal(torch.isnan(out), empty), what
    rel = 2 * math.log(2) * (d + 16) * 2.0 ** -24 * delta + keys * 2.0 ** -23
    if fast:
        rel = rel + (3 * 2.0 ** -11 if dtype == BF16 else 2.0 ** -20)
    bound = torch.finfo(dtype).eps / 2 * want.abs() + rel * mag
    bound = bound + keys * top * (2.0 ** -28 if fast else 2.0 ** -123) + 1e-300
    if dtype == FP16:
        bound = bound + 2.0 ** -25  # half a step of its subnormal values
    worst = ((out - want).abs() / bound)[~empty]
    if worst.numel():
        print(f"[close] {what}: max err/bound {worst.max().item():.3g}")
        assert worst.max().item() <= 1.0, (what, worst.max().item())


def run(gpu, P, N, hkv, nrep, lp, lo, d, g, dtype, seed=0, mask=None, token=True, q=None, scale=1.0):
    B = P * N
    gen = torch.Generator(device=gpu).manual_seed(seed + 1)
    pre = cache_of(gpu, P, hkv, lp, max(lp, 1) + 3, d, g, seed + 2, scale)
    own = cache_of(gpu, B, hkv, lo, max(lo, 1) + 2, d, g, seed + 3, scale)
    own.prefix = pre
    if q is None:
        q = 1.5 * torch.randn(B, hkv * nrep, 1, d, device=gpu, generator=gen)
        q = q.to(dtype)
    k = v = None
    if token and lo > 0:
        k = torch.randn(B, hkv, 1, d, device=gpu, generator=gen).to(dtype)
        v = (scale * torch.randn(B, hkv, 1, d, device=gpu, generator=gen)).to(dtype)
    S = lp + lo
    fast = fast_expected(dtype, d, g)
    before = [t.clone() for t in (own.k_packed, own.v_packed, own.k_scale, own.v_scale)]
    pre_before = [t.clone() for t in (pre.k_packed, pre.v_packed, pre.k_scale, pre.v_scale)]
    with require_env("LQ_ATTN_REQUIRE_FAST", fast):
        out = ia.shared_prefix_decode_attention(q, own, S, nrep, g, mask, k, v)
    if k is not None:
        pack_token(k, before[0], before[2], lo - 1, g)
        pack_token(v, before[1], before[3], lo - 1, g)
    # the caches: the token's row, everything else as it was
    for t, w in zip((own.k_packed, own.v_packed, own.k_scale, own.v_scale), before):
        assert torch.equal(t.view(torch.uint8), w.view(torch.uint8))
    for t, w in zip((pre.k_packed, pre.v_packed, pre.k_scale, pre.v_scale), pre_before):
        assert torch.equal(t.view(torch.uint8), w.view(torch.uint8))
    bias = None
    if mask is not None:
        if mask.dim() == 2:
            keep = mask[:, -S:] != 0
            bias = torch.where(keep, 0.0, -math.inf).double()
        else:
            bias = mask.reshape(B, -1).double() if mask.dtype != torch.bool else \
                torch.where(mask.reshape(B, -1), 0.0, -math.inf).double()
        short = S - bias.shape[1]
        if short > 0:
            bias = torch.nn.functional.pad(bias, (0, short), value=-math.inf)
        bias = bias[:, :S]
    ref = reference(q, own, S, nrep, g, bias)
    assert_near(out, ref, dtype, d, S, fast, f"P{P} N{N} {hkv}x{nrep} lp{lp} lo{lo} d{d} g{g} {dtype}")
    return out, own


@pytest.mark.parametrize("g", [32, 64, 128])
@pytest.mark.parametrize("P,N,hkv,nrep,lp,lo", [
    (1, 1, 1, 1, 1, 1), (1, 4, 8, 4, 777, 18), (2, 3, 2, 4, 31, 33), (1, 5, 2, 3, 32, 1),
    (3, 1, 1, 16, 65, 64), (1, 8, 1, 8, 1000, 0), (2, 2, 2, 2, 0, 100), (1, 33, 1, 1, 129, 2),
    (1, 16, 2, 4, 2000, 40), (1, 64, 1, 4, 515, 7), (2, 7, 1, 5, 4097, 130), (1, 2, 1, 32, 300, 31)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_shapes(gpu, P, N, hkv, nrep, lp, lo, g, dtype):
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, seed=lp + lo)


@pytest.mark.parametrize("lo", [1, 40, 64, 65, 100, 129, 250, 300])
@pytest.mark.parametrize("masked", [False, True])
def test_many_own_rows(gpu, lo, masked):
    """Own units behind a prefix that fills the GPU: one, two or four waves each, odd numbers of them."""
    P, N, hkv, nrep, lp, g = 5, 13, 8, 4, 2500, 32
    mask = None
    if masked:
        gen = torch.Generator(device=gpu).manual_seed(lo)
        mask = (torch.rand(P * N, lp + lo, device=gpu, generator=gen) < 0.8).long()
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, BF16, lo, mask)


@pytest.mark.parametrize("mask", ["none", "keep", "bias"])
@pytest.mark.parametrize("nrep,lp", [(1, 4300), (17, 2300), (17, 2047)])
def test_long_units(gpu, nrep, lp, mask):
    """More prefix units than places: every wave takes 16 to 34 tiles, masks among them in stretches."""
    P, N, hkv, lo, g = 8, 1, 64, 40, 64
    gen = torch.Generator(device=gpu).manual_seed(lp)
    keep = (torch.rand(P * N, lp + lo, device=gpu, generator=gen) < 0.7).long()
    keep[1, 100:2000] = 0
    keep[2, :lp] = 0
    m = {"none": None, "keep": keep}.get(mask)
    if mask == "bias":
        m = torch.where(keep != 0, torch.randn(keep.shape, device=gpu, generator=gen), -torch.inf)
        m = m[:, None, None, :]
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, BF16, lp, m)


@pytest.mark.parametrize("d,g,dtype", [(64, 32, BF16), (128, 32, FP32), (128, 16, BF16), (96, 96, FP16),
                                       (512, 64, BF16), (80, 2, FP32)])
def test_general_kernel(gpu, d, g, dtype):
    run(gpu, 2, 3, 2, 2, 150, 70, d, g, dtype, seed=d)
    run(gpu, 1, 2, 1, 1, 0, 3, d, g, dtype, seed=d)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("lp,lo", [(100, 30), (1500, 3), (5, 700)])
def test_masks(gpu, dtype, lp, lo):
    """Padded prompts, rows without a key, short masks, biases of every kind, -inf and the lowest."""
    P, N, hkv, nrep, g = 2, 3, 2, 4, 64
    B, S = P * N, lp + lo
    keep = torch.ones(B, S + 2, dtype=torch.int64, device=gpu)
    keep[:N, 2:2 + lp // 2] = 0
    keep[N, 2:] = 0
    keep[N + 1, 2:-1] = 0
    keep[N + 2, -lo:] = 0
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 1, keep)
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 1, keep[:, 2:])
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 1, keep.to(torch.uint8))
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 1, (keep != 0)[:, None, None, 2:])
    torch.manual_seed(lp)
    bias = torch.randn(B, 1, 1, S, device=gpu)
    bias[:, :, :, ::3] = -torch.inf
    bias[0] = torch.finfo(torch.float32).min
    bias[1, :, :, : S // 2] = torch.finfo(torch.float32).min
    bias[2, :, :, :lp] = -torch.inf
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 2, bias)
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 2, bias[..., :S - 2], token=False)
    run(gpu, P, N, hkv, nrep, lp, lo, 128, g, dtype, 2, bias[..., :lp], token=False)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_masked_rows_may_hold_anything(gpu, dtype):
    """Infinities and NaN in cache rows that no row attends to, in whole tiles and inside them."""
    P, N, hkv, nrep, lp, lo, g = 2, 2, 1, 4, 200, 40, 32
    pre = cache_of(gpu, P, hkv, lp, lp + 8, 128, g, 1)
    own = cache_of(gpu, P * N, hkv, lo, lo + 8, 128, g, 2)
    own.prefix = pre
    keep = torch.ones(P * N, lp + lo, dtype=torch.int64, device=gpu)
    for c, at in ((pre, 0), (own, lp)):
        for j in (0, 5, 17, 31, 33):
            keep[:, at + j] = 0
            c.k_scale[:, :, j], c.v_scale[:, :, j] = torch.nan, torch.inf
    pre.v_scale[:, :, 64:100] = torch.nan
    keep[:, 64:100] = 0
    q = torch.randn(P * N, hkv * nrep, 1, 128, device=gpu).to(dtype)
    out = ia.shared_prefix_decode_attention(q, own, lp + lo, nrep, g, keep)
    bias = torch.where(keep != 0, 0.0, -math.inf).double()
    for c in (pre, own):
        c.k_scale.nan_to_num_(0, 0, 0)
        c.v_scale.nan_to_num_(0, 0, 0)
    assert_near(out, reference(q, own, lp + lo, nrep, g, bias), dtype, 128, lp + lo, dtype == BF16)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale", [1e-6, 3e4, 1e30])
def test_ranges(gpu, dtype, scale):
    """Value scales far from 1 (fp16 outputs stay in their range), large and tiny queries."""
    if dtype == FP16:
        scale = min(scale, 3e3)
    run(gpu, 1, 4, 2, 4, 300, 40, 128, 32, dtype, 5, scale=scale)
    q = torch.randn(4, 8, 1, 128, device=gpu) * torch.tensor([1e-30, 1e-4, 1.0, 8.0], device=gpu)[:, None, None, None]
    q[3, 0, 0, 5] = 0
    q[1, 1] = 0
    run(gpu, 1, 4, 2, 4, 300, 40, 128, 32, dtype, 6, q=q.to(dtype))


@pytest.mark.parametrize("span", [10, 20])
def test_value_scales_across_keys(gpu, span):
    """A key's value scale 2^span times the others', with most of the weight on a small one."""
    P, N, hkv, nrep, lp, lo, g = 1, 4, 1, 4, 256, 32, 32
    own = cache_of(gpu, N, hkv, lo, lo, 128, g, 2)
    own.prefix = pre = cache_of(gpu, P, hkv, lp, lp, 128, g, 1)
    pre.v_scale[:, :, 3::50] *= 2.0 ** span
    pre.v_scale[:, :, 130] *= 2.0 ** -span
    q = 3 * torch.randn(N, hkv * nrep, 1, 128, device=gpu).to(FP16)
    q = q.to(BF16)
    out = ia.shared_prefix_decode_attention(q, own, lp + lo, nrep, g)
    assert_near(out, reference(q, own, lp + lo, nrep, g), BF16, 128, lp + lo, True)


def test_layouts(gpu):
    """Strided queries, outputs' types through the ABI, caches as slices of larger buffers."""
    P, N, hkv, nrep, lp, lo, g = 2, 4, 2, 4, 333, 21, 64
    B = P * N
    big_pre = cache_of(gpu, P, hkv + 1, lp, 400, 128, g, 1)
    big_own = cache_of(gpu, B, hkv + 1, lo, 50, 128, g, 2)
    part = lambda c: ia.Int4KVLayerCache(*(t[:, 1:] for t in (c.k_packed, c.v_packed, c.k_scale,  # noqa: E731
                                                             c.v_scale)), length=c.length)
    own = part(big_own)
    own.prefix = part(big_pre)
    base = torch.randn(B, 1, hkv * nrep, 130, device=gpu).to(BF16)
    for q in (base.transpose(1, 2)[..., :128], base.transpose(1, 2)[..., 1:129],
              base.transpose(1, 2).repeat_interleave(2, -1)[..., ::2][..., 2:],
              base[..., :128].transpose(1, 2).expand(B, hkv * nrep, 1, 128)):
        ref = reference(q, own, lp + lo, nrep, g)
        out = ia.shared_prefix_decode_attention(q, own, lp + lo, nrep, g)
        assert_near(out, ref, BF16, 128, lp + lo, True)
        for dt in (FP32, FP16, BF16):
            o = torch.empty(128, hkv * nrep, B, device=gpu, dtype=dt).permute(2, 1, 0)
            pre = own.prefix
            _abi.int4_shared_decode_attention(
                q, None, None, (pre.k_packed, pre.v_packed, pre.k_scale, pre.v_scale),
                (own.k_packed, own.v_packed, own.k_scale, own.v_scale), None, o, lp, lp + lo, nrep, g)
            assert_near(o, ref, dt, 128, lp + lo, True)


def test_token_scale(gpu):
    """The token's scales: within one unit in the last place of the pack kernel's quotients, and those
    of int4_quant_dequant on the GPU, in both kernels."""
    B, hkv, g = 64, 8, 32
    own = cache_of(gpu, B, hkv, 5, 8, 128, g, 2)
    own.prefix = cache_of(gpu, 8, hkv, 40, 40, 128, g, 1)
    k, v = torch.randn(2, B, hkv, 1, 128, device=gpu).to(BF16)
    q = torch.randn(B, hkv * 4, 1, 128, device=gpu).to(BF16)
    packed = ia._allocate_layer_cache(B, hkv, 8, 128, 4, gpu)
    _abi.int4_pack_kv_pair(k, v, packed.k_packed, packed.v_packed, packed.k_scale, packed.v_scale,
                           torch.tensor([4], device=gpu), g)
    for generic in (False, True):
        own.k_scale[:, :, 4], own.v_scale[:, :, 4] = 0, 0
        with require_env("LQ_ATTN_FORCE_GENERIC", generic):
            ia.shared_prefix_decode_attention(q, own, 45, 4, g, None, k, v)
        for x, s, w, n in ((k, own.k_scale, packed.k_scale, own.k_packed),
                           (v, own.v_scale, packed.v_scale, own.v_packed)):
            got, want = s[:, :, 4], w[:, :, 4]
            assert (got.view(torch.int32) - want.view(torch.int32)).abs().max() <= 1
            values = oik.dequantize(n[:, :, 4:5].cpu(), s[:, :, 4:5].cpu(), g)
            assert torch.equal(values.to(BF16), ia.int4_quant_dequant(x, g).cpu())


def test_matches_the_plain_decode_attention(gpu):
    """The same keys in one cache per row, through the unshared operator."""
    P, N, hkv, nrep, lp, lo, g = 2, 4, 8, 4, 900, 60, 64
    own = cache_of(gpu, P * N, hkv, lo, lo, 128, g, 2)
    own.prefix = pre = cache_of(gpu, P, hkv, lp, lp, 128, g, 1)
    one = ia.Int4KVLayerCache(*(torch.cat((a.repeat_interleave(N, 0), b), 2) for a, b in
                                ((pre.k_packed, own.k_packed), (pre.v_packed, own.v_packed),
                                 (pre.k_scale, own.k_scale), (pre.v_scale, own.v_scale))))
    q = torch.randn(P * N, hkv * nrep, 1, 128, device=gpu).to(BF16)
    a = ia.shared_prefix_decode_attention(q, own, lp + lo, nrep, g)
    b = ia._decode_attention(q, one, lp + lo, nrep, g)
    ref = reference(q, own, lp + lo, nrep, g)
    assert_near(a, ref, BF16, 128, lp + lo, True)
    assert_near(b, ref, BF16, 128, lp + lo, True)


def test_stream_and_capture(gpu):
    """Two captured steps and eager calls of other shapes between their replays."""
    P, N, hkv, nrep, lp, g = 1, 8, 8, 4, 1500, 32
    own = cache_of(gpu, P * N, hkv, 20, 64, 128, g, 2)
    own.prefix = cache_of(gpu, P, hkv, lp, lp + 4, 128, g, 1)
    other = cache_of(gpu, 64, hkv, 40, 64, 128, g, 3)
    other.prefix = cache_of(gpu, 8, hkv, 8000, 8000, 128, g, 4)
    q = torch.randn(P * N, hkv * nrep, 1, 128, device=gpu).to(BF16)
    big = torch.randn(64, hkv * nrep, 1, 128, device=gpu).to(BF16)
    k, v = torch.randn(2, P * N, hkv, 1, 128, device=gpu).to(BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for S in (lp + 21, lp + 10):
            g_ = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g_, stream=side):
                out = ia.shared_prefix_decode_attention(q, own, S, nrep, g, None, k, v)
            graphs.append((g_, S, out))
    torch.cuda.current_stream().wait_stream(side)
    for i in range(3):
        q.normal_()
        k.normal_()
        ia.shared_prefix_decode_attention(big, other, 8040, nrep, g)
        for g_, S, out in graphs:
            g_.replay()
            ref = reference(q, own, S, nrep, g)
            assert_near(out, ref, BF16, 128, S, True, f"replay {i}")


def test_threads_on_one_stream(gpu):
    """Two threads whose calls (a launch that leaves partials, a merge that reads them) interleave on one
    stream."""
    hkv, nrep, g = 8, 4, 32
    calls = []
    for P, N, lp, seed in ((1, 4, 2000, 1), (2, 3, 1500, 2)):
        own = cache_of(gpu, P * N, hkv, 20, 32, 128, g, seed)
        own.prefix = cache_of(gpu, P, hkv, lp, lp, 128, g, seed + 10)
        q = torch.randn(P * N, hkv * nrep, 1, 128, device=gpu).to(BF16)
        calls.append((q, own, lp + 20, nrep, g))
    alone = [ia.shared_prefix_decode_attention(*c) for c in calls]
    outs = [[], []]
    start = threading.Barrier(2)

    def work(i):
        start.wait()
        for _ in range(200):
            outs[i].append(ia.shared_prefix_decode_attention(*calls[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(outs[i]) == 200
        assert all(torch.equal(o, alone[i]) for o in outs[i])


def test_long_prefix_offsets(gpu):
    """A prefix whose byte offsets pass 32 bits between the prompts and between the heads."""
    P, N, hkv, nrep, lp, lo, g = 2, 2, 9, 1, 70, 2, 128
    cap = 1 << 22
    shape = (P, hkv, cap, 64)
    pre = cache_of(gpu, P, hkv, lp, lp, 128, g, 1)
    big = [torch.zeros(shape, dtype=torch.uint8, device=gpu) for _ in range(2)] + \
          [torch.zeros(P, hkv, cap, 1, device=gpu) for _ in range(2)]
    for t, s in zip(big, (pre.k_packed, pre.v_packed, pre.k_scale, pre.v_scale)):
        t[:, :, :lp] = s
    own = cache_of(gpu, P * N, hkv, lo, lo, 128, g, 2)
    own.prefix = ia.Int4KVLayerCache(*big, length=lp)
    q = torch.randn(P * N, hkv * nrep, 1, 128, device=gpu).to(BF16)
    out = ia.shared_prefix_decode_attention(q, own, lp + lo, nrep, g)
    assert_near(out, reference(q, own, lp + lo, nrep, g), BF16, 128, lp + lo, True)
