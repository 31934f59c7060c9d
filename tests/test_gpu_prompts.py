"""The prompt operators on the GPU against their definitions in 64 bits (prompt_reference.py, with the
error bounds' derivation)."""
import math

import pytest
import torch

import prompt_reference as ref
from layer_quant_amd import prompts

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def starts_of(lengths, device, dtype=torch.int32, first=0):
    s = [first]
    for n in lengths:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=dtype, device=device)


def within(got, want, bound, what):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN places"
    err = torch.where(got == want, torch.zeros_like(want), (got - want).abs())
    worst = torch.nan_to_num(err / bound.clamp_min(1e-300), nan=0.0).amax().item() if got.numel() else 0
    print(f"[{what}] worst error over bound {worst:.3g}")
    assert worst <= 1, f"{what}: {worst:.3g}"


def attention_inputs(gpu, rows, hq, hkv, d, dtype, seed=0):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    make = lambda h: torch.randn(rows, h, d, device=gpu, generator=gen).to(dtype)  # noqa: E731
    return make(hq), make(hkv), make(hkv)


def check_attention(gpu, q, k, v, starts, what, scale=None, out=None):
    got = prompts.prompt_attention(q, k, v, starts, scale=scale, out=out)
    want, weight, score = ref.attention(q, k, v, starts.tolist(), scale)
    within(got, want, ref.attention_bound(want, weight, score, q.dtype, q.shape[-1]), what)
    return got


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("lengths", [[1], [0], [2, 0, 5], [31, 32, 33], [63, 64, 65, 1], [200], [129, 3, 0]],
                         ids=str)
@pytest.mark.parametrize("heads", [(8, 2), (3, 3), (5, 1)], ids=str)
def test_attention_lengths(gpu, dtype, lengths, heads):
    q, k, v = attention_inputs(gpu, sum(lengths), *heads, 128, dtype)
    check_attention(gpu, q, k, v, starts_of(lengths, gpu), f"{lengths} {heads} {dtype}")


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("d", [1, 7, 32, 64, 72, 80, 96, 112, 128, 160, 256])
def test_attention_head_dims(gpu, dtype, d):
    q, k, v = attention_inputs(gpu, 101, 6, 2, d, dtype)
    check_attention(gpu, q, k, v, starts_of([70, 31], gpu, torch.int64), f"D {d} {dtype}")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_model_heads(gpu, dtype):
    lengths = [1, 300, 0, 77, 128, 2]
    q, k, v = attention_inputs(gpu, sum(lengths), 32, 8, 128, dtype, seed=1)
    k = k * (1 + 20 * (torch.arange(128, device=gpu) % 37 == 0)).to(dtype)  # peaked rows
    check_attention(gpu, q, k, v, starts_of(lengths, gpu), f"model {dtype}")


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_attention_strides(gpu, dtype):
    """A batch from [B, heads, L, D] projections, and rows, heads and dims in other orders."""
    gen = torch.Generator(device=gpu).manual_seed(2)
    make = lambda *s: torch.randn(*s, device=gpu, generator=gen).to(dtype)  # noqa: E731
    q, k, v = make(3, 4, 50, 64), make(3, 2, 50, 64), make(3, 2, 50, 64)
    got = prompts.prompt_attention(*(t.transpose(1, 2) for t in (q, k, v)))
    flat = [t.transpose(1, 2).reshape(150, -1, 64) for t in (q, k, v)]
    want, weight, score = ref.attention(*flat, [0, 50, 100, 150])
    bound = ref.attention_bound(want, weight, score, dtype, 64)
    within(got.reshape(150, 4, 64), want, bound, "batch")
    starts = starts_of([50] * 3, gpu)
    for form in ("dims", "odd", "wide"):
        if form == "dims":
            views = [t.permute(1, 2, 0).contiguous().permute(2, 0, 1) for t in flat]
            out = torch.empty(64, 4, 150, device=gpu, dtype=dtype).permute(2, 1, 0)
        elif form == "odd":  # rows that begin off any alignment
            views = [torch.empty(150, t.shape[1] * 64 + 3, device=gpu, dtype=dtype)[:, 1:-2]
                     .unflatten(1, (-1, 64)).copy_(t) for t in flat]
            out = torch.empty(150, 4 * 64 + 1, device=gpu, dtype=dtype)[:, 1:].unflatten(1, (4, 64))
        else:  # q, k and v of one tensor
            fused = torch.cat([t.flatten(1) for t in flat], 1)
            views = [t.unflatten(1, (-1, 64)) for t in fused.split([256, 128, 128], 1)]
            out = torch.empty(150, 4, 128, device=gpu, dtype=dtype)[:, :, 64:]
        got = prompts.prompt_attention(*views, starts, out=out)
        assert got is out
        within(got, want, bound, f"{form} {dtype}")


@pytest.mark.parametrize("dtype", [BF, F16])
def test_attention_kernels_by_layout(gpu, dtype, diag):
    """16-bit rows of 64 or 128 dims, 16-byte aligned, take the matrix kernel, and agree with the general
    one; anything else takes the general one."""
    from layer_quant_amd import _abi

    for d in (64, 128):
        q, k, v = attention_inputs(gpu, 333, 8, 2, d, dtype, seed=11)
        starts = starts_of([300, 33], gpu)
        want, weight, score = ref.attention(q, k, v, starts.tolist())
        bound = ref.attention_bound(want, weight, score, dtype, d)
        diag.set("LQ_PROMPT_REQUIRE_MFMA")
        within(prompts.prompt_attention(q, k, v, starts), want, bound, f"matrix {d}")
        wide = torch.zeros(333, 2, d + 8, device=gpu, dtype=dtype)
        prompts.prompt_attention(q, wide[..., :d], wide[..., 8:], starts)
        for bad in (wide[..., 1:d + 1], wide[:1].expand(333, 2, d + 8)[..., :d], k[:, :, ::2].repeat(1, 1, 2)
                    .transpose(0, 2).contiguous().transpose(0, 2)):
            with pytest.raises(_abi.LQError, match="general kernel"):
                prompts.prompt_attention(q, bad, v, starts)
        diag.clear("LQ_PROMPT_REQUIRE_MFMA")
        diag.set("LQ_PROMPT_FORCE_GENERIC")
        within(prompts.prompt_attention(q, k, v, starts), want, bound, f"general {d}")
        diag.clear("LQ_PROMPT_FORCE_GENERIC")


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_nothing_from_behind(gpu, dtype, bad):
    """Rows behind a row, of its prompt and of the next one, and rows of no prompt never reach it; a
    row at or before it does."""
    lengths, first, total = [70, 40], 5, 140
    q, k, v = attention_inputs(gpu, total, 4, 2, 128, dtype, seed=3)
    clean = [t.clone() for t in (q, k, v)]
    starts = starts_of(lengths, gpu, first=first)
    for row in (0, first + 66, first + 70 + 11, 120, 139):
        k[row], v[row] = bad, bad
    got = prompts.prompt_attention(q, k, v, starts).cpu()
    want, weight, score = ref.attention(*clean, starts.tolist())
    bound = ref.attention_bound(want, weight, score, dtype, 128)
    good = [*range(first, first + 66), *range(first + 70, first + 81)]
    within(got[good], want[good], bound[good], "in front of it")
    hit = [*range(first + 66, first + 70), *range(first + 81, first + 110)]
    assert not torch.isfinite(got[hit]).any()
    rest = [*range(first), *range(first + 110, total)]
    assert (got[rest] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_attention_masked_scores(gpu, dtype):
    """Keys whose score is -inf have no weight, wherever they stand; a row of such keys alone is NaN."""
    q, k, v = attention_inputs(gpu, 150, 4, 1, 128, dtype, seed=4)
    q = q.abs()
    k[:100, 0, 0] = -math.inf
    starts = starts_of([150], gpu)
    got = prompts.prompt_attention(q, k, v, starts).cpu()
    assert torch.isnan(got[:100]).all()
    want, weight, score = ref.attention(q[100:], k[100:], v[100:], [0, 50])
    within(got[100:], want, ref.attention_bound(want, weight, score, dtype, 128), "behind them")


def test_attention_scale_and_large_scores(gpu):
    q, k, v = attention_inputs(gpu, 90, 4, 4, 64, BF, seed=5)
    starts = starts_of([90], gpu)
    check_attention(gpu, q, k, v, starts, "scale 0", scale=0.0)
    check_attention(gpu, q, k, v, starts, "negative scale", scale=-0.3)
    check_attention(gpu, (q * 30).contiguous(), k, v, starts, "large scores", scale=1.0)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_attention_small_values(gpu, dtype):
    """Values, and products of scores, below the type's smallest normal number."""
    q, k, v = attention_inputs(gpu, 70, 4, 2, 128, dtype, seed=12)
    least = torch.finfo(dtype).tiny
    starts = starts_of([70], gpu)
    got = prompts.prompt_attention(q, (k.float() * least).to(dtype), (v.float() * least / 4).to(dtype), starts,
                                   scale=1.0)
    want, weight, score = ref.attention(q, (k.float() * least).to(dtype), (v.float() * least / 4).to(dtype),
                                        [0, 70], 1.0)
    within(got, want, ref.attention_bound(want, weight, score, dtype, 128), f"{dtype}")


def test_attention_in_place(gpu):
    q, k, v = attention_inputs(gpu, 300, 4, 2, 128, BF, seed=13)
    starts = starts_of([200, 100], gpu)
    want = prompts.prompt_attention(q, k, v, starts)
    assert torch.equal(prompts.prompt_attention(q, k, v, starts, out=q), want)


def test_offsets_past_32_bits(gpu):
    """Rows 128 KiB apart and more: the same as rows one behind another."""
    rows, apart = 40000, 65536
    far = torch.empty(rows * apart, device=gpu, dtype=BF)
    gen = torch.Generator(device=gpu).manual_seed(14)
    tight = torch.randn(rows, 1, 384, device=gpu, generator=gen).to(BF)
    wide = far.as_strided((rows, 1, 384), (apart, 384, 1))
    wide.copy_(tight)
    starts = torch.tensor([0, 7, rows], device=gpu)
    split = lambda t: t.split(128, 2)  # noqa: E731
    assert torch.equal(prompts.prompt_attention(*split(wide), starts),
                       prompts.prompt_attention(*split(tight), starts))
    x = lambda t: t.as_strided((rows, 2, 64), (t.stride(0), 64, 1), t.storage_offset())  # noqa: E731
    dt, A = torch.randn(rows, 2, device=gpu, generator=gen), -torch.rand(2, device=gpu, generator=gen)
    got = [prompts.prompt_scan(x(t), dt, A, *split(t)[1:], starts, dt_softplus=True) for t in (wide, tight)]
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    logits = torch.randn(20, 131072, device=gpu, generator=gen).to(BF)
    spread = far.as_strided((20, 131072), (1 << 27, 1))
    spread.copy_(logits)
    tokens = torch.arange(20, device=gpu)
    for a, b in zip(prompts.token_logprobs(spread, tokens, 4), prompts.token_logprobs(logits, tokens, 4)):
        assert torch.equal(a, b)


def test_attention_out_of_range_starts(gpu):
    """Starts past the rows count as the last row: nothing outside is read or written."""
    q, k, v = attention_inputs(gpu, 60, 4, 2, 128, BF, seed=6)
    wild = torch.tensor([-7, 20, 1 << 40], device=gpu)
    got = prompts.prompt_attention(q, k, v, wild)
    assert torch.equal(got, prompts.prompt_attention(q, k, v, torch.tensor([0, 20, 60], device=gpu)))


def test_attention_many_prompts(gpu):
    """More prompts than a wave looks at at once, single tokens among them: v itself."""
    lengths = [1, 0, 3, 1, 2] * 60
    q, k, v = attention_inputs(gpu, sum(lengths), 4, 2, 128, F16, seed=7)
    starts = starts_of(lengths, gpu)
    got = check_attention(gpu, q, k, v, starts, "300 prompts")
    ones = [int(s) for s, n in zip(starts.tolist(), lengths) if n == 1]
    assert torch.equal(got[ones], v[ones].repeat_interleave(2, 1))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_long_prompt_rows(gpu, dtype):
    """Sampled rows of a long prompt."""
    q, k, v = attention_inputs(gpu, 5000, 4, 1, 128, dtype, seed=8)
    got = prompts.prompt_attention(q, k, v, starts_of([5000], gpu)).cpu()
    for t in (0, 63, 64, 2047, 4095, 4999):
        s = (k[:t + 1, 0].double() @ q[t].double().T) / math.sqrt(128)
        p = torch.softmax(s, 0).cpu()
        vv = v[:t + 1, 0].double().cpu()
        want, weight = p.T @ vv, p.T @ vv.abs()
        score = ((k[:t + 1, 0].double().abs() @ q[t].double().abs().T) / math.sqrt(128)).amax(0).cpu()
        within(got[t], want, ref.attention_bound(want, weight, score, dtype, 128), f"row {t}")


def scan_inputs(gpu, rows, h, p, n, g, dtype, seed=0, dt_dtype=None):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen)  # noqa: E731
    rand = lambda *s: torch.rand(*s, device=gpu, generator=gen)  # noqa: E731
    return dict(x=randn(rows, h, p).to(dtype), dt=randn(rows, h).to(dt_dtype or dtype),
                A=-(0.5 + 4 * rand(h)), B=randn(rows, g, n).to(dtype), C=randn(rows, g, n).to(dtype),
                D=randn(h), z=randn(rows, h, p).to(dtype), dt_bias=randn(h) - 3)


def scan_bounds(y, s, wy, ws, dtype, state_dtype, rows):
    """bf16 products: the mixing weights and the state in front of a chunk are rounded to bf16 (half a
    step, 2^-8 of the terms' sum); the state's own terms to two bf16 numbers (2^-16) or
    three. fp32 sums, decays
    and steps: less than 2^-21 of the terms' sum per 64 rows, and 2^-18 for logarithms and exponentials
    of decays (a decay exp(-u) is off by u 2^-22 of itself at most, u exp(-u) < 1 where it counts). A result below the type's
    smallest normal number is rounded to a multiple of tiny * eps."""
    half = torch.finfo(dtype).eps / 2
    fp32 = 2.0 ** -18 + (rows / 64 + 1) * 2.0 ** -21
    put = 0.0 if state_dtype == F32 else torch.finfo(state_dtype).eps / 2
    own = fp32 if dtype != BF else 2.0 ** -16 + fp32
    mix = fp32 if dtype != BF else 2.0 ** -8 + own
    step = lambda t: torch.finfo(t).tiny * torch.finfo(t).eps  # noqa: E731
    return (half * y.abs() + mix * wy + step(dtype) / 2 + 1e-30,
            put * s.abs() + own * ws + step(state_dtype) / 2 + 1e-30)


def check_scan(gpu, t, starts, what, *, use=("D", "dt_bias"), softplus=True, limit=(0.0, math.inf),
               initial=None, states=None, first_states=None):
    opt = {k: t[k] for k in use}
    y, st = prompts.prompt_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], starts, dt_softplus=softplus,
                                dt_limit=limit, initial_states=initial, states=states, **opt)
    want, ws, wy, size = ref.scan(t["x"], t["dt"], t["A"], t["B"], t["C"], starts.tolist(),
                                  dt_softplus=softplus, dt_limit=limit,
                                  initial=first_states if first_states is not None else initial, **opt)
    by, bs = scan_bounds(want, ws, wy, size, t["x"].dtype, st.dtype, t["x"].shape[0])
    within(y, want, by, f"{what} y")
    within(st, ws, bs, f"{what} states")
    return y, st


GEOMETRIES = [(16, 64, 128, 2), (8, 16, 32, 2), (3, 64, 128, 1), (4, 70, 100, 2), (2, 5, 3, 1),
              (2, 128, 256, 2), (6, 64, 64, 2)]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("geometry", GEOMETRIES, ids=str)
def test_scan_geometries(gpu, dtype, geometry):
    lengths = [65, 1, 0, 130]
    t = scan_inputs(gpu, sum(lengths), *geometry, dtype)
    check_scan(gpu, t, starts_of(lengths, gpu), f"{geometry} {dtype}", use=("D", "dt_bias", "z"))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("lengths", [[1], [0], [63, 64], [128, 0, 1], [2, 3, 300]], ids=str)
@pytest.mark.parametrize("state", [BF, F16, F32])
def test_scan_lengths_and_states(gpu, dtype, lengths, state):
    h, p, n = 8, 64, 128
    t = scan_inputs(gpu, sum(lengths), h, p, n, 2, dtype, seed=1)
    gen = torch.Generator(device=gpu).manual_seed(2)
    initial = torch.randn(len(lengths), h, p, n, device=gpu, generator=gen).to(state)
    first = initial.clone()
    # in place: the state behind the prompts takes the initial one's tensor
    y, st = check_scan(gpu, t, starts_of(lengths, gpu, torch.int64), f"{lengths} {state} {dtype}",
                       initial=initial, states=initial, first_states=first)
    assert st is initial


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_segments(gpu, dtype):
    """Prompts of more than one segment next to short ones, states in place, rows of no prompt around."""
    h, p, n = 4, 64, 128
    lengths, first, total = [700, 3, 1100, 0, 256, 257], 9, 2340
    t = scan_inputs(gpu, total, h, p, n, 1, dtype, seed=3)
    t["A"] *= 0.05  # long memory: the carried states count
    gen = torch.Generator(device=gpu).manual_seed(4)
    initial = torch.randn(len(lengths), h, p, n, device=gpu, generator=gen)
    y, _ = check_scan(gpu, t, starts_of(lengths, gpu, first=first), f"segments {dtype}",
                      initial=initial, states=initial, first_states=initial.clone())
    assert (y[:first] == 0).all() and (y[first + sum(lengths):] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F16])
def test_scan_many_segments(gpu, dtype):
    """One long prompt in ten segments and more, the state in place, and without states before it."""
    t = scan_inputs(gpu, 2600, 4, 64, 128, 1, dtype, seed=20)
    t["A"] *= 0.02
    starts = starts_of([2600], gpu)
    state = torch.randn(1, 4, 64, 128, device=gpu, generator=torch.Generator(device=gpu).manual_seed(21))
    check_scan(gpu, t, starts, "in place", initial=state, states=state, first_states=state.clone())
    check_scan(gpu, t, starts, "bf16 states", states=torch.empty(1, 4, 64, 128, device=gpu, dtype=BF))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_scan_strides_and_options(gpu, dtype):
    """Views of one tensor as the convolution leaves them, a batch, fp32 steps, limits, no softplus."""
    h, p, n, g, b, rows = 8, 64, 128, 2, 3, 90
    gen = torch.Generator(device=gpu).manual_seed(5)
    xbc = torch.randn(b, rows, h * p + 2 * g * n, device=gpu, generator=gen).to(dtype)
    t = scan_inputs(gpu, b * rows, h, p, n, g, dtype, seed=6, dt_dtype=F32)
    t["x"], t["B"], t["C"] = (v.unflatten(-1, (hh, -1)) for v, hh in
                              zip(xbc.split([h * p, g * n, g * n], -1), (h, g, g)))
    t["dt"] = t["dt"].abs().reshape(b, rows, h) * 0.3
    y, st = prompts.prompt_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], D=t["D"].to(dtype),
                                z=t["z"].reshape(b, rows, h, p), dt_limit=(0.05, 0.4))
    flat = {k: t[k].flatten(0, 1) for k in ("x", "dt", "B", "C")}
    starts = [0, rows, 2 * rows, 3 * rows]
    want, ws, wy, size = ref.scan(flat["x"], flat["dt"], t["A"], flat["B"], flat["C"], starts,
                                  D=t["D"].to(dtype), z=t["z"], dt_limit=(0.05, 0.4))
    by, bs = scan_bounds(want, ws, wy, size, dtype, F32, rows)
    within(y.flatten(0, 1), want, by, "batch y")
    within(st, ws, bs, "batch states")
    # rows that begin off any alignment, transposed states
    odd = {k: torch.empty(b * rows, v.shape[1] * v.shape[2] + 1, device=gpu, dtype=dtype)[:, 1:]
           .unflatten(1, v.shape[1:]).copy_(v) for k, v in flat.items() if k != "dt"}
    states = torch.empty(b, h, n, p, device=gpu).transpose(2, 3)
    y, st = prompts.prompt_scan(odd["x"], flat["dt"], t["A"], odd["B"], odd["C"],
                                torch.tensor(starts, device=gpu), D=t["D"].to(dtype), z=t["z"],
                                dt_limit=(0.05, 0.4), states=states)
    within(y, want, by, "odd y")
    within(st, ws, bs, "odd states")


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_scan_nothing_from_behind(gpu, dtype, bad):
    h, p, n = 4, 64, 128
    lengths = [100, 60]
    t = scan_inputs(gpu, 160, h, p, n, 1, dtype, seed=7)
    starts = starts_of(lengths, gpu)
    want, ws, wy, size = ref.scan(t["x"], t["dt"], t["A"], t["B"], t["C"], starts.tolist(),
                                  D=t["D"], dt_bias=t["dt_bias"], dt_softplus=True)
    by, bs = scan_bounds(want, ws, wy, size, dtype, F32, 160)
    for field in ("x", "B", "C", "dt"):
        broken = dict(t, **{field: t[field].clone()})
        broken[field][70] = bad
        y, st = prompts.prompt_scan(broken["x"], broken["dt"], t["A"], broken["B"], broken["C"], starts,
                                    D=t["D"], dt_bias=t["dt_bias"], dt_softplus=True)
        within(y[:70], want[:70], by[:70], f"{field} y in front of it")
        within(y[100:], want[100:], by[100:], f"{field} y of the next prompt")
        within(st[1], ws[1], bs[1], f"{field} the next prompt's state")
        if field != "C":
            assert not torch.isfinite(st[0]).all()
        assert not torch.isfinite(y[70]).all()


def test_scan_large_and_small_steps(gpu):
    """Decays that end a state at once, and steps so small that log(1 + e^x) needs its small values."""
    t = scan_inputs(gpu, 200, 4, 64, 128, 1, F32, seed=8)
    t["dt"][:100] *= 30
    t["dt"][100:] -= 14
    t["A"] = -torch.tensor([0.0, 1e-4, 1.0, 300.0], device=gpu)
    check_scan(gpu, t, starts_of([200], gpu), "fp32")
    for k in ("x", "B", "C"):
        t[k] = t[k].to(BF)
    check_scan(gpu, t, starts_of([200], gpu), "bf16")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_no_prompts_at_all(gpu, dtype):
    """One start, no prompt: every row is of none."""
    starts = torch.tensor([5], device=gpu)
    t = scan_inputs(gpu, 3000, 8, 64, 128, 1, dtype)
    y, st = prompts.prompt_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], starts)
    assert st.shape == (0, 8, 64, 128) and y.shape == t["x"].shape and not y.any()
    q, k, v = attention_inputs(gpu, 3000, 4, 2, 64, dtype)
    assert not prompts.prompt_attention(q, k, v, starts).any()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("size", [1e-3, 1.0, 30.0])
def test_scan_decays_of_a_block(gpu, dtype, size):
    """Sixteen rows that decay by little, by almost 2^-40, by little more, by 2^-400, that grow, and whose steps
    are negative: the state is scaled within some of them and not in others."""
    h = 6
    t = scan_inputs(gpu, 150, h, 64, 128, 1, dtype, seed=11, dt_dtype=F32)
    t["x"] *= size
    t["dt"] = torch.ones(150, h, device=gpu) / 8
    per_row = torch.tensor([0.01, 39.9 / 16, 40.1 / 16, 25.0, -0.02, 2.0], device=gpu)
    t["A"] = -per_row * 8 * math.log(2)
    t["dt"][20:22, 5] *= -1
    t["dt"][60:, 1] *= 1.01
    check_scan(gpu, t, starts_of([150], gpu), f"{dtype} {size}", use=("D",), softplus=False,
               limit=(-math.inf, math.inf))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lengths", [[200], [258], [0, 150, 129], [300, 1, 290], [256], [700]], ids=str)
def test_scan_few_short_prompts(gpu, dtype, lengths):
    """Many heads and few rows: whole prompts, or segments of 64 rows."""
    t = scan_inputs(gpu, sum(lengths), 128, 4, 16, 2, dtype, seed=12)
    first = torch.randn(len(lengths), 128, 4, 16, device=gpu)
    check_scan(gpu, t, starts_of(lengths, gpu), f"{lengths}", use=("D", "dt_bias", "z"), initial=first)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_starts_out_of_order(gpu, dtype):
    """Starts that do not ascend give no defined values, and read and write nothing outside."""
    t = scan_inputs(gpu, 1500, 4, 64, 128, 1, dtype, seed=16)
    for s in ([0, 1500, 0, 1500, 0, 1500], [1500, 0], [-5, 3000, 7, -1, 1500], [900, 900, 100, 1500]):
        starts = torch.tensor(s, device=gpu)
        y, st = prompts.prompt_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], starts, dt_softplus=True)
        prompts.prompt_attention(t["x"], t["x"], t["x"], starts)
        torch.cuda.synchronize()
        assert y.shape == t["x"].shape and st.shape[0] == len(s) - 1


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scan_growing_and_nan_decays(gpu, dtype):
    """A > 0 (states that grow), A = 0, and NaN in A: that head's rows and state alone."""
    t = scan_inputs(gpu, 90, 4, 64, 128, 1, dtype, seed=17)
    t["A"] = torch.tensor([0.5, 0.0, math.nan, -1.0], device=gpu)
    y, st = prompts.prompt_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], starts_of([90], gpu),
                                dt_bias=t["dt_bias"], dt_softplus=True)
    assert torch.isnan(y[:, 2]).all() and torch.isnan(st[0, 2]).all()
    good = [0, 1, 3]
    pick = dict(t, x=t["x"][:, good], dt=t["dt"][:, good], A=t["A"][good], dt_bias=t["dt_bias"][good])
    want, ws, wy, size = ref.scan(pick["x"], pick["dt"], pick["A"], t["B"], t["C"], [0, 90],
                                  dt_bias=pick["dt_bias"], dt_softplus=True)
    by, bs = scan_bounds(want, ws, wy, size, dtype, F32, 90)
    within(y[:, good], want, by, "y")
    within(st[:, good], ws, bs, "states")


def test_scan_single_row_strides(gpu):
    """A batch of single rows whose row strides say nothing (a transposed view of one row)."""
    t = scan_inputs(gpu, 3, 8, 64, 128, 2, BF, seed=18)
    y, st = prompts.prompt_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], starts_of([1, 1, 1], gpu))
    odd = {k: t[k].as_strided((3, 1, *t[k].shape[1:]), (t[k].stride(0), 0, *t[k].stride()[1:]))
           for k in ("x", "dt", "B", "C")}
    y1, st1 = prompts.prompt_scan(odd["x"], odd["dt"], t["A"], odd["B"], odd["C"])
    want, ws, wy, size = ref.scan(t["x"], t["dt"], t["A"], t["B"], t["C"], [0, 1, 2, 3])
    by, bs = scan_bounds(want, ws, wy, size, BF, F32, 3)
    for a, b in ((y, st), (y1[:, 0], st1)):
        within(a, want, by, "y")
        within(b, ws, bs, "states")


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_scan_kernels_by_layout(gpu, dtype, diag):
    """bf16 with 64 x 128 states, 16-byte aligned, takes the matrix kernel, anything else the rows one."""
    from layer_quant_amd import _abi

    t = scan_inputs(gpu, 400, 8, 64, 128, 2, dtype, seed=19)
    starts = starts_of([300, 100], gpu)
    diag.set("LQ_PROMPT_REQUIRE_MFMA")
    if dtype == BF:
        check_scan(gpu, t, starts, "matrix")
    else:
        with pytest.raises(_abi.LQError, match="general kernel"):
            check_scan(gpu, t, starts, "rows")
    diag.clear("LQ_PROMPT_REQUIRE_MFMA")
    diag.set("LQ_PROMPT_FORCE_GENERIC")
    check_scan(gpu, t, starts, "rows")


def test_scan_agrees_with_single_tokens(gpu):
    """A prompt, then one token at a time from its state: the scan of the whole."""
    from layer_quant_amd import mamba_state_8b_kernel as ms

    h, p, n, g = 8, 64, 128, 2
    t = scan_inputs(gpu, 80, h, p, n, g, F32, seed=9)
    one = dict(D=t["D"], dt_bias=t["dt_bias"], dt_softplus=True)
    whole, last = prompts.prompt_scan(t["x"], t["dt"], t["A"], t["B"], t["C"], starts_of([80], gpu), **one)
    cut = {k: t[k][:75] for k in ("x", "dt", "B", "C")}
    _, st = prompts.prompt_scan(cut["x"], cut["dt"], t["A"], cut["B"], cut["C"], starts_of([75], gpu), **one)
    wide = lambda v: v[:, None].expand(h, p)  # noqa: E731
    for i in range(75, 80):
        y = ms.selective_state_update(st, t["x"][i:i + 1], t["dt"][i:i + 1, :, None].expand(1, h, p),
                                      t["A"][:, None, None].expand(h, p, n), t["B"][i:i + 1],
                                      t["C"][i:i + 1], wide(t["D"]), dt_bias=wide(t["dt_bias"]),
                                      dt_softplus=True)
        assert (y[0] - whole[i]).norm() <= 1e-5 * whole[i].norm()
    assert (st - last).norm() <= 1e-5 * last.norm()


def check_scores(gpu, logits, tokens, top, what):
    got = prompts.token_logprobs(logits, tokens, top)
    flat, vocab = logits.reshape(-1, logits.shape[-1]), logits.shape[-1]
    want, entropy, lp = ref.logprobs(flat, tokens.reshape(-1))
    # fp32: sums of V terms in runs of less than 64 (2^-18 of the sum), the exponentials' arguments and
    # values (2^-21 of them), the result's own rounding
    bound = lambda t: 2.0 ** -17 + 2.0 ** -21 * t.abs()  # noqa: E731
    within(got.logprobs.reshape(-1), want, bound(want), f"{what} logprobs")
    spread = entropy + (flat.double().cpu().clamp(-1e30).amax(-1) * 0)
    within(got.entropy.reshape(-1), entropy, bound(spread) + 2.0 ** -18 * entropy.abs(), f"{what} entropy")
    assert got.logprobs.shape == tokens.shape == got.entropy.shape
    if not top:
        assert got.top_logprobs is None and got.top_tokens is None
        return got
    best = torch.sort(flat.float().cpu() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    known = ~torch.isnan(entropy)
    assert torch.equal(got.top_tokens.reshape(-1, top).cpu()[known], best[known]), what
    want = lp.gather(1, best)
    within(got.top_logprobs.reshape(-1, top)[known.to(gpu)], want[known], bound(want[known]), f"{what} top")
    rest = got.top_tokens.reshape(-1, top).cpu()[~known]
    assert (rest == torch.arange(top)).all()
    assert torch.isnan(got.top_logprobs.reshape(-1, top).cpu()[~known]).all()
    return got


def scores_inputs(gpu, rows, vocab, dtype, seed=0):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    logits = (3 * torch.randn(rows, vocab, device=gpu, generator=gen)).to(dtype)
    return logits, torch.randint(0, vocab, (rows,), device=gpu, generator=gen)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 255, 32), (4, 8191, 0), (3, 8192, 5), (2, 8193, 32),
    (9, 32000, 1), (2, 50257, 20), (1, 131072, 32), (700, 999, 4), (3, 200001, 8), (300, 16391, 0)])
def test_scores_sizes(gpu, dtype, rows, vocab, top):
    logits, tokens = scores_inputs(gpu, rows, vocab, dtype)
    check_scores(gpu, logits, tokens, top, f"{rows} x {vocab} {dtype}")


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_scores_ties_and_masks(gpu, dtype):
    """Equal logits by the thousand, zeros of both signs, the type's lowest value, -inf rows, NaN, +inf,
    tokens outside the vocabulary."""
    logits, tokens = scores_inputs(gpu, 12, 20011, dtype, seed=1)
    logits[0] = 1.5
    logits[1] = -math.inf
    logits[1, 17] = 2.0
    logits[2, 5000] = math.nan
    logits[3, 5000] = math.inf
    logits[4] = -math.inf
    logits[5] = torch.finfo(dtype).min
    logits[5, ::3] = 0.0
    logits[5, 1::6] = -0.0
    logits[6] = logits[6].round()
    logits[7, :] = -math.inf
    logits[7, 30:33] = 1.0
    logits[8] *= 1000 if dtype != F16 else 100
    logits[9, 9000] = 60000.0
    tokens[10], tokens[11], tokens[1] = -100, 20011, 17
    tokens[7] = 4  # a masked token: -inf
    check_scores(gpu, logits, tokens, 32, f"ties {dtype}")
    assert prompts.token_logprobs(logits, tokens).logprobs[7] == -math.inf


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_scores_strides(gpu, dtype):
    """A text's window of [B, L, V] logits, rows off any alignment, a transposed matrix."""
    gen = torch.Generator(device=gpu).manual_seed(3)
    logits = torch.randn(2, 9, 8201, device=gpu, generator=gen).to(dtype)
    ids = torch.randint(0, 8201, (2, 9), device=gpu, generator=gen)
    check_scores(gpu, logits[:, :-1], ids[:, 1:], 3, "window")
    check_scores(gpu, logits[..., 1:-3], ids - 5, 3, "odd")
    check_scores(gpu, logits[0].T.contiguous().T, ids[0], 3, "transposed")
    check_scores(gpu, logits[:1, :1].expand(2, 9, 8201), ids, 2, "expanded")


def test_scores_of_nothing(gpu):
    got = prompts.token_logprobs(torch.empty(0, 50, device=gpu), torch.empty(0, dtype=torch.int64, device=gpu), 4)
    assert got.logprobs.shape == (0,) and got.top_tokens.shape == (0, 4)
