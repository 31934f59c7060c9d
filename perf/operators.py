"""Performance cases of beam decoding: several rows per prompt over the quantized decode states.

Geometry is the 8B model's: attention with 32 query and 8 KV heads of 128 dims over an INT4 KV cache
(4 layers, group 32, 64 or 128), 24 Mamba2 layers with a state of 128 heads x 64 x 128 and a
convolution state of 10240 channels x 4.

Kinds of case
  shared    one attention layer's decode step of `prompts` x `beams` rows: pack the step's token into
            each row's own cache, attend over the prompt's cache (one for all its rows) and the own one;
            with `mask` the prompts are left-padded and the call gets the 2-D keep-mask
  select    the best continuations of each prompt from the step's logits and the running scores
  reorder   the states of the rows follow the selected beams, in place: the own INT4 caches, and with
            `state` those of the Mamba2 layers (MX8, MX4, compact MX4 or bf16) and of the convolutions
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
HQ, HKV, D = 32, 8, 128
NREP = HQ // HKV
ATT_LAYERS, MAMBA_LAYERS = 4, 24
MH, MP, MN = 128, 64, 128
CONV = (10240, 4)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LOG2E = 1.4426950408889634


def listed():
    return [
        # one user's short chat with four beams, some tokens in: latency
        dict(name="shared_p1_n4_ctx777", kind="shared", prompts=1, beams=4, prompt=777, own=18,
             group=64, mask=False, dtype="bf16"),
        # two padded prompts of different lengths, eight beams each
        dict(name="shared_mask_p2_n8_ctx4001", kind="shared", prompts=2, beams=8, prompt=4001,
             own=129, group=32, mask=True, dtype="bf16"),
        # many sampled answers to one long document
        dict(name="shared_p1_n64_ctx8192", kind="shared", prompts=1, beams=64, prompt=8192, own=200,
             group=128, mask=False, dtype="fp16"),
        # a full serving batch: eight long prompts with eight beams
        dict(name="shared_p8_n8_ctx16384", kind="shared", prompts=8, beams=8, prompt=16384, own=64,
             group=32, mask=False, dtype="bf16"),
        # one user, four beams, a small vocabulary
        dict(name="select_p1_n4_v32000", kind="select", prompts=1, beams=4, vocab=32000, num=4,
             dtype="bf16", done=0, slots=True),
        # an odd batch in fp32 with two finished beams per prompt, 2 x beams candidates
        dict(name="select_p3_n5_v50257", kind="select", prompts=3, beams=5, vocab=50257, num=10,
             dtype="fp32", done=2, slots=False),
        # the serving batch at the model's vocabulary
        dict(name="select_p8_n8_v131072", kind="select", prompts=8, beams=8, vocab=131072, num=8,
             dtype="bf16", done=0, slots=True),
        # a large batch of wide beams
        dict(name="select_p16_n16_v131072", kind="select", prompts=16, beams=16, vocab=131072,
             num=32, dtype="bf16", done=0, slots=False),
        # the attention layers' own caches alone, four beams, short answers: latency
        dict(name="reorder_kv_p1_n4", kind="reorder", prompts=1, beams=4, kept=2, own=33, group=64,
             state="none"),
        # a whole model's states, MX4 in compact tensors, eight beams of two prompts
        dict(name="reorder_mx4c_p2_n8", kind="reorder", prompts=2, beams=8, kept=5, own=129, group=32,
             state="mx4c"),
        # the bf16 states of five beams
        dict(name="reorder_bf16_p1_n5", kind="reorder", prompts=1, beams=5, kept=3, own=301, group=128,
             state="bf16"),
        # a serving batch with MX8 states
        dict(name="reorder_mx8_p4_n8", kind="reorder", prompts=4, beams=8, kept=4, own=257, group=32,
             state="mx8"),
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "select", "select", "reorder"])
    beams = _log_int(rng, 2, 32)
    if kind == "shared":
        beams = _log_int(rng, 1, 64)
        prompts = _log_int(rng, 1, max(1, min(8, 64 // beams)))
        return dict(kind=kind, prompts=prompts, beams=beams, prompt=_log_int(rng, 48, 16384),
                    own=_log_int(rng, 1, 256), group=rng.choice([32, 64, 128]),
                    mask=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "select":
        prompts = _log_int(rng, 1, 256 // beams)
        num = rng.choice([beams, beams, min(2 * beams, 64)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = (32 << 20) // (prompts * beams * (2 if dtype == "fp32" else 1))
        return dict(kind=kind, prompts=prompts, beams=beams, vocab=_log_int(rng, 999, min(most, 200000)),
                    num=num, dtype=dtype, done=rng.choice([0, 0, beams // 2]),
                    slots=num == beams and rng.random() < 0.5)
    state = rng.choice(["none", "mx4", "mx4c", "mx8", "bf16"])
    beams = _log_int(rng, 2, 16)
    return dict(kind=kind, prompts=_log_int(rng, 1, 16 // beams), beams=beams,
                kept=rng.randint(1, beams - 1), own=_log_int(rng, 1, 512), group=rng.choice([32, 64, 128]),
                state=state)


def _quantize(x, group):
    """Nibbles (uint8, even dim low) and fp32 group scales of x [..., D] in the cache's format."""
    xg = x.float().reshape(*x.shape[:-1], D // group, group)
    scale = (xg.abs().amax(-1, keepdim=True) / 7.0).clamp_min(1e-8)
    n = (xg / scale).round().clamp(-8, 7).to(torch.int32).reshape(x.shape)
    return ((n[..., 0::2] & 15) | ((n[..., 1::2] & 15) << 4)).to(torch.uint8), scale[..., 0]


def _values(packed, scale, group, dtype=torch.float32):
    """The values of an INT4 cache tensor and its scales."""
    b = packed.to(torch.int32)
    n = torch.stack((b & 15, b >> 4), -1).reshape(*packed.shape[:-1], D)
    n = torch.where(n > 7, n - 16, n).to(dtype).reshape(*packed.shape[:-1], D // group, group)
    return (n * scale.to(dtype)[..., None]).reshape(*packed.shape[:-1], D)


def _capacity(rows):
    return max(16, 1 << (rows - 1).bit_length())


def _filled_cache(gen, batch, rows, group):
    """An INT4 cache (k_packed, v_packed, k_scale, v_scale) whose first `rows` rows hold keys with a
    few large channels, and values; the rest of its capacity is zero."""
    def half(x):
        packed, scale = _quantize(x, group)
        p = torch.zeros(batch, HKV, _capacity(rows), D // 2, dtype=torch.uint8, device=DEV)
        s = torch.zeros(batch, HKV, _capacity(rows), D // group, device=DEV)
        p[:, :, :rows], s[:, :, :rows] = packed, scale
        return p, s

    k = torch.randn(batch, HKV, rows, D, device=DEV, generator=gen)
    k *= 1 + 4 * (torch.rand(1, HKV, 1, D, device=DEV, generator=gen) < 0.03)
    kp, ks = half(k)
    vp, vs = half(torch.randn(batch, HKV, rows, D, device=DEV, generator=gen))
    return [kp, vp, ks, vs]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    P, N = case["prompts"], case["beams"]
    B = P * N
    st = dict(case=case)
    if case["kind"] == "shared":
        dt, g = DTYPES[case["dtype"]], case["group"]
        st["prefix"] = _filled_cache(gen, P, case["prompt"], g)
        st["cache"] = _filled_cache(gen, B, case["own"], g)
        st["q"] = torch.randn(B, HQ, 1, D, device=DEV, generator=gen).to(dt)
        st["k"] = torch.randn(B, HKV, 1, D, device=DEV, generator=gen).to(dt)
        st["v"] = torch.randn(B, HKV, 1, D, device=DEV, generator=gen).to(dt)
        st["mask"] = None
        if case["mask"]:
            pad = torch.randint(0, case["prompt"] // 4 + 1, (P, 1, 1), device=DEV, generator=gen)
            at = torch.arange(case["prompt"] + case["own"], device=DEV)
            st["mask"] = (at >= pad).long().expand(P, N, -1).reshape(B, -1).contiguous()
    elif case["kind"] == "select":
        logits = 3 * torch.randn(B, case["vocab"], device=DEV, generator=gen)
        # tokens that the program does not allow
        banned = torch.rand(B, case["vocab"], device=DEV, generator=gen) < 0.01
        st["logits"] = logits.masked_fill(banned, -math.inf).to(DTYPES[case["dtype"]])
        st["scores"] = -40 * torch.rand(P, N, device=DEV, generator=gen)
        st["finished"] = None
        if case["done"]:
            order = torch.rand(P, N, device=DEV, generator=gen).argsort(-1)
            st["finished"] = order < case["done"]
    else:
        # `kept` beams of each prompt go on in their own places, the others' places are given to them
        order = torch.rand(P, N, device=DEV, generator=gen).argsort(-1)
        kept, free = order[:, :case["kept"]], order[:, case["kept"]:]
        beams = torch.empty(P, N, dtype=torch.int64, device=DEV)
        beams.scatter_(1, kept, kept)
        takes = torch.arange(N - case["kept"], device=DEV) % case["kept"]
        beams.scatter_(1, free, kept[:, takes])
        st["beams"] = beams
        cap, g = _capacity(case["own"]), case["group"]
        nib = lambda *s: torch.randint(0, 256, s, dtype=torch.uint8, device=DEV, generator=gen)  # noqa: E731
        pos = lambda *s: 0.5 + torch.rand(s, device=DEV, generator=gen)  # noqa: E731
        st["caches"] = [nib(ATT_LAYERS, B, HKV, cap, D // 2), nib(ATT_LAYERS, B, HKV, cap, D // 2),
                        pos(ATT_LAYERS, B, HKV, cap, D // g), pos(ATT_LAYERS, B, HKV, cap, D // g)]
        lead = (MAMBA_LAYERS, B, MH, MP)
        st["states"] = []
        if case["state"] != "none":
            st["states"].append(torch.randn(MAMBA_LAYERS, B, *CONV, device=DEV, generator=gen,
                                            dtype=torch.bfloat16))
        if case["state"] == "bf16":
            st["states"].append(torch.randn(*lead, MN, device=DEV, generator=gen, dtype=torch.bfloat16))
        elif case["state"] == "mx4c":
            st["states"] += [nib(*lead, MN // 2), nib(*lead, MN // 16), nib(*lead, MN // 16)]
        elif case["state"] in ("mx4", "mx8"):
            top = 7 if case["state"] == "mx4" else 63
            st["states"] += [torch.randint(-top, top + 1, (*lead, MN), dtype=torch.int8, device=DEV,
                                           generator=gen),
                             nib(*lead, MN // 16), nib(*lead, MN // 2) & 1]
    return st


def _run_shared(st):
    case = st["case"]
    P, N, g, lp, ls = (case[k] for k in ("prompts", "beams", "group", "prompt", "own"))
    if own:
        from layer_quant_amd import int4_8b_attention as ia

        cache = ia.Int4KVLayerCache(*st["cache"], length=ls - 1,
                                    prefix=ia.Int4KVLayerCache(*st["prefix"], length=lp))
        out = ia.shared_prefix_decode_attention(st["q"], cache, lp + ls, NREP, g, st["mask"],
                                                st["k"], st["v"])
        return dict(out=out, cache=st["cache"])
    kp, vp, ks, vs = st["cache"]
    kp[:, :, ls - 1:ls], ks[:, :, ls - 1:ls] = _quantize(st["k"], g)
    vp[:, :, ls - 1:ls], vs[:, :, ls - 1:ls] = _quantize(st["v"], g)
    pkp, pvp, pks, pvs = (t[:, :, :lp] for t in st["prefix"])
    kp, vp, ks, vs = (t[:, :, :ls] for t in st["cache"])
    q = st["q"].float().reshape(P, N, HKV, NREP, D)
    rows = q.transpose(1, 2).reshape(P, HKV, N * NREP, D)
    s0 = torch.matmul(rows, _values(pkp, pks, g).transpose(-1, -2))
    s0 = s0.reshape(P, HKV, N, NREP, lp).transpose(1, 2)
    s1 = torch.matmul(q.reshape(P * N, HKV, NREP, D), _values(kp, ks, g).transpose(-1, -2))
    s = torch.cat((s0, s1.reshape(P, N, HKV, NREP, ls)), -1) / math.sqrt(D)
    if st["mask"] is not None:
        s = s.masked_fill(st["mask"].reshape(P, N, 1, 1, -1) == 0, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    p0 = p[..., :lp].transpose(1, 2).reshape(P, HKV, N * NREP, lp)
    o0 = torch.matmul(p0, _values(pvp, pvs, g)).reshape(P, HKV, N, NREP, D).transpose(1, 2)
    o1 = torch.matmul(p[..., lp:].reshape(P * N, HKV, NREP, ls), _values(vp, vs, g))
    out = o0.reshape(P * N, HQ, D) + o1.reshape(P * N, HQ, D)
    return dict(out=out.to(st["q"].dtype), cache=st["cache"])


def _slots(beams, scores, tokens):
    """The same beams ordered by place: the best continuation of a beam keeps that beam's place, the
    others fill the free places in order."""
    P, N = beams.shape
    earlier = (beams[:, :, None] == beams[:, None, :]).tril(-1).any(-1)
    used = (beams[:, :, None] == torch.arange(N, device=beams.device)).any(1)
    free = torch.sort(used.long(), dim=1, stable=True).indices
    nth = (earlier.long().cumsum(1) - 1).clamp_min(0)
    place = torch.where(earlier, free.gather(1, nth), beams)
    at = torch.sort(place, dim=1).indices
    return scores.gather(1, at), beams.gather(1, at), tokens.gather(1, at)


def _run_select(st):
    case = st["case"]
    P, N, V, num = (case[k] for k in ("prompts", "beams", "vocab", "num"))
    if own:
        from layer_quant_amd import beam_decode as bd

        return bd.beam_select(st["logits"], st["scores"], num, finished=st["finished"], pad_token=0,
                              keep_slots=case["slots"])
    x = st["logits"].double().reshape(P, N, V)
    m = x.amax(-1, keepdim=True)
    total = st["scores"].double()[..., None] + x - (m + (x - m).exp().sum(-1, keepdim=True).log())
    if st["finished"] is not None:
        # a finished beam goes on as itself alone
        alone = torch.full((V,), -math.inf, dtype=torch.float64, device=DEV)
        alone[0] = 0
        total = torch.where(st["finished"][..., None], st["scores"].double()[..., None] + alone, total)
    best = torch.sort(total.reshape(P, N * V), dim=-1, descending=True, stable=True)
    scores, at = best.values[:, :num].float(), best.indices[:, :num]
    found = scores, at // V, at % V
    if case["slots"]:
        found = _slots(found[1], found[0], found[2])
    return found


def _run_reorder(st):
    case = st["case"]
    if own:
        from layer_quant_amd import beam_decode as bd

        caches = [t for buf in st["caches"] for t in buf.unbind(0)]
        states = [t for buf in st["states"] for t in buf.unbind(0)]
        bd.reorder_beams(caches + states, st["beams"],
                         [case["own"]] * len(caches) + [None] * len(states))
    else:
        first = torch.arange(case["prompts"], device=DEV)[:, None] * case["beams"]
        rows = (first + st["beams"]).reshape(-1)
        live = slice(None, case["own"])
        [t[:, :, :, live].copy_(t[:, rows, :, live]) for t in st["caches"]]
        [t.copy_(t[:, rows]) for t in st["states"]]
    # bytes moved as they are: equal bytes, and so equal values
    return dict(caches=st["caches"], states=st["states"])


def run(state):
    kind = state["case"]["kind"]
    return (_run_shared if kind == "shared" else _run_select if kind == "select" else _run_reorder)(state)


def work(case):
    P, N = case["prompts"], case["beams"]
    B = P * N
    if case["kind"] == "shared":
        key = HKV * (D + 2 * 4 * D // case["group"])  # bytes of a key's K and V with their scales
        total = case["prompt"] + case["own"]
        size = B * (2 * HQ * D * 2 + 2 * HKV * D * 2) + B * total * 8 * case["mask"]
        return dict(bytes=size + key * (P * case["prompt"] + B * case["own"]),
                    flops=4 * D * HQ * B * total)
    if case["kind"] == "select":
        read = P * (N - case["done"]) * case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        return dict(bytes=read * size + 4 * B + P * case["num"] * 20, flops=5 * read)
    row = ATT_LAYERS * HKV * case["own"] * (D + 2 * 4 * D // case["group"])
    if case["state"] != "none":
        per = {"mx8": 1 + 1 / 16 + 1 / 2, "mx4": 1 + 1 / 16 + 1 / 2, "mx4c": 1 / 2 + 1 / 8, "bf16": 2}
        row += MAMBA_LAYERS * (int(MH * MP * MN * per[case["state"]]) + CONV[0] * CONV[1] * 2)
    changed = N - case["kept"]
    return dict(bytes=P * row * (changed + min(changed, case["kept"])) + 8 * B, flops=0)


def exact(case, seed):
    st = prepare(case, seed)
    P, N = case["prompts"], case["beams"]
    if case["kind"] == "shared":
        g, lp, ls = case["group"], case["prompt"], case["own"]
        for i, x in ((0, st["k"]), (1, st["v"])):
            st["cache"][i][:, :, ls - 1:ls], st["cache"][i + 2][:, :, ls - 1:ls] = _quantize(x, g)
        outs = []
        for b in range(P * N):
            pre, suf = [t[b // N, :, :lp] for t in st["prefix"]], [t[b, :, :ls] for t in st["cache"]]
            k, v = (torch.cat((_values(pre[i], pre[i + 2], g, torch.float64),
                               _values(suf[i], suf[i + 2], g, torch.float64)), 1) for i in (0, 1))
            q = st["q"][b, :, 0].double().reshape(HKV, NREP, D)
            s = torch.einsum("hrd,hkd->hrk", q, k) * (LOG2E / math.sqrt(D))
            if st["mask"] is not None:
                s = s + torch.where(st["mask"][b] != 0, 0.0, -math.inf)
            w = torch.exp2(s - s.max(-1, keepdim=True).values)
            outs.append((torch.einsum("hrk,hkd->hrd", w, v) / w.sum(-1, keepdim=True)).reshape(HQ, D))
        return dict(out=torch.stack(outs), cache=[None, None, st["cache"][2].double(), st["cache"][3].double()])
    if case["kind"] == "select":
        x = st["logits"].double().cpu().numpy().reshape(P, N, -1)
        base = st["scores"].double().cpu().numpy()
        done = None if st["finished"] is None else st["finished"].cpu().numpy()
        scores = np.zeros((P, case["num"]))
        for p in range(P):
            pool = []
            for n in range(N):
                if done is not None and done[p, n]:
                    pool.append((-base[p, n], n, 0))
                    continue
                row = x[p, n]
                top = row.max()
                norm = top + np.log(np.sum(np.exp(row - top)))
                at = np.lexsort((np.arange(row.size), -row))[:case["num"]] if row.size < 4096 else None
                if at is None:
                    some = np.flatnonzero(row >= np.partition(row, -case["num"])[-case["num"]])
                    at = some[np.lexsort((some, -row[some]))][:case["num"]]
                pool += [(-(base[p, n] + row[t] - norm), n, int(t)) for t in at]
            pool = sorted(pool)[:case["num"]]
            if case["slots"]:
                places = [None] * N
                rest = []
                for c in pool:
                    if places[c[1]] is None:
                        places[c[1]] = c
                    else:
                        rest.append(c)
                pool = [c if c is not None else rest.pop(0) for c in places]
            scores[p] = [-c[0] for c in pool]
        return torch.from_numpy(scores), None, None
    beams = st["beams"].cpu().tolist()

    def moved(t, rows=None):
        if not t.is_floating_point():
            return None
        out = t.double()
        for p in range(P):
            for n in range(N):
                to, frm = out[:, p * N + n], t[:, p * N + beams[p][n]].double()
                if rows is None:
                    to.copy_(frm)
                else:
                    to[:, :, :rows].copy_(frm[:, :, :rows])
        return out

    return dict(caches=[moved(t, case["own"]) for t in st["caches"]],
                states=[moved(t) for t in st["states"]])
