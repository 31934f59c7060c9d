"""Performance cases of prompts and their scores: packed prompts through the hybrid model's two mixers,
and the log-probabilities of given tokens.

Geometry is the 8B model's: attention with 32 query and 8 KV heads of 128 dims, Mamba2 layers of 128
heads x 64 with a state of 128 and 8 groups, vocabularies of 32000 to 131072 tokens; `small` is the
test model's (8 query and 2 KV heads; 8 Mamba2 heads x 16, a state of 32, 2 groups).

Kinds of case
  attention  causal attention of whole prompts over their own keys: one prompt [1, L, heads, dim], or
             `seqs` prompts of different lengths packed one behind another
  scan       the Mamba2 recurrence over whole prompts from the state before them: y, and the state
             behind each prompt. x, B and C are views of one tensor, as the convolution leaves them
  scores     log-probability of each row's token, the row's entropy and its `top` likeliest tokens
"""
from __future__ import annotations

import math
import random

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# query heads, KV heads, head_dim
ATTENTION = {"8b": (32, 8, 128), "small": (8, 2, 128)}
# heads, head_dim, state, groups
MAMBA = {"8b": (128, 64, 128, 8), "small": (8, 16, 32, 2)}
CHUNK = 64  # of the plain scan


def listed():
    return [
        # one user's short question: latency
        dict(name="attention_l333", kind="attention", seqs=1, longest=333, mix=0, model="8b",
             dtype="bf16"),
        # texts of a scoring batch, none to 700 tokens, packed
        dict(name="attention_s24_l700_fp16", kind="attention", seqs=24, longest=700, mix=1, model="8b",
             dtype="fp16"),
        # a long document
        dict(name="attention_l16384", kind="attention", seqs=1, longest=16384, mix=0, model="8b",
             dtype="bf16"),
        # an fp32 check run of three texts
        dict(name="attention_s3_l1001_fp32", kind="attention", seqs=3, longest=1001, mix=2, model="8b",
             dtype="fp32"),
        # one user's short question: latency
        dict(name="scan_l200", kind="scan", seqs=1, longest=200, mix=0, model="8b", dtype="bf16",
             initial=False, state="bf16", gate=False),
        # texts of a scoring batch behind a state each, packed
        dict(name="scan_s24_l700", kind="scan", seqs=24, longest=700, mix=1, model="8b", dtype="bf16",
             initial=True, state="fp32", gate=False),
        # a long document
        dict(name="scan_l16384", kind="scan", seqs=1, longest=16384, mix=0, model="8b", dtype="bf16",
             initial=False, state="bf16", gate=False),
        # an fp32 check run of three texts, gated
        dict(name="scan_s3_l1001_fp32", kind="scan", seqs=3, longest=1001, mix=2, model="8b",
             dtype="fp32", initial=True, state="fp32", gate=True),
        # a decode step of one user with the five likeliest tokens
        dict(name="scores_t1_v32000", kind="scores", rows=1, vocab=32000, top=5, dtype="bf16"),
        # a short text in fp32, an odd vocabulary
        dict(name="scores_t37_v50257_fp32", kind="scores", rows=37, vocab=50257, top=20, dtype="fp32"),
        # a decode step of the serving batch at the model's vocabulary
        dict(name="scores_t64_v131072", kind="scores", rows=64, vocab=131072, top=8, dtype="bf16"),
        # a window of a text that is scored
        dict(name="scores_t2048_v131072", kind="scores", rows=2048, vocab=131072, top=0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "scan", "scores"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "scores":
        rows = _log_int(rng, 1, 2048)
        most = (256 << 20) // (rows * (2 if dtype == "fp32" else 1))
        return dict(kind=kind, rows=rows, vocab=_log_int(rng, 999, min(most, 200000)),
                    top=rng.choice([0, rng.randint(1, 8), rng.randint(1, 32)]), dtype=dtype)
    seqs = rng.choice([1, 1, _log_int(rng, 2, 32)])
    model = rng.choice(["8b", "8b", "8b", "small"])
    case = dict(kind=kind, seqs=seqs, mix=rng.randrange(1 << 20), model=model, dtype=dtype)
    if kind == "attention":
        most = int((2048 if dtype == "fp32" else 16384) / math.sqrt(seqs))
        return dict(case, longest=_log_int(rng, 1, most))
    return dict(case, longest=_log_int(rng, 1, (2048 if dtype == "fp32" else 16384) // seqs),
                initial=rng.random() < 0.5, state=rng.choice(["fp32", "bf16"]), gate=rng.random() < 0.25)


def _lengths(case):
    """The prompts' lengths: the longest one, the others spread over their logarithm, and where there
    are many of them an empty one."""
    rng = random.Random(case["mix"])
    lengths = [case["longest"]] + [_log_int(rng, 1, case["longest"]) for _ in range(case["seqs"] - 1)]
    if case["seqs"] >= 8:
        lengths[-1] = 0
    rng.shuffle(lengths)
    return lengths


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device=DEV, generator=gen)

    def rand(*shape):
        return torch.rand(shape, device=DEV, generator=gen)

    dtype = DTYPES[case["dtype"]]
    st = dict(case=case)
    if case["kind"] == "scores":
        rows, vocab = case["rows"], case["vocab"]
        logits = 3 * randn(rows, vocab)
        # tokens that the program does not allow
        logits = logits.masked_fill(rand(rows, vocab) < 0.01, -math.inf).to(dtype)
        # a text's tokens are mostly likely ones; a few rows have none to be scored
        likely = torch.topk(logits.float(), 64).indices.gather(
            1, torch.randint(0, 64, (rows, 1), device=DEV, generator=gen))[:, 0]
        any_ = torch.randint(0, vocab, (rows,), device=DEV, generator=gen)
        any_ = torch.where(torch.isinf(logits.gather(1, any_[:, None])[:, 0]), likely, any_)
        tokens = torch.where(rand(rows) < 0.3, any_, likely)
        if rows > 16:
            tokens = tokens.masked_fill(rand(rows) < 0.05, -100)
        return dict(st, logits=logits, tokens=tokens)
    lengths = _lengths(case)
    total = sum(lengths)
    lead = (total,) if case["seqs"] > 1 else (1, total)
    st["starts"] = None
    if case["seqs"] > 1:
        ends = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
        st["starts"] = torch.tensor(ends, dtype=torch.int32, device=DEV)
    if case["kind"] == "attention":
        hq, hkv, d = ATTENTION[case["model"]]
        # keys with a few large channels, as the model has them
        k = randn(*lead, hkv, d) * (1 + 4 * (rand(hkv, d) < 0.03))
        return dict(st, q=randn(*lead, hq, d).to(dtype), k=k.to(dtype), v=randn(*lead, hkv, d).to(dtype))
    h, p, n, g = MAMBA[case["model"]]
    xbc = F.silu(randn(*lead, h * p + 2 * g * n)).to(dtype)
    st["x"] = xbc[..., :h * p].unflatten(-1, (h, p))
    st["B"] = xbc[..., h * p:h * p + g * n].unflatten(-1, (g, n))
    st["C"] = xbc[..., h * p + g * n:].unflatten(-1, (g, n))
    st["dt"] = randn(*lead, h).to(dtype)
    # softplus(dt_bias) between 0.001 and 0.1, as such models begin with
    first = torch.exp(math.log(0.001) + math.log(100) * rand(h))
    st["dt_bias"] = first + torch.log(-torch.expm1(-first))
    st["A"] = -(1 + 15 * rand(h))
    st["D"] = randn(h)
    st["z"] = randn(*lead, h, p).to(dtype) if case["gate"] else None
    shape = (case["seqs"], h, p, n)
    st["initial"] = 0.5 * randn(*shape).to(DTYPES[case["state"]]) if case["initial"] else None
    st["states"] = torch.empty(shape, device=DEV, dtype=DTYPES[case["state"]])
    return st


def _places(st, device=DEV):
    """Where the rows are that stand at place l of sequence s ([S, longest], any row where there is
    none), which places hold one, and each row's sequence and place."""
    case = st["case"]
    starts = st["starts"]
    if starts is None:
        starts = torch.tensor([0, case["longest"]], dtype=torch.int32, device=device)
    starts = starts.long()
    total = sum(_lengths(case))
    at = torch.arange(case["longest"], device=device)
    there = at < (starts[1:] - starts[:-1])[:, None]
    rows = (starts[:-1, None] + at).clamp_max(total - 1)
    row = torch.arange(total, device=device)
    seq = torch.searchsorted(starts, row, right=True) - 1
    return rows, there, seq, row - starts[seq]


def _packed(t):
    return t if t.dim() == 3 else t.flatten(0, 1)


def _run_attention(st):
    if own:
        from layer_quant_amd import prompts

        return prompts.prompt_attention(st["q"], st["k"], st["v"], st["starts"])
    q, k, v = (_packed(st[i]) for i in "qkv")
    hq, hkv, d = ATTENTION[st["case"]["model"]]
    rows, there, seq, place = _places(st)
    S, L = rows.shape
    # [S, KV head, query head of it x place, dim] against [S, KV head, dim, place]
    qf = q[rows].float().reshape(S, L, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(S, hkv, -1, d)
    kf = k[rows].float().permute(0, 2, 3, 1).contiguous()
    vf = v[rows].float().transpose(1, 2).contiguous()
    s = torch.matmul(qf * (1 / math.sqrt(d)), kf).reshape(S, hkv, hq // hkv, L, L)
    s.masked_fill_(torch.ones(L, L, dtype=torch.bool, device=q.device).triu(1), -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    s.div_(s.sum(-1, keepdim=True))
    o = torch.matmul(s.reshape(S, hkv, -1, L), vf).reshape(S, hq, L, d)
    return o[seq, :, place].to(q.dtype).reshape(st["q"].shape)


def _run_scan(st):
    case = st["case"]
    if own:
        from layer_quant_amd import prompts

        return prompts.prompt_scan(st["x"], st["dt"], st["A"], st["B"], st["C"], st["starts"], D=st["D"],
                                   z=st["z"], dt_bias=st["dt_bias"], dt_softplus=True,
                                   initial_states=st["initial"], states=st["states"])
    x, B, C = (_packed(st[i]) for i in ("x", "B", "C"))
    h, p, n, g = MAMBA[case["model"]]
    raw = st["dt"].reshape(-1, h)
    rows, there, seq, place = _places(st)
    pad = -rows.shape[1] % CHUNK
    rows, there = F.pad(rows, (0, pad)), F.pad(there, (0, pad))
    S, nc = rows.shape[0], rows.shape[1] // CHUNK
    rows = rows.reshape(S, nc, CHUNK)
    dt = F.softplus(raw.float() + st["dt_bias"])[rows] * there.reshape(S, nc, CHUNK, 1)
    # [S, chunk, head, place]: steps, and the logarithm of the decay since the chunk's beginning
    dt = dt.transpose(2, 3)
    cum = (st["A"].double()[:, None] * dt.double()).cumsum(-1)
    total = cum[..., -1]
    xf = x[rows].float().permute(0, 1, 3, 2, 4)  # [S, chunk, head, place, p]
    Bf = B[rows].float().permute(0, 1, 3, 2, 4)  # [S, chunk, group, place, n]
    Cf = C[rows].float().permute(0, 1, 3, 2, 4)
    # within a chunk
    later = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=x.device).triu(1)
    decay = (cum[..., :, None] - cum[..., None, :]).float().masked_fill_(later, -math.inf).exp_()
    mix = torch.matmul(Cf, Bf.transpose(-1, -2).contiguous())[:, :, :, None]
    mix = decay.reshape(S, nc, g, h // g, CHUNK, CHUNK) * mix
    mix = mix.reshape(S, nc, h, CHUNK, CHUNK) * dt[..., None, :]
    y = torch.matmul(mix, xf)
    # what each chunk adds to the state, and the state before each chunk and behind the last one
    weight = (total[..., None] - cum).float().exp() * dt
    xw = (xf * weight[..., None]).transpose(-1, -2).contiguous().reshape(S, nc, g, -1, CHUNK)
    added = torch.matmul(xw, Bf).reshape(S, nc, h, p * n)
    before = torch.zeros(S, 1, h, p * n, device=x.device)
    if st["initial"] is not None:
        before = st["initial"].float().reshape(S, 1, h, p * n)
    terms = torch.cat((before, added), 1).transpose(1, 2).contiguous()  # [S, head, 1 + chunk, p n]
    upto = F.pad(total.transpose(1, 2).cumsum(-1), (1, 0))  # [S, head, 1 + chunk]
    over = torch.ones(nc + 1, nc + 1, dtype=torch.bool, device=x.device).triu(1)
    carry = (upto[..., :, None] - upto[..., None, :]).float().masked_fill_(over, -math.inf).exp_()
    held = torch.matmul(carry, terms).transpose(1, 2).reshape(S, nc + 1, h, p, n)
    back = held[:, :-1].reshape(S, nc, g, -1, n).transpose(-1, -2).contiguous()
    away = torch.matmul(Cf, back).reshape(S, nc, g, CHUNK, h // g, p).permute(0, 1, 2, 4, 3, 5)
    y = y + away.reshape(S, nc, h, CHUNK, p) * cum.float().exp()[..., None]
    y = y.transpose(2, 3).reshape(S, nc * CHUNK, h, p)[seq, place]
    y = y + st["D"][:, None] * x.float()
    if st["z"] is not None:
        zf = _packed(st["z"]).float()
        y = y * (zf * torch.sigmoid(zf))
    st["states"].copy_(held[:, -1])
    return y.to(x.dtype).reshape(st["x"].shape), st["states"]


def _run_scores(st):
    top, vocab = st["case"]["top"], st["case"]["vocab"]
    if own:
        from layer_quant_amd import prompts

        found = prompts.token_logprobs(st["logits"], st["tokens"], top)
        return tuple(found) if top else (found.logprobs, found.entropy)
    x, tokens = st["logits"].float(), st["tokens"]
    z = x - x.amax(-1, keepdim=True)
    e = z.exp()
    total = e.sum(-1, keepdim=True)
    logprob = z - total.log()
    scored = (tokens >= 0) & (tokens < vocab)
    at = logprob.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0]
    at = torch.where(scored, at, torch.zeros_like(at))
    entropy = -(torch.where(e > 0, e * logprob, torch.zeros_like(e)) / total).sum(-1)
    if not top:
        return at, entropy
    # values in order as whole numbers, the lower token ahead among equal ones
    bits = z.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    ids = torch.arange(vocab, device=x.device)
    best = torch.topk(order * (1 << 20) - ids, top).indices
    return at, entropy, logprob.gather(1, best), best


def run(state):
    kind = state["case"]["kind"]
    return (_run_attention if kind == "attention" else _run_scan if kind == "scan" else _run_scores)(state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "scores":
        rows, vocab = case["rows"], case["vocab"]
        return dict(bytes=rows * vocab * size + rows * (16 + 12 * case["top"]), flops=6 * rows * vocab)
    lengths = _lengths(case)
    total = sum(lengths)
    if case["kind"] == "attention":
        hq, hkv, d = ATTENTION[case["model"]]
        return dict(bytes=total * (2 * hq + 2 * hkv) * d * size,
                    flops=4 * d * hq * sum(n * (n + 1) // 2 for n in lengths))
    h, p, n, g = MAMBA[case["model"]]
    states = case["seqs"] * h * p * n * (4 if case["state"] == "fp32" else 2) * (1 + case["initial"])
    return dict(bytes=total * ((2 + case["gate"]) * h * p + 2 * g * n + h) * size + states,
                flops=4 * h * p * n * total)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "scores":
        outs, parts = [], 128
        for at in range(0, case["rows"], parts):
            x, tok = st["logits"][at:at + parts].double(), st["tokens"][at:at + parts]
            lp = torch.log_softmax(x, -1)
            given = torch.where(tok >= 0, lp.gather(1, tok.clamp_min(0)[:, None])[:, 0], 0.0)
            entropy = -torch.nan_to_num(lp.exp() * lp, nan=0.0).sum(-1)
            outs.append((given, entropy, torch.sort(lp, -1, descending=True).values[:, :case["top"]]))
        given, entropy, best = (torch.cat(o) for o in zip(*outs))
        return (given, entropy, best, None) if case["top"] else (given, entropy)
    ends = [0]
    for length in _lengths(case):
        ends.append(ends[-1] + length)
    if case["kind"] == "attention":
        hq, hkv, d = ATTENTION[case["model"]]
        q, k, v = (st[i].reshape(-1, st[i].shape[-2], d) for i in "qkv")
        out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
        for a, b in zip(ends, ends[1:]):
            for head in range(hq if b > a else 0):
                kk, vv = (t[a:b, head * hkv // hq].double() for t in (k, v))
                for r in range(a, b, 4096):
                    to = min(b, r + 4096)
                    s = q[r:to, head].double() @ kk[:to - a].T.contiguous() * d ** -0.5
                    ahead = torch.arange(a, to, device=DEV) > torch.arange(r, to, device=DEV)[:, None]
                    out[r:to, head] = torch.softmax(s.masked_fill(ahead, -math.inf), -1) @ vv[:to - a]
        return out.reshape(st["q"].shape)
    h, p, n, g = MAMBA[case["model"]]
    x, dt = (st[i].reshape(ends[-1], h, -1).double() for i in ("x", "dt"))
    B, C = (st[i].reshape(ends[-1], g, n) for i in ("B", "C"))
    dt = dt[..., 0] + st["dt_bias"].double()
    dt = dt.clamp_min(0) + torch.log1p(torch.exp(-dt.abs()))
    decay = torch.exp(st["A"].double() * dt)
    first = torch.tensor(ends[:-1], device=DEV)
    length = torch.tensor(ends[1:], device=DEV) - first
    state = torch.zeros(case["seqs"], h, p, n, dtype=torch.float64, device=DEV)
    if st["initial"] is not None:
        state.copy_(st["initial"])
    y = torch.empty(ends[-1] + 1, h, p, dtype=torch.float64, device=DEV)
    zeros = torch.zeros((), dtype=torch.float64, device=DEV)
    for step in range(case["longest"]):
        # a sequence that has ended keeps its state; what it would give goes behind the last row
        on = step < length
        row = torch.where(on, first + step, 0)
        live = on[:, None]
        a = torch.where(live, decay[row], zeros + 1)
        dx = torch.where(live, dt[row], zeros)[..., None] * x[row]
        Bt, Ct = (t[row].double().repeat_interleave(h // g, 1) for t in (B, C))
        state.mul_(a[..., None, None]).addcmul_(dx[..., None], Bt[:, :, None])
        y[torch.where(on, row, ends[-1])] = torch.matmul(state, Ct[..., None])[..., 0]
    y = y[:-1] + st["D"].double()[:, None] * x
    if st["z"] is not None:
        z = st["z"].reshape(y.shape).double()
        y = y * z / (1 + torch.exp(-z))
    return y.reshape(st["x"].shape), state
