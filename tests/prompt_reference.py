"""The prompt operators in 64 bits, from their definitions, with the magnitudes that their error bounds
are made of."""
import math

import torch


def spans(starts, rows):
    s = [int(v) for v in starts]
    return [(a, b) for a, b in zip(s, s[1:])], (s[0], s[-1], rows)


def attention(q, k, v, starts, scale=None):
    """(out, sum of weight * |value|, largest sum of |q k| * scale) of packed q [T, Hq, D], float64.
    Rows of no prompt are zero; what is masked is not read."""
    q, k, v = (t.double().cpu() for t in (q, k, v))
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    rep = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    out, weight, score = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[:2]).double()
    for a, b in spans(starts, q.shape[0])[0]:
        for t in range(a, b):
            s = (k[a:t + 1] * q[t]).sum(-1) * scale
            p = torch.softmax(s, 0)[..., None]
            out[t] = (p * v[a:t + 1]).sum(0)
            weight[t] = (p * v[a:t + 1].abs()).sum(0)
            score[t] = ((k[a:t + 1] * q[t]).abs().sum(-1) * abs(scale)).amax(0)
    return out, weight, score


def attention_bound(ref, weight, score, dtype, head_dim):
    """|out - ref| at most: the output's rounding and the weights' (each half a step of the type); a
    score is off by less than (D + 2) 2^-23 of its terms' sum (products exact or rounded once, fp32
    sums in any order) and the exponential's argument and value by 2^-22 of what they are, which moves a
    weight, and the weights' sum, by that much."""
    half = torch.finfo(dtype).eps / 2
    moved = ((head_dim + 2) * 2.0 ** -23 * score + (score + 1) * 2.0 ** -21)[..., None]
    least = torch.finfo(dtype).tiny * half  # half a step below the smallest normal number
    return half * ref.abs() + (half + 2 * moved + 2.0 ** -18) * weight + least


def softplus(x):
    return x.clamp_min(0) + torch.log1p(torch.exp(-x.abs()))


def scan(x, dt, A, B, C, starts, D=None, z=None, dt_bias=None, dt_softplus=False,
         dt_limit=(0.0, math.inf), initial=None):
    """(y, states, |y|'s terms, |states|' terms) of packed x [T, H, P], float64."""
    f = lambda t: None if t is None else t.double().cpu()  # noqa: E731
    x, dt, A, B, C, D, z, bias, initial = map(f, (x, dt, A, B, C, D, z, dt_bias, initial))
    if bias is not None:
        dt = dt + bias
    if dt_softplus:
        dt = softplus(dt)
    dt = dt.clamp(*dt_limit)
    rep = x.shape[1] // B.shape[1]
    B, C = B.repeat_interleave(rep, 1), C.repeat_interleave(rep, 1)
    S = len(starts) - 1
    shape = (S, x.shape[1], x.shape[2], B.shape[2])
    state = torch.zeros(shape).double() if initial is None else initial.clone()
    size = state.abs()
    y, wy = torch.zeros_like(x), torch.zeros_like(x)
    for i, (a, b) in enumerate(spans(starts, x.shape[0])[0]):
        for t in range(a, b):
            keep = torch.exp(A * dt[t])[:, None, None]
            dx = (dt[t][:, None] * x[t])[:, :, None]
            state[i] = state[i] * keep + dx * B[t][:, None]
            size[i] = size[i] * keep + dx.abs() * B[t].abs()[:, None]
            y[t] = (state[i] * C[t][:, None]).sum(-1)
            wy[t] = (size[i] * C[t].abs()[:, None]).sum(-1)
            if D is not None:
                y[t] += D[:, None] * x[t]
                wy[t] += (D[:, None] * x[t]).abs()
            if z is not None:
                gate = z[t] / (1 + torch.exp(-z[t]))
                y[t] *= gate
                wy[t] *= gate.abs()
    return y, state, wy, size


def logprobs(logits, tokens):
    """(logprob of each row's token, entropy, log-softmax) of logits [R, V] in float64."""
    x = logits.double().cpu()
    lp = torch.log_softmax(x, -1)
    tokens = tokens.cpu()
    given = (tokens >= 0) & (tokens < x.shape[1])
    at = lp.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    p = lp.exp()
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    entropy = torch.where(torch.isnan(lp).any(-1), torch.nan, entropy)
    return torch.where(given, at, torch.zeros_like(at)), entropy, lp
