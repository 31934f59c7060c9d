"""The prompt operators as a user runs them: packed texts through hybrid layers to their scores, decode
steps from the states they leave, captured and replayed, on other streams, in the patched model."""
import threading

import pytest
import torch
import torch.nn.functional as F

import fake_nemotron as fake
import prompt_reference as ref
from layer_quant_amd import int4_8b_attention as ia
from layer_quant_amd import mamba_state_8b_kernel as ms
from layer_quant_amd import nemotron_8b_decode_eval as de
from layer_quant_amd import prompts

pytestmark = pytest.mark.gpu


def model_of(gpu, dtype, **config):
    torch.manual_seed(0)
    cfg = fake.make_config(hybrid_override_pattern="M*M", num_attention_heads=4, num_key_value_heads=2,
                           head_dim=64, mamba_num_heads=8, mamba_head_dim=64, ssm_state_size=128,
                           n_groups=2, vocab_size=300, **config)
    return fake.FakeNemotronHForCausalLM(cfg).to(gpu, dtype).eval()


def mixer_inputs(mixer, h):
    """x, dt, B, C of a Mamba2 mixer's projection of h [..., hidden], as views of it."""
    inner, gn = mixer.num_heads * mixer.head_dim, mixer.n_groups * mixer.ssm_state_size
    x, B, C, dt = mixer.in_proj(h).split([inner, gn, gn, mixer.num_heads], -1)
    return (x.unflatten(-1, (mixer.num_heads, -1)), dt, B.unflatten(-1, (mixer.n_groups, -1)),
            C.unflatten(-1, (mixer.n_groups, -1)))


@torch.no_grad()
def packed_forward(model, ids, starts):
    """Logits of packed ids [T], and each Mamba2 layer's states and each attention layer's K and V."""
    h = model.backbone.embeddings(ids)
    held = []
    for block in model.backbone.layers:
        y, mixer = block.norm(h), block.mixer
        if block.block_type == "mamba":
            x, dt, B, C = mixer_inputs(mixer, y)
            y, states = prompts.prompt_scan(x, dt, -torch.exp(mixer.A_log.float()), B, C, starts,
                                            D=mixer.D, dt_bias=mixer.dt_bias, dt_softplus=True)
            held.append(states)
            y = mixer.out_proj(y.flatten(1))
        else:
            q, k, v = (p(y).unflatten(-1, (-1, mixer.head_dim))
                       for p in (mixer.q_proj, mixer.k_proj, mixer.v_proj))
            held.append((k, v))
            y = mixer.o_proj(prompts.prompt_attention(q, k, v, starts).flatten(1))
        h = h + y
    return model.lm_head(h), held


@torch.no_grad()
def reference_forward(model, ids):
    """Logits of one text in 64 bits on the CPU."""
    m = model.double().cpu()
    h = m.backbone.embeddings(ids.cpu())
    for block in m.backbone.layers:
        y, mixer = block.norm(h), block.mixer
        if block.block_type == "mamba":
            x, dt, B, C = mixer_inputs(mixer, y)
            y = ref.scan(x, dt, -torch.exp(mixer.A_log), B, C, [0, len(ids)], D=mixer.D,
                         dt_bias=mixer.dt_bias, dt_softplus=True)[0]
            y = mixer.out_proj(y.flatten(1))
        else:
            q, k, v = (p(y).unflatten(-1, (-1, mixer.head_dim))
                       for p in (mixer.q_proj, mixer.k_proj, mixer.v_proj))
            y = mixer.o_proj(ref.attention(q, k, v, [0, len(ids)])[0].flatten(1))
        h = h + y
    return m.lm_head(h)


def texts_of(gpu, lengths, vocab=300, seed=1):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    ids = torch.randint(0, vocab, (sum(lengths),), device=gpu, generator=gen)
    ends = torch.tensor([0, *lengths], device=gpu).cumsum(0)
    return ids, ends


def next_tokens(ids, starts):
    """Each row's next token, -100 at the texts' ends."""
    nxt = torch.cat((ids[1:], ids.new_full((1,), -100)))
    ends = starts[1:][starts[1:] > starts[:-1]] - 1
    return nxt.index_fill(0, ends, -100)


def test_packed_texts_to_scores(gpu):
    """fp32: the scores of texts of 1 to 150 tokens, and of none, against each one alone in 64 bits."""
    model = model_of(gpu, torch.float32)
    lengths = [40, 1, 0, 150, 66]
    ids, starts = texts_of(gpu, lengths)
    logits, _ = packed_forward(model, ids, starts)
    scores = prompts.token_logprobs(logits, next_tokens(ids, starts), 3)
    s = starts.tolist()
    for a, b in zip(s, s[1:]):
        if a == b:
            continue
        want = reference_forward(model, ids[a:b])
        lp = torch.log_softmax(want, -1)
        got = scores.logprobs[a:b].double().cpu()
        assert got[-1] == 0
        given = lp[:-1].gather(1, ids[a + 1:b, None].cpu())[:, 0]
        assert torch.allclose(got[:-1], given, atol=2e-4)
        assert torch.allclose(scores.entropy[a:b].double().cpu(), -(lp.exp() * lp).sum(-1), atol=2e-4)
        assert torch.allclose(scores.top_logprobs[a:b].double().cpu(), lp.topk(3).values, atol=2e-4)
        model.to(gpu, torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_packed_is_each_alone(gpu, dtype):
    """A text's rows, states and scores do not depend on what it is packed with, bit for bit."""
    gen = torch.Generator(device=gpu).manual_seed(2)
    lengths = [70, 3, 0, 200, 1, 129]
    _, starts = texts_of(gpu, lengths)
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen).to(dtype)  # noqa: E731
    total = sum(lengths)
    q, k, v = randn(total, 8, 128), randn(total, 2, 128), randn(total, 2, 128)
    x, dt, B, C = randn(total, 8, 64), randn(total, 8), randn(total, 2, 128), randn(total, 2, 128)
    A, initial = -torch.rand(8, device=gpu, generator=gen), randn(len(lengths), 8, 64, 128)
    logits, tokens = randn(total, 500), torch.randint(0, 500, (total,), device=gpu, generator=gen)
    out = prompts.prompt_attention(q, k, v, starts)
    y, states = prompts.prompt_scan(x, dt, A, B, C, starts, dt_softplus=True, initial_states=initial)
    scores = prompts.token_logprobs(logits, tokens, 5)
    s = starts.tolist()
    for i, (a, b) in enumerate(zip(s, s[1:])):
        one = slice(a, b)
        assert torch.equal(out[one], prompts.prompt_attention(q[None, one], k[None, one], v[None, one])[0])
        y1, s1 = prompts.prompt_scan(x[None, one], dt[None, one], A, B[None, one], C[None, one],
                                     dt_softplus=True, initial_states=initial[i:i + 1])
        assert torch.equal(y[one], y1[0]) and torch.equal(states[i], s1[0])
        for got, alone in zip(scores, prompts.token_logprobs(logits[one], tokens[one], 5)):
            assert torch.equal(got[one], alone)


def test_decode_from_the_states(gpu):
    """Prompts, then a token each: the states go on in the selective-state update and in MX8, K and V in
    an INT4 cache."""
    model = model_of(gpu, torch.bfloat16)
    lengths = [65, 30]
    ids, starts = texts_of(gpu, lengths, seed=3)
    more = torch.tensor([5, 7], device=gpu)
    longer = torch.cat((ids[:65], more[:1], ids[65:], more[1:]))
    later = torch.tensor([0, 66, 97], device=gpu)
    _, held = packed_forward(model, ids, starts)
    _, want = packed_forward(model, longer, later)
    block = model.backbone.layers[0]
    mixer = block.mixer
    wide = lambda t: t[:, None].expand(-1, mixer.head_dim)  # noqa: E731
    with torch.no_grad():
        x, dt, B, C = mixer_inputs(mixer, block.norm(model.backbone.embeddings(more)))
        args = (x, dt[..., None].expand_as(x), (-torch.exp(mixer.A_log.float()))[:, None, None].expand(
            -1, mixer.head_dim, mixer.ssm_state_size), B, C, wide(mixer.D))
        state = held[0].clone()
        ms.selective_state_update(state, *args, dt_bias=wide(mixer.dt_bias), dt_softplus=True)
        assert (state - want[0]).norm() <= 2e-3 * want[0].norm()
        cache = ms.allocate_state_kernel_cache(held[0])
        ms.mx_state_selective_update(cache, *args, dt_bias=wide(mixer.dt_bias), dt_softplus=True)
        # an MX8 value is off by a 64th of its block's largest, twice
        mx = ms.dequantize_state_cache(cache)
        assert (mx - want[0]).norm() <= 0.05 * want[0].norm()
    k, v = held[1]
    holder = type("Cache", (), {})()
    layer = ia._ensure_layer_cache(holder, 1, 1, 2, 65, 64, 32, gpu)
    rows = [t[:65].transpose(0, 1)[None] for t in (k, v)]
    ia._pack_kv_into_cache(layer, *rows, torch.arange(65, device=gpu), 32)
    assert layer.length == 65


def test_captured_calls_take_the_starts_of_the_replay(gpu):
    """One graph of the three calls, replayed with other texts and lengths behind eager work on the same
    stream and scratch, against eager calls."""
    gen = torch.Generator(device=gpu).manual_seed(4)
    total, h = 1500, 8
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen)  # noqa: E731
    starts = torch.zeros(4, dtype=torch.int32, device=gpu)
    q, k, v = (randn(total, n, 128).bfloat16() for n in (8, 2, 2))
    x, dt = randn(total, h, 64).bfloat16(), randn(total, h)
    B, C = randn(total, 2, 128).bfloat16(), randn(total, 2, 128).bfloat16()
    A, logits = -torch.rand(h, device=gpu, generator=gen), randn(40, 40000)
    tokens = torch.randint(0, 40000, (40,), device=gpu, generator=gen)

    def calls():
        return (prompts.prompt_attention(q, k, v, starts),
                *prompts.prompt_scan(x, dt, A, B, C, starts, dt_softplus=True),
                *prompts.token_logprobs(logits, tokens, 4))

    sets = [[0, 700, 700, 1500], [3, 4, 900, 1400], [0, 0, 0, 0], [0, 1500, 1500, 1500], [10, 20, 30, 40]]
    starts.copy_(torch.tensor(sets[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = calls()
    for i, s in enumerate(sets * 2):
        starts.copy_(torch.tensor(s))
        for t in (q, x, logits):
            t.copy_(torch.randn(t.shape, device=gpu, generator=gen))
        want = [t.clone() for t in calls()]
        prompts.prompt_scan(x.repeat(3, 1, 1), dt.repeat(3, 1), A, B.repeat(3, 1, 1), C.repeat(3, 1, 1),
                            torch.tensor([0, 4500], device=gpu))  # grows the eager scratch
        torch.cuda.synchronize()
        for t in held:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(held, want):
            assert torch.equal(got, w), i


def test_streams_and_threads(gpu):
    """Calls of several threads, on one stream and on streams of their own, at once."""
    gen = torch.Generator(device=gpu).manual_seed(5)
    randn = lambda *s: torch.randn(*s, device=gpu, generator=gen)  # noqa: E731
    cases = []
    for rows in (600, 900, 1300, 2000):
        x, dt = randn(rows, 8, 64).bfloat16(), randn(rows, 8)
        B, C = randn(rows, 2, 128).bfloat16(), randn(rows, 2, 128).bfloat16()
        cases.append((x, dt, -torch.rand(8, device=gpu, generator=gen), B, C,
                      torch.tensor([0, rows], device=gpu), randn(8, 33000 + rows)))
    run = lambda c: (*prompts.prompt_scan(*c[:6], dt_softplus=True),  # noqa: E731
                     *prompts.token_logprobs(c[6], torch.arange(8, device=gpu), 3))
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    for own in (False, True):
        got = [None] * len(cases)

        def work(i):
            with torch.cuda.stream(torch.cuda.Stream() if own else torch.cuda.default_stream()):
                for _ in range(10):
                    got[i] = run(cases[i])
                torch.cuda.current_stream().synchronize()

        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
        [t.start() for t in threads]
        [t.join() for t in threads]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_patched_model_prompt_kernel(gpu):
    """patch_nemotron_h_attention_int4_kv(prompt_kernel=True): the prompt's logits within the kernels'
    rounding of the default's, the same INT4 rows, and the default as it was."""
    outs, caches = [], []
    ids = torch.randint(0, 64, (2, 45), device=gpu, generator=torch.Generator(device=gpu).manual_seed(6))
    for kernel in (False, True, True):
        fake.reset_module()
        torch.manual_seed(0)
        model = fake.FakeNemotronHForCausalLM(fake.make_config(hybrid_override_pattern="*-*")).to(
            gpu, torch.bfloat16).eval()
        de.patch_attention_cache_in_blocks(model)
        ia.patch_nemotron_h_attention_int4_kv(model, group_size=64, prompt_kernel=kernel)
        cache = fake.HybridMambaAttentionDynamicCache(model.config, 2, torch.bfloat16, gpu)
        with torch.no_grad():
            outs.append(model(ids, cache_params=cache, cache_position=torch.arange(45, device=gpu)).float())
            step = model(ids[:, :1], cache_params=cache, cache_position=torch.tensor([45], device=gpu))
        assert torch.isfinite(step).all()
        caches.append(cache._int4_kv_layer_caches[0])
        if kernel:
            # with gradients the forward is the default one
            grad = model(ids, cache_params=fake.HybridMambaAttentionDynamicCache(
                model.config, 2, torch.bfloat16, gpu), cache_position=torch.arange(45, device=gpu))
            assert torch.equal(grad.float(), outs[0])
    assert torch.equal(outs[1], outs[2])
    assert (outs[0] - outs[1]).norm() <= 2e-2 * outs[0].norm()
    assert torch.equal(caches[0].k_packed[:, :, :45], caches[1].k_packed[:, :, :45])


def test_padded_batch(gpu):
    """Texts of a batch that is padded behind them, with NaN in the pads, and left-padded ones whose pads
    are prompts of their own."""
    gen = torch.Generator(device=gpu).manual_seed(7)
    lengths, total = [50, 12, 33], 50
    q, k, v = (torch.randn(3, total, n, 128, device=gpu, generator=gen).bfloat16() for n in (8, 2, 2))
    x, dt = torch.randn(3, total, 8, 64, device=gpu, generator=gen).bfloat16(), torch.randn(
        3, total, 8, device=gpu, generator=gen)
    B, C = (torch.randn(3, total, 2, 128, device=gpu, generator=gen).bfloat16() for _ in range(2))
    A = -torch.rand(8, device=gpu, generator=gen)
    whole = prompts.prompt_attention(q, k, v), prompts.prompt_scan(x, dt, A, B, C, dt_softplus=True)[0]
    left = []
    for i, n in enumerate(lengths):
        left += [i * total, i * total + total - n]
    starts = torch.tensor(left + [3 * total], device=gpu)
    packed = prompts.prompt_attention(*(t.flatten(0, 1) for t in (q, k, v)), starts).unflatten(0, (3, total))
    for i, n in enumerate(lengths):
        tail = [t[i:i + 1, total - n:] for t in (q, k, v)]
        assert torch.equal(packed[i, total - n:], prompts.prompt_attention(*tail)[0])
        for t in (q, k, v, x, dt, B, C):
            t[i, n:] = float("nan")
    got = prompts.prompt_attention(q, k, v), prompts.prompt_scan(x, dt, A, B, C, dt_softplus=True)[0]
    for i, n in enumerate(lengths):
        for a, b in zip(got, whole):
            assert torch.equal(a[i, :n], b[i, :n])


def test_no_softmax_of_a_library(gpu):
    """prompt_attention against torch's own attention on repeated K and V (fp32)."""
    gen = torch.Generator(device=gpu).manual_seed(8)
    q, k, v = (torch.randn(2, 77, n, 64, device=gpu, generator=gen) for n in (6, 2, 2))
    want = F.scaled_dot_product_attention(q.cpu().double().transpose(1, 2),
                                          k.cpu().double().repeat_interleave(3, 2).transpose(1, 2),
                                          v.cpu().double().repeat_interleave(3, 2).transpose(1, 2),
                                          is_causal=True).transpose(1, 2)
    got = prompts.prompt_attention(q, k, v).cpu().double()
    assert (got - want).norm() <= 1e-6 * want.norm()
