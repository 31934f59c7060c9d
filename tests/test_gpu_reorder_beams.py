"""reorder_beams against index_select: every byte of the tensors and of what surrounds them."""
import pytest
import torch

from layer_quant_amd import beam_decode as bd

pytestmark = pytest.mark.gpu


def expected(t, beams, rows=None):
    P, N = beams.shape
    src = torch.where((beams >= 0) & (beams < N), beams, torch.arange(N, device=beams.device))
    at = (torch.arange(P, device=beams.device)[:, None] * N + src).reshape(-1)
    out = t.clone()
    if rows is None:
        out.copy_(t[at])
    else:
        out[:, :, :rows] = t[at][:, :, :rows]
    return out


def filled(gpu, shape, dtype, seed=0):
    gen = torch.Generator(device=gpu).manual_seed(seed)
    size = torch.empty(0, dtype=dtype).element_size()
    raw = torch.randint(0, 256, (*shape[:-1], shape[-1] * size), dtype=torch.uint8, device=gpu,
                        generator=gen)
    return raw.view(dtype)


def same_bytes(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def beams_of(gpu, P, N, kind, seed=0):
    gen = torch.Generator().manual_seed(seed)
    if kind == "cycle":
        b = (torch.arange(N) + 1).remainder(N).repeat(P, 1)
    elif kind == "reverse":
        b = torch.arange(N).flip(0).repeat(P, 1)
    elif kind == "one":
        b = torch.full((P, N), N - 1)
    elif kind == "stay":
        b = torch.arange(N).repeat(P, 1)
    elif kind == "bad":
        b = torch.randint(-2, N + 2, (P, N), generator=gen)
        b[0, 0] = 1 << 40
    else:
        b = torch.randint(0, N, (P, N), generator=gen)
    return b.to(gpu)


@pytest.mark.parametrize("kind", ["random", "cycle", "reverse", "one", "stay", "bad"])
@pytest.mark.parametrize("P,N", [(1, 1), (1, 2), (3, 4), (2, 5), (1, 16), (2, 17), (1, 33), (2, 64)])
def test_permutations(gpu, P, N, kind):
    B = P * N
    beams = beams_of(gpu, P, N, kind, N)
    tensors = [filled(gpu, (B, 2, 40, 64), torch.uint8, 1), filled(gpu, (B, 2, 40, 4), torch.float32, 2),
               filled(gpu, (B, 3, 5, 32), torch.int8, 3), filled(gpu, (B, 7), torch.int64, 4),
               filled(gpu, (B, 13, 4), torch.bfloat16, 5), filled(gpu, (B, 1), torch.uint8, 6),
               filled(gpu, (B,), torch.int32, 7), filled(gpu, (B, 3, 3, 3), torch.float16, 8)]
    rows = [29, 29, None, None, None, None, None, 2]
    want = [expected(t, beams, r) for t, r in zip(tensors, rows)]
    bd.reorder_beams(tensors, beams, rows)
    assert all(same_bytes(t, w) for t, w in zip(tensors, want))


@pytest.mark.parametrize("rows", [0, 1, 7, 39, 40])
@pytest.mark.parametrize("offset", [0, 1, 2, 4, 8])
def test_strides_and_surroundings(gpu, rows, offset):
    """Views into a larger buffer: rows, heads and entries with gaps, odd addresses, transposed and
    strided inner dims, reversed rows; the bytes around the view stay."""
    P, N = 2, 3
    beams = beams_of(gpu, P, N, "random", 3)
    views = [lambda t: t[:, :, :, offset:offset + 20], lambda t: t[:, 1:, 3:43, ::3],
             lambda t: t.transpose(1, 3), lambda t: t.transpose(2, 3)[:, :, :45],
             lambda t: t[:, :, 1:, 0], lambda t: t.transpose(0, 1)[0].expand(P * N, -1, -1, -1)
             if t.dim() == 5 else t[:, 0]]
    for view in views:
        whole = filled(gpu, (P * N, 4, 48, 64), torch.uint8, offset)
        ref = whole.clone()
        v, r = view(whole), view(ref)
        live = min(rows, v.shape[2])
        r.copy_(expected(r, beams, live))
        bd.reorder_beams([v], beams, [live])
        assert torch.equal(whole, ref)
    whole = filled(gpu, (64, P * N), torch.float32, 9)  # rows innermost
    ref = expected(whole.t(), beams).t()
    bd.reorder_beams([whole.t()], beams)
    assert same_bytes(whole, ref)
    pair = torch.stack((beams, beams.flip(1)), -1)
    t = filled(gpu, (P * N, 100), torch.uint8, 10)
    w = expected(t, pair[..., 1])
    bd.reorder_beams([t], pair[..., 1])
    assert torch.equal(t, w)


def test_many_tensors(gpu):
    """More tensors and more row shapes than one launch takes."""
    P, N = 2, 4
    beams = beams_of(gpu, P, N, "random", 8)
    tensors = [filled(gpu, (P * N, 1 + i % 37), torch.uint8, i) for i in range(512)]
    want = [expected(t, beams) for t in tensors]
    bd.reorder_beams(tensors, beams)
    assert all(torch.equal(t, w) for t, w in zip(tensors, want))
    bd.reorder_beams([], beams)


def test_large_offsets(gpu):
    """Rows whose places pass 32 bits."""
    P, N = 1, 3
    t = torch.zeros(N, 1 << 31, dtype=torch.uint8, device=gpu)
    t[0, -17:], t[1, -5:], t[2, :9] = 3, 4, 5
    bd.reorder_beams([t], torch.tensor([[2, 0, 1]], device=gpu))
    assert t[1, -17:].eq(3).all() and not t[1, :-17].any()
    assert t[2, -5:].eq(4).all() and t[0, :9].eq(5).all() and not t[0, 9:].any()


def test_stream_and_capture(gpu):
    P, N = 2, 8
    t = filled(gpu, (P * N, 3, 50, 64), torch.uint8, 1)
    beams = beams_of(gpu, P, N, "cycle")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            bd.reorder_beams([t], beams, [33])
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(4):
        beams.copy_(beams_of(gpu, P, N, "random", seed))
        want = expected(t, beams, 33)
        g.replay()
        assert torch.equal(t, want)
