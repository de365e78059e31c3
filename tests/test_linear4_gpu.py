"""Products with weights in 4 bits against 64-bit sums."""
import numpy as np
import pytest
import torch

import fourbit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def case(tokens, rows, columns, group, dtype, seed=0, scale=1.0):
    from xinfer_b200.weights import pack4
    gen = torch.Generator(device=DEV).manual_seed(seed + tokens * 7 + rows * 3 + columns)
    x = (torch.randn((tokens, columns), generator=gen, device=DEV) * scale).to(dtype)
    w = pack4(torch.randn((rows, columns), generator=gen, device=DEV) / columns ** 0.5, group)
    return x, w


def product(x, w, rows, out=None, **more):
    from xinfer_b200 import kernels as k
    if out is None:
        out = torch.full((x.shape[0], rows), 7.0, dtype=x.dtype, device=DEV)
    need = k.linear4_scratch(x.shape[0], rows, x.shape[1], x.dtype)
    k.linear4(out, x, w, scratch=torch.full((need,), float("nan"), device=DEV) if need else None, **more)
    return out


def check(out, x, w, group, rows):
    """Every sum of products is off by at most its longest chain of additions times a unit of the terms' sizes (2^-23: matrix units cut
    off what they add), and the result by half a step of its type."""
    value = torch.from_numpy(fourbit.weight_values(w.cpu().numpy(), group, rows, x.shape[1])).to(DEV)
    want, size = x.double() @ value.T, x.double().abs() @ value.abs().T
    # (a term m * sum(x) and a term s * code: together up to three times the size of the value where they cancel)
    chain = x.shape[1] / 16 + 64
    allowed = torch.finfo(x.dtype).eps / 2 * want.abs() + 3 * chain * 2.0 ** -23 * size + 1e-30
    if x.dtype == torch.bfloat16 and (x.shape[0] > 16 or x.shape[0] > 8 and rows * x.shape[1] > 2 ** 20):
        # many rows, from nine on with larger weights: every weight is rounded to bfloat16, by up to 2^-8 of itself; what sums of such errors reach, six times the root of their squares
        allowed = allowed + 2.0 ** -8 * torch.minimum(size, 6 * (x.double().square() @ value.square().T).sqrt())
    off = (out.double() - want).abs()
    assert bool((off <= allowed).all()), f"{(off / allowed).max().item():.2f} times what is allowed"


SIZES = [(1, 64, 128), (1, 6144, 4096), (2, 16, 32), (3, 777, 1000), (5, 1, 1), (7, 33, 129), (8, 4096, 4096), (9, 100, 640), (16, 512, 2048), (17, 48, 257), (31, 129, 96),
         (64, 256, 1024), (65, 80, 384), (130, 17, 640), (300, 200, 512), (33, 4096, 4096), (257, 129, 136), (1, 24576, 512), (4, 16, 12288), (9, 1030, 1024), (16, 300, 4090),
         (12, 24570, 72)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,rows,columns", SIZES)
def test_sums(tokens, rows, columns, group, dtype):
    x, w = case(tokens, rows, columns, group, dtype)
    check(product(x, w, rows), x, w, group, rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,rows,columns", [(3, 80, 256), (20, 80, 256), (5, 40, 130)])
def test_strides(tokens, rows, columns, dtype):
    x, w = case(tokens, rows, columns, 32, dtype)
    wide_x = torch.full((tokens, columns + 24), float("nan"), dtype=dtype, device=DEV)
    wide_x[:, 5:5 + columns] = x
    wide = torch.full((tokens, rows + 11), 3.0, dtype=dtype, device=DEV)
    product(wide_x[:, 5:5 + columns], w, rows, out=wide[:, 2:2 + rows])
    check(wide[:, 2:2 + rows], x, w, 32, rows)
    assert bool((wide[:, :2] == 3).all()) and bool((wide[:, 2 + rows:] == 3).all())


@pytest.mark.parametrize("scale", [1e-12, 1e-4, 1e4, 1e12])
@pytest.mark.parametrize("tokens", [1, 12, 40])
def test_magnitudes(scale, tokens):
    x, w = case(tokens, 96, 512, 64, torch.bfloat16, scale=scale)
    check(product(x, w, 96), x, w, 64, 96)


def test_rows_that_are_not_finite_stay_alone():
    for tokens in (3, 12, 40):
        x, w = case(tokens, 64, 256, 32, torch.bfloat16)
        clean = product(x, w, 64)
        x[1, 100] = float("inf")
        x[2, 3] = float("nan")
        got = product(x, w, 64)
        assert bool(torch.isnan(got[2]).all()) and not bool(torch.isfinite(got[1]).any())
        keep = [i for i in range(tokens) if i not in (1, 2)]
        assert torch.equal(got[keep], clean[keep])


def test_no_tokens():
    from xinfer_b200 import kernels as k
    x, w = case(1, 64, 128, 32, torch.bfloat16)
    out = torch.zeros((0, 64), dtype=torch.bfloat16, device=DEV)
    k.linear4(out, x[:0], w)


@pytest.mark.parametrize("tokens", [1, 40])
def test_graphs_and_streams(tokens):
    x, w = case(tokens, 512, 1024, 64, torch.bfloat16)
    want = product(x, w, 512)
    from xinfer_b200 import kernels as k
    out = torch.zeros_like(want)
    need = k.linear4_scratch(tokens, 512, 1024, x.dtype)
    scratch = torch.zeros(max(1, need), device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        k.linear4(out, x, w, scratch=scratch)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k.linear4(out, x, w, scratch=scratch)
        k.linear4(out, x, w, scratch=scratch)
    x.mul_(2)                    # (a power of two: the same digits)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want * 2)


@pytest.mark.parametrize("tokens", [1, 12, 40])
def test_weights_packed_here_or_laid_out_anew(tokens):
    from xinfer_b200 import kernels as k
    from xinfer_b200.weights import pack4
    gen = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn((tokens, 1024), generator=gen, device=DEV).to(torch.bfloat16)
    matrices = [torch.randn((512, 1024), generator=gen, device=DEV) for _ in range(3)]
    wants = [product(x, pack4(m.cpu(), 64).to(DEV), 512) for m in matrices]
    place = torch.zeros_like(pack4(matrices[0], 64))
    for m, want in zip(matrices * 3, wants * 3):
        out = torch.zeros_like(want)
        k.linear4(out, x, pack4(m, 64))
        assert torch.equal(out, want)
        place.copy_(pack4(m, 64))
        k.linear4(out.zero_(), x, place)
        assert torch.equal(out, want)


def test_calls_at_once():
    from xinfer_b200 import kernels as k
    cases = [case(tokens, 512, 2048, 64, torch.bfloat16) for tokens in (1, 16, 70, 300)]
    wants = [product(x, w, 512) for x, w in cases]
    outs, streams = [torch.zeros_like(y) for y in wants], [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for (x, w), out, stream in zip(cases, outs, streams):
            with torch.cuda.stream(stream):
                out.zero_()
                k.linear4(out, x, w)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, wants))


def test_refusals():
    from xinfer_b200 import kernels as k
    from xinfer_b200.weights import pack4
    x, w = case(3, 64, 256, 32, torch.bfloat16)
    out = torch.zeros((3, 64), dtype=torch.bfloat16, device=DEV)
    flat = torch.zeros(w.numel() + 16, dtype=torch.uint8, device=DEV)
    for args in ((out.float(), x, w), (out, x.half(), w), (out[:2], x, w), (out, x[:, :100], w), (out[:, :40], x, w), (out, x, w[..., :-4].contiguous()), (out, x, w.cpu()),
                 (out, x, w.int()), (out.t(), x, w), (out, x, flat[8:8 + w.numel()].view(w.shape)), (out[:, :0], x, w[:0])):
        with pytest.raises(k.KernelError):
            k.linear4(*args)
    assert np.array_equal(pack4(torch.zeros(3, 5)).shape, (1, 1, 1280))
