"""The 4-bit operators where calls meet, where numbers are very small or large, and at other edges of what their documentation allows."""
import math

import numpy as np
import pytest
import torch

import fourbit
from test_cache4_gpu import BF, DEV, F32, HALF, Attend, Write, i32
from test_linear4_gpu import case, check, product

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [20, 64])
def test_products_on_two_streams_whose_blocks_hold_tensor_memory(tokens):
    """Clusters of the 16-bit product for few rows and of the 4-bit one for many, at the same time again and again: both come to their end with their bits."""
    from xinfer_b200 import kernels as k
    x, w = case(tokens, 2048, 8192, 64, BF)
    gen = torch.Generator(device=DEV).manual_seed(3)
    x16, w16 = (torch.randn(s, generator=gen, device=DEV).to(BF) for s in ((8, 4096), (4096, 4096)))
    err = i32([0])
    want, want16 = product(x, w, 2048), torch.zeros((8, 4096), dtype=BF, device=DEV)
    assert k.gemm_skinny_tc(want16, x16, w16, err)
    out, out16 = torch.zeros_like(want), torch.zeros_like(want16)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(100):
        with torch.cuda.stream(streams[0]):
            k.linear4(out, x, w)
        with torch.cuda.stream(streams[1]):
            k.gemm_skinny_tc(out16, x16, w16, err)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(out16, want16) and int(err) == 0


@pytest.mark.parametrize("tokens", [1, 12, 40])
@pytest.mark.parametrize("between", [False, True])
def test_a_weight_that_the_kernel_ahead_has_just_written(tokens, between):
    """In front of the product a kernel writes the weight, or one that does and another that lets its successor start early; called and captured."""
    from xinfer_b200 import kernels as k
    from xinfer_b200.weights import pack4
    gen = torch.Generator(device=DEV).manual_seed(7)
    x = torch.randn((tokens, 4096), generator=gen, device=DEV).to(BF)
    weights = [pack4(torch.randn((2048, 4096), generator=gen, device=DEV), 64) for _ in range(2)]
    wants = [product(x, w, 2048) for w in weights]
    for w, want in zip(weights, wants):
        assert torch.equal(product(x, w, 2048, weight_ready=True), want)
    place, none, step = torch.zeros_like(weights[0]), torch.zeros_like(weights[0]), Write(1, 4, 2, 64, BF, 16)
    outs = [torch.zeros_like(w) for w in wants]

    def both():
        for w, out in zip(weights, outs):
            torch.bitwise_or(w, none, out=place)
            if between:
                step.run()
            k.linear4(out, x, place)

    for _ in range(20):
        both()
        assert all(torch.equal(a, b) for a, b in zip(outs, wants))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for _ in range(5):
        for out in outs:
            out.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, wants))


@pytest.mark.parametrize("tokens", [1, 40])
def test_products_report_to_the_word_they_are_given(tokens):
    from xinfer_b200 import kernels as k
    x, w = case(tokens, 128, 512, 64, BF)
    out, err, own = torch.zeros((tokens, 128), dtype=BF, device=DEV), i32([0]), k.own_err_word()
    own.value.value = k.ERR_WAIT                 # (as if a wait of an earlier call without a word had run out)
    k.linear4(out, x, w, err=err)
    assert int(err) == 0 and own.value.value == k.ERR_WAIT
    with pytest.raises(k.KernelError):
        k.linear4(out, x, w)
    k.linear4(out, x, w)
    for bad in (err.long(), err[:0], err.cpu(), 0):
        with pytest.raises(k.KernelError):
            k.linear4(out, x, w, err=bad)


@pytest.mark.parametrize("tokens,columns", [(1, 1100), (8, 1100), (12, 1100), (16, 1100), (40, 1100), (40, 1104), (300, 1104)])
@pytest.mark.parametrize("x_size,w_size", [(1e-16, 1.0), (1e-22, 1.0), (1e-30, 1.0), (1e-35, 1.0), (1e20, 1.0), (1e30, 1e-3), (1.0, 1e-16), (1.0, 1e-25), (1.0, 1e30), (1e-30, 1e30), (1e30, 1e-25),
                                           (1e-10, 1e-15)])
def test_products_of_small_and_large_numbers(x_size, w_size, tokens, columns):
    """The tolerance of test_linear4_gpu.check without its 1e-30: of each sum's terms, and of what is rounded; sums that bfloat16 holds as ordinary numbers."""
    from xinfer_b200.weights import pack4
    rows, group = 96, 64
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    x = torch.randn((tokens, columns), generator=gen, device=DEV)
    x = (x * x_size * 2.0 ** -torch.arange(tokens, device=DEV).remainder(4)[:, None].float()).to(BF)       # (rows of their own size)
    x[tokens // 2, columns // 3:columns // 2] *= 2.0 ** -20
    x[:, columns // 2:columns // 2 + 200] = 0
    w = pack4(torch.randn((rows, columns), generator=gen, device=DEV) / columns ** 0.5 * w_size, group)
    if tokens == 12:                       # (an odd start: the kernel for few rows reads x number by number)
        x = torch.cat([torch.zeros_like(x[:, :1]), x], 1)[:, 1:]
    got = product(x, w, rows)
    value = torch.from_numpy(fourbit.weight_values(w.cpu().numpy(), group, rows, columns)).to(DEV)
    want, size = x.double() @ value.T, x.double().abs() @ value.abs().T
    allowed = 2.0 ** -8 * want.abs() + 3 * (columns / 16 + 64) * 2.0 ** -23 * size
    if tokens > 16:
        allowed = allowed + 2.0 ** -8 * torch.minimum(size, 6 * (x.double().square() @ value.square().T).sqrt())
    off = (got.double() - want).abs()
    assert bool((off <= allowed).all()), f"{(off / allowed).max().item():.2f} times what is allowed"


@pytest.mark.parametrize("tokens,columns", [(1, 4096), (5, 4090), (8, 12288), (12, 1024), (40, 1100), (40, 4096)])
@pytest.mark.parametrize("low,high", [(1e-30, 1.0), (1.0, 1e30), (0.0, 1.0), (0.0, 1e-25), (1e-12, 1e2)])
def test_products_of_rows_whose_numbers_grow(low, high, tokens, columns):
    """Columns of one size in front of some of another, in every 512 columns and in the whole row; the rows beside such a row keep their bits."""
    rows, group = 80, 32
    x, w = case(tokens, rows, columns, group, BF)
    clean = product(x, w, rows)
    at, sizes = torch.arange(columns, device=DEV), torch.ones((tokens, columns), device=DEV)
    sizes[0] = torch.where(at % 512 < 300, low, high)
    sizes[tokens // 2] = torch.where(at < columns - 200, low, high)
    x = (x.float() * sizes).to(BF)
    got = product(x, w, rows)
    value = torch.from_numpy(fourbit.weight_values(w.cpu().numpy(), group, rows, columns)).to(DEV)
    want, size = x.double() @ value.T, x.double().abs() @ value.abs().T
    allowed = 2.0 ** -8 * want.abs() + 3 * (columns / 16 + 64) * 2.0 ** -23 * size
    if tokens > 16:
        allowed = allowed + 2.0 ** -8 * torch.minimum(size, 6 * (x.double().square() @ value.square().T).sqrt())
    off = (got.double() - want).abs()
    assert bool((off <= allowed).all()), f"{(off / allowed).max().item():.2f} times what is allowed"
    keep = [i for i in range(tokens) if i not in (0, tokens // 2)]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("news,keys", [([1], 200), ([1], 3000), ([1] * 40, 500), ([70], 400)])
def test_no_number_stays_where_later_scores_are_far_above(news, keys, dtype):
    """A value's group of NaN that a row sees reaches its channels, however small the probability of its key is beside later ones."""
    a = Attend(news, [keys] * len(news), 2, 1, 64, dtype, scale=1.0)
    a.q.fill_(1.0)
    level = torch.arange(a.pages, dtype=torch.float64)
    for b in range(len(news)):             # pages in the order of the table: every 64 keys 160 above the last
        for i, page in enumerate(a.table[b][:-(-a.lengths[b] // a.ps)]):
            level[page] = 160.0 / 64 * (i * a.ps // 64)
    a.data[0] = fourbit.page_bytes(np.broadcast_to(level.numpy()[:, None, None, None], (a.pages, 1, a.ps, 64)).copy(), a.ps)
    clean = a.run().clone()
    assert bool(torch.isfinite(clean).all())
    words = a.data[1][..., 2 * a.ps * 16:].reshape(a.pages, 1, a.ps, 2, 4)
    for b in range(len(news)):
        words[a.table[b, 0], 0, 3, 1] = 0xFF               # key 3, the second group
    got = a.run()
    rows = sum(news)
    assert bool(torch.isnan(got[:rows, :, 32:]).all()) and torch.equal(got[:rows, :, :32], clean[:rows, :, :32])


def with_values(a, sizes):
    """The same request with new values, of a size for each page of the pool in the order of the tables."""
    rng = np.random.default_rng(11)
    nkv, d = a.sizes[1:]
    level = np.ones(a.pages)
    for b, length in enumerate(a.lengths):
        held = -(-length // a.ps)
        level[a.table[b, :held]] = sizes(np.arange(held) / max(1, held - 1))
    a.data[1] = fourbit.page_bytes(rng.normal(size=(a.pages, nkv, a.ps, d)) * level[:, None, None, None], a.ps)
    return a


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [128, 48, 256])
@pytest.mark.parametrize("news,contexts", [([1, 6], [100, 37]), ([1], [3000]), ([100], [137])])
@pytest.mark.parametrize("size", [1e-11, 1e-15, 1e-20, 1e-24, 1e-31, 1e10, 1e25])
def test_values_of_any_size(size, news, contexts, d, dtype):
    """Values' sizes apart from the keys', in each of the kernels."""
    a = with_values(Attend(news, contexts, 8, 2, d, dtype), lambda at: size)
    a.run()
    a.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("news,contexts", [([1, 3], [700, 300]), ([1], [3000]), ([2] * 30, [400] * 30)])
@pytest.mark.parametrize("first,last", [(1e-20, 1.0), (1.0, 1e-20), (1e-8, 1e8), (0.0, 1.0), (0.0, 1e-20)])
def test_values_whose_sizes_change_from_page_to_page(first, last, news, contexts, d, dtype):
    grow = lambda at: np.where(at < 0.4, 0.0, last) if first == 0 else first * (last / first) ** at  # noqa: E731
    a = with_values(Attend(news, contexts, 8, 2, d, dtype), grow)
    a.run()
    a.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [128, 96, 256])
@pytest.mark.parametrize("news,contexts", [([1, 1], [40, 700]), ([3], [500]), ([1], [3000]), ([60, 2], [100, 20])])
def test_a_group_of_no_numbers_keeps_to_its_channels(news, contexts, d, dtype):
    a = Attend(news, contexts, 4, 2, d, dtype)
    clean = a.run().clone()
    groups = d // 32
    whole = a.data[1].copy()
    words = a.data[1][..., groups * a.ps * 16:].reshape(a.pages, 2, a.ps, groups, 4)
    for b in range(len(news)):
        words[a.table[b, 1], 1, 3, 1] = 0xFF           # key 19, the second key/value head, channels 32 to 63
    got, bad = a.run().clone(), torch.zeros_like(clean, dtype=torch.bool)
    bad[:sum(news), 2:, 32:64] = True
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[:, :2], clean[:, :2])
    # the other channels of these heads may have been summed up in another order: against 64 bits, like any sum
    a.data[1] = whole
    a.out.copy_(torch.where(bad, clean, got))
    a.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [128, 48, 7])
@pytest.mark.parametrize("size", [1e-30, 1e-36, 1e-37, 1e-38, 1e-39, 1e30, 1e37])
def test_write_numbers_of_any_size(size, d, dtype):
    """Scales below the ordinary float32 numbers, whose reciprocals are infinite, and large ones: the definition's codes."""
    w = Write(40, 2, 2, d, dtype, 16, norm=False, rot=0)
    w.qkv.copy_((w.qkv.double() * size).to(dtype))
    w.run()
    w.check()
    assert int(w.err) == 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 40 + 1])
@pytest.mark.parametrize("news,contexts", [([1, 5], [150, 60]), ([70], [30])])
def test_windows_and_longest_requests_that_32_bits_do_not_hold(news, contexts, window, dtype):
    """A window of more keys than there are is none; a request brings no more tokens than the step has."""
    a = Attend(news, contexts, 4, 2, 64, dtype)
    want = a.run().clone()
    a.window = window
    assert torch.equal(a.run(), want)
    a.run(longest=window)
    a.check()


@pytest.mark.parametrize("d,window", [(128, None), (64, 100), (96, None), (40, None)])
@pytest.mark.parametrize("news,contexts", [([12, 3, 4, 15, 0], [200, 900, 31, 0, 9]), ([4, 13, 6], [640, 200, 77]), ([15], [1500])])
def test_requests_of_16_to_63_rows_beside_larger_ones(news, contexts, d, window):
    """Steps whose largest request has 48 rows and more: requests of 16 and more have the kernel for many, with float16 operands, and its bound: a probability and
    a value are off by 2^-11 of themselves (values by 2^-25 of the largest at least), a key by that in every product of a score."""
    nh, nkv = 8, 2
    a = Attend(news, contexts, nh, nkv, d, BF, window=window)
    got = a.run().double().cpu().numpy()
    keys, vals = (fourbit.page_values(x, a.ps, d) for x in a.data)
    q = a.q.double().cpu().numpy()
    assert max(news) * (nh // nkv) >= 48
    for b, n in enumerate(news):
        if n * (nh // nkv) < 16:
            continue
        j = np.arange(a.lengths[b])
        page = a.table[b][j // a.ps]
        for i in range(n):
            pos, t = a.lengths[b] - n + i, a.start[b] + i
            seen = (j <= pos) & (j > pos - (window or 2 ** 31))
            for h in range(nh):
                kk, vv = keys[page, h // 4, j % a.ps][seen], vals[page, h // 4, j % a.ps][seen]
                x = kk @ q[t, h] * a.scale
                p = np.exp(x - x.max())
                p /= p.sum()
                want, size = p @ vv, p @ np.abs(vv)
                steps = np.abs(kk).max() * np.abs(q[t, h]).sum() * a.scale
                allowed = HALF[BF] * np.abs(want) + (2 * (d + 16) * 2.0 ** -23 * steps + (64 + seen.sum() / 16) * 2.0 ** -23) * size
                allowed = allowed + (2 + 2 * float((p * (np.abs(kk) @ np.abs(q[t, h]))).sum() * a.scale)) * 2.0 ** -11 * size + 2.0 ** -25 * np.abs(vv).max()
                off = np.abs(got[t, h] - want)
                assert np.all(off <= allowed), (b, i, h, (off / allowed).max())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [128, 96, 256])
@pytest.mark.parametrize("small", [1e-12, 1e-20, 1e-30])
def test_small_values_beside_larger_ones_that_hardly_count(small, d, dtype):
    """The second page's values are ordinary and its scores 200 below the others'."""
    a = with_values(Attend([1, 2], [300, 90], 4, 1, d, dtype, scale=1.0), lambda at: np.where(np.arange(len(at)) == 1, 1.0, small))
    a.q.fill_(1.0)
    rng, level = np.random.default_rng(3), np.zeros(a.pages)
    level[a.table[:, 1]] = -200.0 / d
    a.data[0] = fourbit.page_bytes(rng.normal(size=(a.pages, 1, a.ps, d)) * 0.05 + level[:, None, None, None], a.ps)
    a.run()
    a.check()


@pytest.mark.parametrize("d,ps", [(128, 16), (48, 8), (128, 4), (64, 12)])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("power", [10, 18, 24, 40, 60])
@pytest.mark.parametrize("news,contexts", [([100], [137]), ([1, 40, 200, 20], [300, 90, 64, 10])])
def test_portions_with_a_key_or_value_far_larger_than_the_others(news, contexts, power, which, d, ps):
    """A token in the middle of a portion and its last one, whose key or value is 2^power times the others' size: rows that do not see it, and rows that see it with a
    score far below the others', have their digits."""
    nh, nkv = 8, 2
    a = Attend(news, contexts, nh, nkv, d, BF, ps=ps)
    rng = np.random.default_rng(5)
    x = [rng.normal(size=(a.pages, nkv, ps, d)) for _ in range(2)]
    b = len(news) // 2                       # the longest portion's request
    for pos in (a.lengths[b] - 1, a.lengths[b] - news[b] // 2 - 1):
        at = a.table[b, pos // ps], slice(None), pos % ps
        x[which][at] *= 2.0 ** power
        x[0][at] = -np.abs(x[0][at]) - (30 if which else 0)          # (queries of positive numbers give it a low score)
    a.q.abs_()
    a.data = [fourbit.page_bytes(y, ps) for y in x]
    got = a.run().double().cpu().numpy()
    keys, vals = (fourbit.page_values(y, ps, d) for y in a.data)
    q = a.q.double().cpu().numpy()
    for b, n in enumerate(news):
        j = np.arange(a.lengths[b])
        page = a.table[b][j // ps]
        for i in range(n):
            pos, t = a.lengths[b] - n + i, a.start[b] + i
            seen = j <= pos
            for h in (0, 5):
                kk, vv = keys[page, h // 4, j % ps][seen], vals[page, h // 4, j % ps][seen]
                s = kk @ q[t, h] * a.scale
                p = np.exp(s - s.max())
                p /= p.sum()
                want, size = p @ vv, p @ np.abs(vv)
                # float16 operands (see above) or a bfloat16 probability times a scale; scores of the keys that count
                steps = (p * (np.abs(kk) @ np.abs(q[t, h]))).sum() * a.scale
                allowed = HALF[BF] * np.abs(want) + (4 * (d + 16) * 2.0 ** -23 * steps + (64 + seen.sum() / 16) * 2.0 ** -23 + (2 + 2 * steps) * 2.0 ** -11 + 2 * 3 * 2.0 ** -8) * size
                off = np.abs(got[t, h] - want)
                # values up to 2^12 times the others': 2^-31 of the largest for every key
                allowed = allowed + (seen.sum() * 2.0 ** -31 * 2.0 ** power if which and power <= 12 else 0)
                assert np.all(off <= allowed), (b, i, h, (off / allowed).max())


def check_few_rows(a, heads=None):
    """Against 64 bits with the bound of the kernel for few rows: bfloat16 roundings of a probability, by itself and times a group's scale, for both parts of
    m + s code, and float32 sums (test_cache4_gpu.Attend.check), which is also what requests that the kernel for many rows leaves get."""
    nh, nkv, d = a.sizes
    got, q = a.out.double().cpu().numpy(), a.q.double().cpu().numpy()
    keys, vals = (fourbit.page_values(x, a.ps, d) for x in a.data)
    codes, s, m = fourbit.page_parts(a.data[1], a.ps, d)
    parts = np.abs(m)[..., np.arange(d) // 32] + s[..., np.arange(d) // 32] * codes
    for b, n in enumerate(a.news):
        j = np.arange(a.lengths[b])
        page = a.table[b][j // a.ps]
        for i in range(n):
            seen, t = j <= a.lengths[b] - n + i, a.start[b] + i
            for h in heads or range(nh):
                g = h // (nh // nkv)
                kk, vv, pp = (x[page, :, j % a.ps][seen, g] for x in (keys, vals, parts))
                x = kk @ q[t, h] * a.scale
                p = np.exp(x - x.max())
                p /= p.sum()
                steps = np.abs(kk).max() * np.abs(q[t, h]).sum() * a.scale
                allowed = HALF[BF] * np.abs(p @ vv) + (2 * (d + 16) * 2.0 ** -23 * steps + (64 + seen.sum() / 16) * 2.0 ** -23) * (p @ np.abs(vv)) + 2 * 2.0 ** -8 * (p @ pp)
                assert np.all(np.abs(got[t, h] - p @ vv) <= allowed), (b, i, h)


def test_a_captured_step_whose_values_come_to_differ():
    """The same graph before and after a value grows: which kernel gives a request's rows is seen on the device."""
    from xinfer_b200 import kernels as k
    a = Attend([100, 30, 2], [137, 60, 500], 8, 2, 128, BF)
    caches, lengths, start, table = a.tensors()
    scratch = torch.zeros(k.cache4_attention_scratch(a.q.shape[0], 3, 8, 2, 128, BF, 100), device=DEV)

    def call():
        k.cache4_attention(a.out, a.q, *caches, lengths, start, table, a.ps, a.scale, a.err, scratch=scratch, longest=100)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    plain = a.data[1].copy()
    grown = with_values(a, lambda at: np.where(np.arange(len(at)) == 1, 2.0 ** 30, 1.0)).data[1].copy()
    for data in (plain, grown, plain, grown):
        a.data[1] = data
        want = a.run().clone()
        (a.check if data is plain else lambda: check_few_rows(a))()
        for cache, part in zip(caches, a.data):
            cache.copy_(torch.from_numpy(part))
        a.out.fill_(9.0)
        graph.replay()
        assert torch.equal(a.out, want) and int(a.err) == 0


@pytest.mark.parametrize("below,power", [(13.4, 0), (8.4, 11), (13.4, 11), (13.4, 16)])
def test_portions_whose_many_small_probabilities_count(below, power):
    """One key's score is far above 2,000 others', which together count too, beside a value 2^power times theirs whose key counts for nothing; so many
    requests and heads that a block has a job's keys to itself."""
    d, nkv = 32, 37
    a = Attend([50] * 4, [2000] * 4, nkv, nkv, d, BF, scale=1.0)
    a.q.fill_(1.0)
    rng = np.random.default_rng(9)
    level = np.full((a.pages, 1, a.ps, 1), -below * math.log(2) / d)
    level[a.table[:, 0], :, 0] = 0.0
    level[a.table[:, 1], :, 0] = -300.0 / d
    values = 1 + 0.1 * rng.normal(size=(a.pages, nkv, a.ps, d))
    values[a.table[:, 1], :, 0] = 2.0 ** power
    a.data = [fourbit.page_bytes(np.broadcast_to(level, values.shape).copy(), a.ps), fourbit.page_bytes(values, a.ps)]
    a.run()
    check_few_rows(a, heads=(0, 17, 36))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [128, 96, 256, 32])
@pytest.mark.parametrize("news,contexts,times", [([1], [300], 1), ([1], [300], 1500), ([3, 1], [90, 700], 1), ([60], [100], 1)])
def test_heads_of_a_group_that_count_values_of_different_sizes(news, contexts, times, d, dtype):
    """Half of a group's heads give all their weight to a page of ordinary values, the other half to the small values of the other pages.  With so many requests
    (of the same pages) that a request's keys are one segment, too."""
    a = with_values(Attend(news, contexts, 4, 1, d, dtype, scale=1.0), lambda at: np.where(np.arange(len(at)) == 1, 1.0, 1e-18))
    if times > 1:
        a.news, a.lengths, a.table, a.start = a.news * times, a.lengths * times, np.repeat(a.table, times, 0), list(range(times + 1))
        a.q, a.out = (torch.zeros((times + 2, 4, d), dtype=dtype, device=DEV) for _ in range(2))
    a.q.fill_(1.0)
    a.q[:, 1::2] = -1.0
    rng, level = np.random.default_rng(4), np.zeros(a.pages)
    level[a.table[:, 1]] = -200.0 / d
    a.data[0] = fourbit.page_bytes(rng.normal(size=(a.pages, 1, a.ps, d)) * 0.02 + level[:, None, None, None], a.ps)
    a.run()
    if times > 1:                      # (all requests are the same one: twenty of them are looked at)
        a.news, a.start = a.news[:20], a.start[:21]
        a.out[20:] = 9.0
    if dtype == F32:
        a.check()
    else:
        check_few_rows(a)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [128, 48])
@pytest.mark.parametrize("news,contexts", [([1, 6], [100, 37]), ([100], [137])])
@pytest.mark.parametrize("k_size,q_size", [(1e-28, 1.0), (1e-20, 1.0), (1e12, 1.0), (1e20, 1.0), (1e30, 1.0), (1.0, 1e-30), (1.0, 1e-12), (1.0, 1e20), (1.0, 1e34), (1e-20, 1e20), (1e15, 1e-30)])
def test_keys_and_queries_of_any_size(k_size, q_size, news, contexts, d, dtype):
    a = Attend(news, contexts, 8, 2, d, dtype, scale=0.1 / (k_size * q_size))
    rng = np.random.default_rng(6)
    a.data[0] = fourbit.page_bytes(rng.normal(size=(a.pages, 2, a.ps, d)) * k_size, a.ps)
    a.q.copy_((a.q.double() * q_size).to(dtype))
    a.run()
    a.check()
