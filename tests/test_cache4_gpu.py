"""Writing a cache of 4-bit codes and attending over it, against plain loops in 64 bits."""
import math

import numpy as np
import pytest
import torch

import fourbit

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
HALF = {BF: 2.0 ** -8, F32: 2.0 ** -24}
i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731


# ---- writing -----------------------------------------------------------------------------------------------------------

class Write:
    def __init__(self, tokens, nh, nkv, d, dtype, ps, norm=True, rot=None, interleaved=False, pad=0, seed=0, gap=0):
        self.sizes, self.dtype, self.ps, self.interleaved = (nh, nkv, d), dtype, ps, interleaved
        rng = np.random.default_rng(seed + tokens + d)
        gen = torch.Generator(device=DEV).manual_seed(seed + tokens * 3 + d)
        rot = d if rot is None else rot
        T = tokens + pad
        self.pages = -(-tokens // ps) + 2
        width = (nh + 2 * nkv) * d
        self.wide = torch.randn((T, width + gap), generator=gen, device=DEV, dtype=F32).mul_(2).to(dtype)
        self.qkv = self.wide[:, gap:]
        self.slots = torch.full((T,), -1, dtype=torch.int64, device=DEV)
        self.slots[:tokens] = torch.tensor(rng.permutation(self.pages * ps)[:tokens], device=DEV)
        self.positions = i32(rng.integers(0, 500, T))
        self.q_norm, self.k_norm = [1 + 0.3 * torch.randn(d, generator=gen, device=DEV) for _ in range(2)] if norm else (None, None)
        self.cos = self.sin = None
        if rot:
            angle = torch.arange(500, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
            self.cos, self.sin = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
        self.caches = [torch.full((self.pages, nkv, ps * 20 * -(-d // 32)), 0xA5, dtype=torch.uint8, device=DEV) for _ in range(2)]
        self.q_out = torch.full((T, nh, d), 7.0, dtype=dtype, device=DEV)
        self.values = [torch.full((T, nkv, d), 7.0, dtype=BF, device=DEV) for _ in range(2)]
        self.err = i32([0])

    def run(self, values=True):
        from xinfer_b200 import kernels as k
        k.cache4_write(self.q_out, *self.caches, self.qkv, self.positions, self.slots, self.ps, self.err, q_norm=self.q_norm, k_norm=self.k_norm, eps=1e-5, cos=self.cos,
                       sin=self.sin, interleaved=self.interleaved, values=self.values if values else None)

    def want(self):
        """Queries, keys and values in 64 bits."""
        nh, nkv, d = self.sizes
        x = self.qkv.double().cpu().numpy().reshape(-1, nh + 2 * nkv, d).copy()
        for h0, h1, w in ((0, nh, self.q_norm), (nh, nh + nkv, self.k_norm)):
            if w is not None:
                y = x[:, h0:h1]
                x[:, h0:h1] = y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-5) * w.double().cpu().numpy()
        if self.cos is not None:
            at = self.positions.cpu().numpy().clip(0, 499)
            c, s = (t.double().cpu().numpy()[at][:, None] for t in (self.cos, self.sin))
            half = c.shape[-1]
            y = x[:, :nh + nkv]
            a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if self.interleaved else (slice(0, half), slice(half, 2 * half))
            u, v = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
            y[..., a], y[..., b] = u, v
        return x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]

    def check(self):
        nh, nkv, d = self.sizes
        q, keys, vals = self.want()
        # a dozen float32 operations on numbers of the head's size, then one rounding
        most = np.abs(q).max(-1, keepdims=True)
        assert np.all(np.abs(self.q_out.double().cpu().numpy() - q) <= HALF[self.dtype] * np.abs(q) + 16 * 2.0 ** -24 * most)
        slots = self.slots.cpu().numpy()
        live = (slots >= 0) & (slots < self.pages * self.ps)
        at = slots[live]
        before = np.full((1,), 0xA5, np.uint8)
        for cache, rows, values, same in ((self.caches[0], keys, self.values[0], self.k_norm is None and self.cos is None), (self.caches[1], vals, self.values[1], True)):
            data = cache.cpu().numpy()
            codes, s, m = (p[at // self.ps, :, at % self.ps] for p in fourbit.page_parts(data, self.ps, d))
            got = m[..., np.arange(d) // 32] + s[..., np.arange(d) // 32] * codes
            out = values.double().cpu().numpy()
            assert np.array_equal(out[live], fourbit.bf16(got))
            for j in range(s.shape[-1]):
                g = rows[live][..., j * 32:(j + 1) * 32]
                lo, hi = g.min(-1), g.max(-1)
                if same:           # numbers as they came: the definition's own codes and words
                    ws, wm = fourbit.bf16((hi - lo) / 15), fourbit.bf16(lo)
                    gs = s[..., j]
                    if self.dtype == F32:      # (hi - lo) / 15 is off by two roundings of 2^-24: next to the middle of two bfloat16 numbers s may be either
                        off = np.abs((gs + ws) / 2 - (hi - lo) / 15)
                        ws = np.where((gs != ws) & (off <= 2 * 2.0 ** -24 * ws), gs, ws)
                    quotient = np.where(gs[..., None] > 0, (g - wm[..., None]) / np.where(gs > 0, gs, 1)[..., None], 0)
                    differ = codes[..., j * 32:(j + 1) * 32] != np.clip(np.rint(quotient), 0, 15)
                    assert np.array_equal(gs, ws) and np.array_equal(m[..., j], wm)
                    # bfloat16: x - m has 24 bits or is a whole step away from a half, so its quotient rounds to a half only if it is one.  float32: x - m
                    # is off by 2^-24 of itself and the quotient by as much again, together below 2 * 2^-24 * 16: what lies that near to a half may go
                    # either way.
                    near = 0 if self.dtype == BF else 2 * 2.0 ** -24 * 16
                    assert not differ[np.abs(np.abs(quotient - np.floor(quotient)) - 0.5) > near].any() and (self.dtype != BF or not differ.any())
                else:              # half a step, and what the rounding of s and m moves the range's ends
                    size = np.abs(g).max(-1)
                    assert np.all(np.abs(s[..., j] - (hi - lo) / 15) <= 2.0 ** -8 * (hi - lo) / 15 + 2.0 ** -18 * size) and np.all(np.abs(m[..., j] - lo) <= 2.0 ** -8 * np.abs(lo) + 2.0 ** -18 * size)
                    assert np.all(np.abs(got[..., j * 32:(j + 1) * 32] - g) <= (0.5 * s[..., j] + 2.0 ** -8 * np.abs(lo) + 15 * 2.0 ** -8 * s[..., j] + 2.0 ** -18 * size)[..., None])
            # slots that no token has are as they were
            free = np.setdiff1d(np.arange(self.pages * self.ps), at)
            groups = -(-d // 32)
            c = data[..., :groups * self.ps * 16].reshape(self.pages, nkv, groups, self.ps, 16)[free // self.ps, :, :, free % self.ps]
            w = data[..., groups * self.ps * 16:].reshape(self.pages, nkv, self.ps, groups * 4)[free // self.ps, :, free % self.ps]
            assert np.all(c == before) and np.all(w == before)


HEADS = [(4, 2, 128), (1, 1, 64), (8, 8, 32), (6, 2, 48), (5, 5, 80), (9, 3, 96), (4, 1, 256), (3, 1, 7), (2, 2, 40), (16, 8, 128), (2, 1, 192)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("tokens,ps", [(1, 16), (37, 8), (70, 5), (200, 64)])
def test_write(tokens, ps, nh, nkv, d, dtype):
    w = Write(tokens, nh, nkv, d, dtype, ps, rot=d - d % 2, pad=3)
    w.run()
    w.check()
    assert int(w.err) == 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("norm,rot,interleaved", [(False, 0, False), (True, 0, False), (False, 64, False), (True, 32, False), (True, 128, True), (False, 10, True), (True, 126, False), (True, 64, True)])
def test_write_forms(norm, rot, interleaved, dtype):
    w = Write(19, 4, 2, 128, dtype, 16, norm=norm, rot=rot, interleaved=interleaved)
    w.run(values=False)
    w.run()
    w.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("gap", [1, 8, 24])
def test_write_rows_that_lie_apart(gap, dtype):
    w = Write(21, 4, 2, 128, dtype, 16, gap=gap)
    w.run()
    w.check()


@pytest.mark.parametrize("d", [128, 64, 48])
def test_write_slots_and_positions_outside(d):
    from xinfer_b200 import kernels as k
    w = Write(9, 4, 2, d, BF, 16)
    w.slots[3] = w.pages * 16
    w.slots[5] = 2 ** 40
    w.run()
    w.check()
    assert int(w.err) == k.ERR_BAD_PAGE
    w = Write(9, 4, 2, d, BF, 16)
    w.positions[2], w.positions[4] = 500, -1
    w.run()
    w.check()
    assert int(w.err) == k.ERR_BAD_POSITION
    w.err.zero_()
    w.slots[2] = w.slots[4] = -1         # (a token that is not cached may have any position)
    w.run()
    assert int(w.err) == 0


@pytest.mark.parametrize("d", [128, 48])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_write_numbers_that_are_not_finite(what, d):
    w = Write(5, 2, 1, d, BF, 8, norm=False, rot=0)
    w.qkv[1, 2 * d + 3] = what           # a key's first group
    w.qkv[3, 3 * d + d - 1] = what       # a value's last one
    w.run()
    keys, vals = (t[:, 0].float().cpu() for t in w.values)
    bad_k, bad_v = torch.zeros(5, d, dtype=torch.bool), torch.zeros(5, d, dtype=torch.bool)
    bad_k[1, :32] = True
    bad_v[3, (d - 1) // 32 * 32:] = True
    assert torch.equal(torch.isnan(keys), bad_k) and torch.equal(torch.isnan(vals), bad_v)
    assert bool(torch.isfinite(keys[~bad_k]).all()) and bool(torch.isfinite(vals[~bad_v]).all())


@pytest.mark.parametrize("d", [128, 40])
def test_write_groups_of_one_number(d):
    w = Write(4, 2, 2, d, BF, 8, norm=False, rot=0)
    w.qkv[1] = 0.0
    w.qkv[2] = -3.0e38                   # (the spread is zero, the least value holds it)
    w.run()
    for t in w.values:
        assert bool((t[1] == 0).all()) and torch.equal(t[2], torch.full_like(t[2], -3.0e38))
    w.check()


def test_write_no_tokens():
    w = Write(0, 4, 2, 64, BF, 16)
    w.run()


# ---- attending -----------------------------------------------------------------------------------------------------------

class Attend:
    """Requests with `news` tokens behind `contexts` cached ones."""

    def __init__(self, news, contexts, nh, nkv, d, dtype, ps=16, window=None, seed=0, apart=0, scale=None, size=1.0):
        rng = np.random.default_rng(seed + sum(news) + d)
        self.sizes, self.ps, self.window, self.dtype = (nh, nkv, d), ps, window, dtype
        self.news, self.lengths = list(news), [n + c for n, c in zip(news, contexts)]
        held = [-(-n // ps) for n in self.lengths]
        self.pages = sum(held) + 3
        ids = rng.permutation(self.pages)
        self.table = np.full((len(news), max(1, max(held)) + 1), -1)
        at = 0
        for b, h in enumerate(held):
            self.table[b, :h] = ids[at:at + h]
            at += h
        self.data = [fourbit.page_bytes(rng.normal(size=(self.pages, nkv, ps, d)) * size, ps) for _ in range(2)]
        T = sum(news)
        self.start = [0] + list(np.cumsum(news))
        gen = torch.Generator(device=DEV).manual_seed(seed + T)
        self.q_rows = torch.randn((T + 2, nh * d + apart), generator=gen, device=DEV).mul_(1.5).to(dtype)
        self.out_rows = torch.full((T + 2, nh * d + apart), 9.0, dtype=dtype, device=DEV)
        self.q, self.out = (t[:, apart:].unflatten(1, (nh, d)) for t in (self.q_rows, self.out_rows))
        self.scale = scale if scale is not None else 1 / math.sqrt(d)
        self.err, self.bad = i32([0]), []

    def tensors(self):
        return [torch.from_numpy(x).to(DEV) for x in self.data], i32(self.lengths), i32(self.start), i32(self.table)

    def run(self, longest="known", err=0):
        from xinfer_b200 import kernels as k
        caches, lengths, start, table = self.tensors()
        nh, nkv, d = self.sizes
        longest = max(1, max(self.news)) if longest == "known" else longest
        need = k.cache4_attention_scratch(self.q.shape[0], len(self.news), nh, nkv, d, self.dtype, longest)
        scratch = torch.full((need,), float("nan"), device=DEV) if need else None
        self.out.fill_(9.0)
        k.cache4_attention(self.out, self.q, *caches, lengths, start, table, self.ps, self.scale, self.err, scratch=scratch, window=self.window, longest=longest)
        assert int(self.err) == err
        return self.out

    def check(self, hidden=lambda b, j: False):
        """Sums in 64 bits.  What float32 sums, bfloat16 probabilities and one rounding may be off: see `allowed`."""
        nh, nkv, d = self.sizes
        got = self.out.double().cpu().numpy()
        keys, vals = (fourbit.page_values(x, self.ps, d) for x in self.data)
        codes, s, m = fourbit.page_parts(self.data[1], self.ps, d)
        parts = np.abs(m)[..., np.arange(d) // 32] + s[..., np.arange(d) // 32] * codes
        q = self.q.double().cpu().numpy()
        for b, n in enumerate(self.news):
            length = self.lengths[b]
            j = np.arange(length)
            page = self.table[b][j // self.ps]
            k_all, v_all = keys[page, :, j % self.ps], vals[page, :, j % self.ps]
            bad = np.array([hidden(b, x) for x in j], bool)
            for i in range(n):
                pos, t = length - n + i, self.start[b] + i
                seen = (j <= pos) & ~bad
                if self.window:
                    seen &= j > pos - self.window
                for h in range(nh):
                    g = h // (nh // nkv)
                    if not seen.any():
                        assert np.all(got[t, h] == 0), (b, i, h)
                        continue
                    kk, vv = k_all[seen, g], v_all[seen, g]
                    x = kk @ q[t, h] * self.scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    want, size = p @ vv, p @ np.abs(vv)
                    # a score is a chain of d products and as many parts of a group; both it and the maximum enter an exponential
                    steps = np.abs(kk).max() * np.abs(q[t, h]).sum() * abs(self.scale)
                    allowed = HALF[self.dtype] * np.abs(want) + (2 * (d + 16) * 2.0 ** -23 * steps + (64 + seen.sum() / 16) * 2.0 ** -23) * size
                    if self.dtype == BF and n * (nh // nkv) >= 64 and d <= 128 and self.scale > 0:
                        # many rows: float16 operands.  A probability and a value are off by 2^-11 of themselves (values by 2^-25 of the largest at least),
                        # a key by that in every product of a score
                        allowed = allowed + (2 + 2 * float((p * (np.abs(kk) @ np.abs(q[t, h]))).sum() * self.scale)) * 2.0 ** -11 * size + 2.0 ** -25 * np.abs(vv).max()
                    elif self.dtype == BF:     # the probabilities' rounding, by themselves and times a group's scale, for both parts of m + s code
                        allowed = allowed + 2 * 2.0 ** -8 * (p @ parts[page, :, j % self.ps][seen, g])
                    off = np.abs(got[t, h] - want)
                    assert np.all(off <= allowed), (b, i, h, (off / allowed).max())
        assert np.all(got[self.start[-1]:] == 9)               # rows behind the last request


LAYOUTS = [(4, 2, 128), (8, 8, 64), (8, 1, 128), (32, 2, 128), (6, 2, 48), (5, 5, 80), (9, 3, 96), (4, 1, 256), (12, 4, 32), (3, 1, 20), (40, 1, 64), (10, 2, 128)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,d", LAYOUTS)
@pytest.mark.parametrize("news,contexts", [([1], [0]), ([1], [15]), ([1, 1, 1, 1], [16, 200, 0, 63]), ([3, 0, 1, 17], [40, 9, 130, 0])])
def test_attention(news, contexts, nh, nkv, d, dtype):
    a = Attend(news, contexts, nh, nkv, d, dtype)
    a.run()
    a.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ps", [1, 5, 8, 16, 32, 64, 128])
@pytest.mark.parametrize("window", [None, 1, 17, 100])
def test_pages_and_windows(ps, window, dtype):
    a = Attend([1, 5, 2], [150, 60, 3], 4, 2, 64, dtype, ps=ps, window=window)
    a.run()
    a.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("news,contexts", [([70], [0]), ([33, 1, 100], [500, 700, 28]), ([129], [300]), ([1], [3000]), ([1] * 40, list(range(0, 400, 10)))])
def test_more_tokens(news, contexts, dtype):
    a = Attend(news, contexts, 4, 1, 128, dtype)
    a.run()
    a.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("apart", [1, 8, 40])
def test_rows_that_lie_apart(apart, dtype):
    a = Attend([3, 20], [50, 30], 4, 2, 128, dtype, apart=apart)
    a.run()
    a.check()
    assert bool((a.out_rows[:, :apart] == 9).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_scales(scale, dtype):
    a = Attend([1, 4], [100, 37], 4, 2, 128, dtype, scale=scale)
    a.run()
    a.check()


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e3, 1e6])
def test_magnitudes(size):
    a = Attend([1, 6], [100, 37], 8, 2, 128, BF, size=size, scale=0.1 / size)
    a.run()
    a.check()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_what_the_longest_request_is_said_to_be_changes_nothing(dtype):
    a = Attend([2, 40, 1], [100, 37, 70], 4, 2, 128, dtype)
    for longest in (1, 2, 40, None, 1000):
        a.run(longest)
        a.check()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_requests_shorter_than_their_tokens(dtype):
    """A length below the number of tokens: the first tokens stand before the beginning and see nothing."""
    a = Attend([4, 2], [0, 30], 4, 2, 128, dtype)
    a.lengths[0] = 2
    a.run()
    a.check()
    a.lengths[0] = 0
    a.run()
    a.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d,ps", [(128, 16), (48, 5)])
def test_pages_outside_the_pool(d, ps, dtype):
    from xinfer_b200 import kernels as k
    a = Attend([1, 3], [50, 200], 4, 2, d, dtype, ps=ps)
    a.table[1, 2], a.table[1, 4] = a.pages, -7
    a.run(err=k.ERR_BAD_PAGE)
    good = a.table.copy()
    a.table[1, 2] = a.table[1, 4] = 0
    a.check(hidden=lambda b, j: b == 1 and good[1, j // ps] in (a.pages, -7))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_lengths_beyond_the_table(dtype):
    from xinfer_b200 import kernels as k
    a = Attend([1], [31], 4, 2, 128, dtype)
    a.table = a.table[:, :2]
    a.lengths[0] = 1000
    a.run(err=k.ERR_BAD_PAGE)
    assert bool(torch.isfinite(a.out).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d,ps", [(128, 16), (64, 32), (48, 8)])
def test_what_is_not_seen_does_not_matter(d, ps, dtype):
    """Words of NaN behind a request's end, in front of its window and between a prompt's tokens reach nobody who does not see them."""
    a = Attend([1, 20], [100, 45], 4, 2, d, dtype, ps=ps, window=40)
    want = a.run().clone()
    groups = -(-d // 32)
    for data in a.data:
        words = data[..., groups * ps * 16:].reshape(a.pages, 2, ps, groups, 4)
        for b, length in enumerate(a.lengths):
            for j in list(range(0, length - a.news[b] - 40 + 1)) + list(range(length, -(-length // ps) * ps)):
                words[a.table[b, j // ps], :, j % ps] = 0xFF
    assert torch.equal(a.run(), want)
    # the prompt's last key: its own token sees it, the others do not
    for data in a.data:
        words = data[..., groups * ps * 16:].reshape(a.pages, 2, ps, groups, 4)
        words[a.table[1, 64 // ps], :, 64 % ps] = 0xFF
    got = a.run()
    assert torch.equal(got[:20], want[:20]) and bool(torch.isnan(got[20]).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("longest", [1, 3, 60])
def test_graphs_and_streams(longest, dtype):
    from xinfer_b200 import kernels as k
    a, other = (Attend([1, longest, 1], c, 8, 2, 128, dtype, seed=3) for c in ([900, 33, 128], [5, 333, 600]))
    wants = [x.run().clone() for x in (a, other)]
    caches, lengths, start, table = a.tensors()
    more = [torch.zeros((max(a.pages, other.pages), *c.shape[1:]), dtype=torch.uint8, device=DEV) for c in caches]
    table = i32(np.full((3, 80), -1))
    out = torch.full_like(a.out, 9.0)
    need = k.cache4_attention_scratch(out.shape[0], 3, 8, 2, 128, dtype, longest)
    scratch = torch.zeros(max(1, need), device=DEV)

    def call():
        k.cache4_attention(out, a.q, *more, lengths, start, table, 16, a.scale, a.err, scratch=scratch, longest=longest)

    def load(x):
        for m, c in zip(more, x.tensors()[0]):
            m[:len(c)] = c
        lengths.copy_(i32(x.lengths))
        table[:, :x.table.shape[1]] = i32(x.table)
        a.q.copy_(x.q)

    load(a)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call()
    stream.synchronize()
    assert torch.equal(out, wants[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
        call()
    for x, want in ((other, wants[1]), (a, wants[0])):
        load(x)
        out.fill_(9.0)
        graph.replay()
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_calls_at_once(dtype):
    """Calls on streams of their own, with scratch of their own: steps of single tokens, of portions, of both."""
    from xinfer_b200 import kernels as k
    calls = [Attend(news, contexts, 8, 2, 128, dtype, seed=i) for i, (news, contexts) in enumerate((([1] * 6, [700] * 6), ([130], [400]), ([1, 90, 1], [300, 20, 900]), ([40], [0])))]
    wants, runs = [x.run().clone() for x in calls], []
    for x in calls:
        caches, lengths, start, table = x.tensors()
        longest = max(x.news)
        scratch = torch.zeros(max(1, k.cache4_attention_scratch(x.q.shape[0], len(x.news), 8, 2, 128, dtype, longest)), device=DEV)
        runs.append(dict(out=x.out, q=x.q, k_cache=caches[0], v_cache=caches[1], lengths=lengths, token_start=start, block_table=table, page_size=x.ps, scale=x.scale, err=x.err,
                         scratch=scratch, longest=longest))
        x.out.fill_(9.0)
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    for _ in range(5):
        for run, stream in zip(runs, streams):
            with torch.cuda.stream(stream):
                k.cache4_attention(**run)
    torch.cuda.synchronize()
    for x, want in zip(calls, wants):
        assert torch.equal(x.out, want) and int(x.err) == 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("news", [[3, 3], [70, 70]])
def test_requests_of_the_same_pages(news, dtype):
    a = Attend(news, [50, 50], 8, 2, 128, dtype)
    a.table[1] = a.table[0]
    a.run()
    a.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("tokens", [1, 70])
def test_batches_with_nobody_in_them(tokens, dtype):
    """Requests without tokens (their lengths and rows of the table are anything), steps without tokens, steps without requests."""
    from xinfer_b200 import kernels as k
    a = Attend([tokens], [100], 8, 2, 128, dtype)
    caches, _, _, table = a.tensors()
    tables = torch.full((5, table.shape[1]), 2 ** 30, dtype=torch.int32, device=DEV)
    tables[2] = table[0]
    lengths, start = i32([0, 2 ** 31 - 1, a.lengths[0], -5, 77]), i32([0, 0, 0, tokens, tokens, tokens])
    scratch = torch.zeros(max(1, k.cache4_attention_scratch(a.q.shape[0], 5, 8, 2, 128, dtype, tokens)), device=DEV)
    a.out.fill_(9.0)
    k.cache4_attention(a.out, a.q, *caches, lengths, start, tables, a.ps, a.scale, a.err, scratch=scratch, longest=tokens)
    # (how often a row's keys are shared out goes by the number of requests, so the bits may be others than those of the request alone)
    a.check()
    assert bool((a.out[tokens:] == 9).all()) and int(a.err) == 0
    k.cache4_attention(a.out[:0], a.q[:0], *caches, lengths, i32([0] * 6), tables, a.ps, a.scale, a.err, scratch=scratch)
    k.cache4_attention(a.out.fill_(9.0), a.q, *caches, lengths[:0], start[:1], tables[:0], a.ps, a.scale, a.err, scratch=scratch)
    k.cache4_attention(a.out, a.q, *caches, lengths, i32([0] * 6), tables, a.ps, a.scale, a.err, scratch=scratch)
    assert bool((a.out == 9).all()) and int(a.err) == 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("news,d,ps", [([1, 2], 128, 8), ([1, 100], 128, 8), ([1, 100], 64, 16), ([3, 70], 48, 5)])
def test_pages_that_a_window_has_left_behind(news, d, ps, dtype):
    """Their entries of the table are gone: nobody reads them and nothing is reported."""
    a = Attend(news, [300, 333], 4, 2, d, dtype, ps=ps, window=37)
    for b, length in enumerate(a.lengths):
        a.table[b, :max(0, length - news[b] - 37 + 1) // ps] = -1
    good = a.table.copy()
    a.run()
    a.table = np.maximum(good, 0)
    a.check()


@pytest.mark.parametrize("news,contexts,nh,nkv,d,window", [([200], [0], 4, 1, 128, None), ([64, 300], [700, 90], 8, 2, 128, None), ([130, 1, 70, 0, 2], [65, 500, 3, 8, 1000], 6, 2, 96, None),
                                                           ([90], [1000], 8, 8, 64, 100), ([257, 65], [31, 64], 3, 1, 32, 300), ([100, 5], [128, 900], 5, 1, 80, 77), ([80], [50], 2, 1, 256, None),
                                                           ([500] * 3, [3000, 10, 600], 16, 8, 48, None), ([12, 3, 4, 15, 0], [200, 900, 31, 0, 9], 8, 2, 128, None),
                                                           ([11, 4, 1], [70, 333, 800], 8, 2, 128, 100), ([3, 16, 2], [64, 40, 500], 16, 1, 64, None)])
@pytest.mark.parametrize("ps", [16, 4, 24])
def test_portions_of_prompts(news, contexts, nh, nkv, d, window, ps):
    a = Attend(news, contexts, nh, nkv, d, BF, ps=ps, window=window)
    a.run()
    a.check()


@pytest.mark.parametrize("d,ps,window", [(128, 16, 40), (64, 8, None), (96, 16, 200)])
def test_portions_do_not_meet_what_they_do_not_see(d, ps, window):
    """As above for tokens of a portion: a key of NaN reaches its own token and those behind it, a value's group of NaN its channels there."""
    a = Attend([150, 3], [200, 45], 4, 2, d, BF, ps=ps, window=window)
    want = a.run().clone()
    groups = -(-d // 32)
    words = [data[..., groups * ps * 16:].reshape(a.pages, 2, ps, groups, 4) for data in a.data]
    for w in words:                              # behind the end
        for b, length in enumerate(a.lengths):
            for j in range(length, -(-length // ps) * ps):
                w[a.table[b, j // ps], :, j % ps] = 0xFF
    assert torch.equal(a.run(), want)
    j = 310                                      # token 110 of the first request
    words[1][a.table[0, j // ps], 1, j % ps, 1] = 0xFF
    got = a.run()
    last = min(150, 110 + (window or 1000))
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[110:last, 2:, 32:64] = True
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], want[~bad])
    words[1][a.table[0, j // ps], 1, j % ps, 1] = 0
    words[0][a.table[0, j // ps], 0, j % ps] = 0xFF
    got = a.run()
    assert bool(torch.isnan(got[110:last, :2]).all()) and torch.equal(got[:110], want[:110]) and torch.equal(got[last:150, :2], want[last:150, :2])
    assert torch.equal(got[150:], want[150:])


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1e3, 1e6])
def test_magnitudes_of_portions(size):
    a = Attend([100], [137], 8, 2, 128, BF, size=size, scale=0.1 / size)
    a.run()
    a.check()


def test_refusals():
    from xinfer_b200 import kernels as k
    a = Attend([1, 2], [30, 40], 4, 2, 64, BF)
    caches, lengths, start, table = a.tensors()
    room = k.cache4_attention_scratch(a.q.shape[0], 2, 4, 2, 64, BF) + 4
    good = dict(out=a.out, q=a.q, k_cache=caches[0], v_cache=caches[1], lengths=lengths, token_start=start, block_table=table, page_size=16, scale=0.1, err=a.err,
                scratch=torch.zeros(room, device=DEV))

    def refused(**change):
        with pytest.raises(k.KernelError):
            k.cache4_attention(**{**good, **change})

    k.cache4_attention(**good)
    refused(out=a.out.float()), refused(q=a.q.half()), refused(k_cache=caches[0].int()), refused(v_cache=caches[1][:-1]), refused(lengths=lengths.long())
    refused(token_start=start[:-1]), refused(block_table=table[:1]), refused(page_size=8), refused(page_size=0), refused(window=0), refused(longest=0)
    refused(q=a.q[:, :3], out=a.out[:, :3]), refused(scratch=torch.zeros(4, device=DEV)), refused(scratch=torch.zeros(room, device=DEV)[1:]), refused(err=a.err.long()), refused(err=a.err[:0]), refused(scale=float("nan")), refused(scale=float("inf"))
    refused(lengths=lengths.cpu()), refused(q=a.q.cpu()), refused(block_table=table.expand(2, table.shape[1])[:, ::2])
    w = Write(3, 4, 2, 64, BF, 16)
    base = dict(q_out=w.q_out, k_cache=w.caches[0], v_cache=w.caches[1], qkv=w.qkv, positions=w.positions, slots=w.slots, page_size=16, err=w.err, cos=w.cos, sin=w.sin)

    def not_written(**change):
        with pytest.raises(k.KernelError):
            k.cache4_write(**{**base, **change})

    k.cache4_write(**base)
    not_written(q_out=w.q_out.float()), not_written(k_cache=w.caches[0][:, :1]), not_written(qkv=w.qkv[:, :-1]), not_written(qkv=w.qkv.half()), not_written(slots=w.slots.int())
    not_written(positions=w.positions.long()), not_written(page_size=8), not_written(cos=None), not_written(sin=w.sin[:4]), not_written(q_norm=torch.ones(32, device=DEV))
    not_written(values=(w.values[0].float(), w.values[1])), not_written(cos=torch.zeros(5, 33, device=DEV), sin=torch.zeros(5, 33, device=DEV))
    not_written(slots=w.slots.cpu()), not_written(positions=w.positions[:-1]), not_written(err=w.err[:0])


# ---- a run of steps ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F32])
def test_steps_of_a_layer(dtype):
    """Prompts in portions, then single tokens, of three requests: products with 4-bit weights, slots from the device, the cache, attention and
    the way back, beside the same layer on whole sequences in 64 bits from the values that the codes stand for."""
    from xinfer_b200 import kernels as k
    from xinfer_b200.weights import pack4
    nh, nkv, d, hidden, ps, B = 8, 2, 64, 256, 16, 3
    gen = torch.Generator(device=DEV).manual_seed(5)
    rand = lambda *s: torch.randn(s, generator=gen, device=DEV)  # noqa: E731
    w_qkv, w_o = pack4(rand((nh + 2 * nkv) * d, hidden) / 16, 64), pack4(rand(hidden, nh * d) / 22, 32)
    norms = [1 + 0.1 * rand(d) for _ in range(2)]
    angle = torch.arange(256, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    cos, sin = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
    caches = [torch.zeros((40, nkv, k.cache4_page_bytes(ps, d)), dtype=torch.uint8, device=DEV) for _ in range(2)]
    table, err = i32(np.full((B, 14), -1)), i32([0])
    state = [i32([0] * B), i32(np.random.default_rng(1).permutation(40)), i32([3, 40])]       # lengths, free pages, ring
    history = [[] for _ in range(B)]               # per request: rows of x
    for news in ([33, 0, 7], [40, 90, 0], [1, 20, 1], [1, 1, 1], [1, 1, 1], [0, 1, 1]):
        T = sum(news)
        x = rand(T, hidden).to(dtype)
        slots, pos, req, start = torch.zeros(T, dtype=torch.int64, device=DEV), i32([0] * T), i32([0] * T), i32([0] * (B + 1))
        after = [torch.zeros_like(state[0]), torch.zeros_like(state[2])]
        k.cache_slots(slots, pos, req, start, after[0], after[1], table, state[1], state[2], state[0], i32(news), ps, err)
        qkv = torch.zeros((T, (nh + 2 * nkv) * d), dtype=dtype, device=DEV)
        q, o, y = torch.zeros((T, nh, d), dtype=dtype, device=DEV), torch.zeros((T, nh, d), dtype=dtype, device=DEV), torch.zeros((T, hidden), dtype=dtype, device=DEV)
        room = lambda n: torch.zeros(max(1, n), device=DEV)  # noqa: E731
        k.linear4(qkv, x, w_qkv, scratch=room(k.linear4_scratch(T, qkv.shape[1], hidden, dtype)))
        k.cache4_write(q, *caches, qkv, pos, slots, ps, err, q_norm=norms[0], k_norm=norms[1], cos=cos, sin=sin)
        k.cache4_attention(o, q, *caches, after[0], start, table, ps, 0.125, err, longest=max(news),
                           scratch=room(k.cache4_attention_scratch(T, B, nh, nkv, d, dtype, max(news))))
        k.linear4(y, o.view(T, -1), w_o, scratch=room(k.linear4_scratch(T, hidden, nh * d, dtype)))
        state[0], state[2] = after
        assert int(err) == 0 and pos.tolist() == sum([list(range(len(h), len(h) + n)) for h, n in zip(history, news)], [])
        # the same in 64 bits from the step's own queries and the cache's codes; then the way back
        vals = [fourbit.page_values(c.cpu().numpy(), ps, d) for c in caches]
        at, rows = 0, table.cpu().numpy()
        for b, n in enumerate(news):
            before = len(history[b])
            history[b] += [None] * n
            j = np.arange(before + n)
            kk, vv = (v[rows[b][j // ps], :, j % ps] for v in vals)
            for i in range(n):
                for h in range(nh):
                    s = kk[:before + i + 1, h // 4] @ q[at + i, h].double().cpu().numpy() * 0.125
                    p = np.exp(s - s.max())
                    want = p @ vv[:before + i + 1, h // 4] / p.sum()
                    # bfloat16: three roundings of 2^-8 (probability, its product with a scale, result) of numbers up to three times a value's size
                    assert np.abs(o[at + i, h].double().cpu().numpy() - want).max() <= (0.03 if dtype == BF else 1e-5) * np.abs(vv).max()
            at += n
        want = o.view(T, -1).double() @ torch.from_numpy(fourbit.weight_values(w_o.cpu().numpy(), 32, hidden, nh * d)).to(DEV).T
        assert float((y.double() - want).abs().max()) <= (2.0 ** -7 if dtype == BF else 1e-5) * float(want.abs().max())
