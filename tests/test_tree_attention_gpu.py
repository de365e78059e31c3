"""Attention of trees of drafted tokens over the paged cache: against 64 bits, over types, head layouts, lengths, windows, pages and
masks, and what it does not see or refuses."""
import math

import numpy as np
import pytest
import torch

from tree_cases import tree, words_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731


class Step:
    """Requests with cached keys and drafted trees; what no request owns holds NaN."""

    def __init__(self, nodes, contexts, nh, nkv, d, ps, dtype=torch.bfloat16, seed=0, kind="mixed", words=None, sharp=1.5):
        rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.nodes, self.contexts, self.nh, self.nkv, self.d, self.ps, self.dtype = nodes, contexts, nh, nkv, d, ps, dtype
        B, T = len(nodes), sum(nodes)
        per = max(1, max(-(-c // ps) for c in contexts))
        self.table = torch.randperm(B * per + 3, generator=g)[: B * per].int().view(B, per)
        self.kc = torch.full((B * per + 3, nkv, ps, d), float("nan"), dtype=dtype)
        self.vc = self.kc.clone()
        self.q = (torch.randn(T, nh, d, generator=g) * sharp).to(dtype)
        self.kn, self.vn = (torch.randn(T, nkv, d, generator=g).to(dtype) for _ in range(2))
        for b, n in enumerate(contexts):
            for i in range(n):
                at = self.table[b, i // ps], slice(None), i % ps
                self.kc[at], self.vc[at] = torch.randn(nkv, d, generator=g).to(dtype), torch.randn(nkv, d, generator=g).to(dtype)
        words = words or max(1, -(-max(nodes) // 32))
        self.depth, self.on, masks = [], [], []
        for n in nodes:
            _, dep, on = tree(rng, n, kind)
            self.depth += dep
            self.on.append(on)
            masks.append(words_of(on, words).view(n, words))
        self.ancestors = torch.cat(masks)
        self.start = [0] + list(np.cumsum(nodes))
        self.scale = d ** -0.5

    def run(self, window=None, out=None, q=None, kn=None, vn=None, token_start=None):
        from xinfer_b200 import kernels as k
        T = self.q.shape[0]
        dev = lambda t, own: t.to(DEV) if own is None else own  # noqa: E731
        out = torch.full((T, self.nh, self.d), 7.0, dtype=self.dtype, device=DEV) if out is None else out
        self.err = torch.zeros(1, dtype=torch.int32, device=DEV)
        need = k.tree_attention_scratch(T, self.nh, self.nkv, self.d, self.dtype)
        scratch = torch.full((max(need, 1),), float("nan"), device=DEV)
        k.tree_attention(out, dev(self.q, q), dev(self.kn, kn), dev(self.vn, vn), self.kc.to(DEV), self.vc.to(DEV), i32(self.contexts),
                         i32(token_start or [int(x) for x in self.start]), self.ancestors.to(DEV), self.table.to(DEV), self.scale, self.err, scratch=scratch,
                         depth=i32(self.depth), window=window)
        return out

    def check(self, out, window=None):
        """The bound: float32 sums of d products move a score by at most (d + 8) 2^-24 of the sum of the products' sizes, and that moves
        the weights by twice as much; a sum over the keys by (keys + 16) 2^-24 of its terms.  In bfloat16 also half a unit in the eighth
        digit of every weight (2^-9, once in its own sum: 2^-8), 2^-13 for exponentials and half a unit of the result."""
        G = self.nh // self.nkv
        for b, (n, c) in enumerate(zip(self.nodes, self.contexts)):
            if not n:
                continue
            a = self.start[b]
            j = torch.arange(c)
            kc, vc = (t[self.table[b, j // self.ps].long(), :, j % self.ps].double() for t in (self.kc, self.vc))
            k, v = torch.cat([kc, self.kn[a:a + n].double()]), torch.cat([vc, self.vn[a:a + n].double()])
            dep = torch.tensor(self.depth[a:a + n])
            seen = torch.cat([torch.ones(n, c, dtype=torch.bool), torch.from_numpy(self.on[b])], 1)
            if window:
                seen &= (c + dep)[:, None] - torch.cat([j, c + dep])[None] < window
            k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
            q = self.q[a:a + n].double()
            s = torch.einsum("nhd,khd->nhk", q, k) * self.scale
            size = torch.einsum("nhd,khd->nhk", q.abs(), k.abs()).mul(self.scale).nan_to_num(0.0).masked_fill(~seen[:, None], 0.0).amax(2, keepdim=True) if c + n else None
            w = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), 2).nan_to_num(0.0)
            v0 = v.nan_to_num(0.0, 0.0, 0.0)
            ref, terms = torch.einsum("nhk,khd->nhd", w, v0), torch.einsum("nhk,khd->nhd", w, v0.abs())
            rel = 2 * (self.d + 8) * 2.0 ** -24 * size + (c + n + 16) * 2.0 ** -24
            bound = rel * terms
            if self.dtype == torch.bfloat16:
                bound = (rel + 2.0 ** -8 + 2.0 ** -13) * terms + 2.0 ** -8 * ref.abs()
            got = out[a:a + n].double().cpu()
            assert ((got - ref).abs() <= bound + 1e-30).all(), (b, n, c, ((got - ref).abs() - bound).max())


LAYOUTS = [  # nodes, contexts, query heads, key/value heads, channels, page, window
    ([1], [1], 1, 1, 64, 16, None), ([1], [0], 4, 2, 128, 16, None), ([16], [1024], 16, 8, 128, 16, None), ([64, 64], [65, 700], 32, 8, 128, 16, None),
    ([5, 0, 1, 33], [17, 100, 0, 64], 8, 2, 64, 16, None), ([100, 3], [300, 2000], 8, 1, 128, 32, None), ([7, 65], [128, 129], 10, 5, 48, 8, None),
    ([13, 20], [63, 1], 6, 2, 96, 64, None), ([31, 32], [15, 16], 20, 4, 80, 16, None), ([12, 9], [200, 31], 12, 1, 112, 16, None), ([40], [90], 24, 1, 128, 16, None),
    ([8, 30], [500, 77], 8, 2, 128, 16, 50), ([64, 2], [64, 400], 4, 1, 64, 16, 1), ([90, 17], [1000, 3], 16, 4, 128, 8, 5), ([6], [40], 4, 2, 128, 16, 200),
    ([3, 129], [10, 257], 3, 3, 128, 128, None), ([11], [50], 4, 2, 128, 12, None), ([9, 4], [33, 70], 4, 2, 256, 16, None), ([5], [21], 6, 3, 40, 16, 9), ([2, 6], [4096, 1500], 32, 8, 128, 16, None)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes,contexts,nh,nkv,d,ps,window", LAYOUTS)
def test_against_64_bits(nodes, contexts, nh, nkv, d, ps, window, dtype):
    s = Step(nodes, contexts, nh, nkv, d, ps, dtype, seed=sum(nodes) + d)
    out = s.run(window)
    assert int(s.err) == 0
    s.check(out, window)
    assert torch.equal(out, s.run(window))                 # no order of additions that changes


@pytest.mark.parametrize("kind", ["chain", "star"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_chains_and_stars(kind, dtype):
    s = Step([70, 64], [100, 64], 8, 4, 128, 16, dtype, kind=kind, words=5)
    s.check(s.run(20), 20)
    s.check(s.run())


def test_a_chain_is_causal_attention():
    """Tokens in a chain see what the tokens of a prompt see."""
    from xinfer_b200 import kernels as k
    s = Step([50], [0], 8, 2, 128, 16, torch.float32, kind="chain")
    cache = torch.zeros(4, 2, 16, 128)
    values = cache.clone()
    for i in range(50):
        cache[i // 16, :, i % 16], values[i // 16, :, i % 16] = s.kn[i], s.vn[i]
    ref = torch.empty(50, 8, 128, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    k.attention_plain(ref, s.q.to(DEV), cache.to(DEV), values.to(DEV), i32(list(range(50))), i32([0] * 50), i32([[0, 1, 2, 3]]), 4, None, s.scale, err)
    # two float32 results of the same formula: both within the bound of `check`, a few 1e-6 of terms of size 1
    assert (s.run() - ref).abs().max() <= 2e-5
    assert int(err) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_whose_masks_leave_nothing(dtype):
    s = Step([40, 6, 70], [0, 30, 64], 8, 2, 128, 16, dtype)
    for b, row in ((0, 0), (0, 33), (2, 69), (2, 1)):
        s.on[b][row] = False
        s.ancestors[s.start[b] + row] = 0
    out = s.run()
    s.check(out)
    assert torch.count_nonzero(out[0]) == 0 and torch.count_nonzero(out[33]) == 0
    # bits behind a tree's last node mean nothing
    s.ancestors[:, -1] |= torch.tensor(-2 ** 31, dtype=torch.int32)
    assert torch.equal(out, s.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", ["key", "value", "both"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_a_token_does_not_see_is_not_in_its_result(dtype, what, bad):
    """Drafted tokens that are not finite reach the tokens below them and nobody else, beside others in the same tile and as a first one."""
    s = Step([70, 20, 9], [0, 100, 50], 8, 2, 128, 16, dtype, kind="mixed")
    spoiled = [(0, 5), (0, 66), (1, 3), (1, 19), (2, 0)]
    clean = s.run()
    for b, i in spoiled:
        for t in ([s.kn] if what == "key" else [s.vn] if what == "value" else [s.kn, s.vn]):
            t[s.start[b] + i, 1, 7] = bad
    out = s.run()
    assert int(s.err) == 0
    touched = torch.zeros(sum(s.nodes), dtype=torch.bool)
    for b, i in spoiled:
        touched[s.start[b]:s.start[b + 1]] |= torch.from_numpy(s.on[b][:, i])
    assert torch.equal(out[~touched], clean[~touched])
    assert torch.equal(out[:, :4], clean[:, :4])            # the heads of the other key/value head
    if what == "value":
        assert not torch.isfinite(out[touched][:, 4:, 7]).any()
        rest = [c for c in range(128) if c != 7]
        s.vn.nan_to_num_(0.0, 0.0, 0.0)
        fine = out.clone()
        fine[:, 4:, 7] = s.run()[:, 4:, 7]
        s.check(fine)
        assert torch.isfinite(out[:, :, rest]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_outside_a_window_are_not_in_the_result(dtype):
    """A cached row that shallow tokens see and deeper ones do not."""
    s = Step([30], [100], 8, 2, 128, 16, dtype, kind="chain")
    at = s.table[0, 90 // 16], 0, 90 % 16
    clean = s.run(20)
    s.vc[at] = float("nan")
    out = s.run(20)
    sees = 100 + torch.tensor(s.depth) - 90 < 20
    assert sees.any() and not sees.all()
    assert torch.equal(out[~sees], clean[~sees]) and torch.isnan(out[sees][:, :4]).all() and torch.equal(out[:, 4:], clean[:, 4:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gap", [0, 8, 24, 3])
def test_tokens_that_lie_apart(dtype, gap):
    """Queries, keys and values as columns of one projection's rows, and a result between other columns."""
    s = Step([33, 8], [40, 129], 8, 2, 64, 16, dtype)
    T, nh, nkv, d = 41, 8, 2, 64
    rows = torch.full((T, (nh + 2 * nkv) * d + gap), float("nan"), dtype=dtype)
    rows[:, : nh * d], rows[:, nh * d:(nh + nkv) * d] = s.q.view(T, -1), s.kn.view(T, -1)
    rows[:, (nh + nkv) * d:(nh + 2 * nkv) * d] = s.vn.view(T, -1)
    rows = rows.to(DEV)
    q, kn, vn = (rows[:, a * d:z * d].view(T, z - a, d) for a, z in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
    wide = torch.full((T, nh * d + gap), 5.0, dtype=dtype, device=DEV)
    out = s.run(out=wide[:, : nh * d].view(T, nh, d), q=q, kn=kn, vn=vn)
    assert torch.equal(out, s.run()) and (wide[:, nh * d:] == 5.0).all()


def test_tokens_of_no_request_stay_as_they_are():
    s = Step([4, 6, 5], [20, 30, 40], 8, 2, 128, 16)
    full = s.run()
    s.nodes, s.contexts, s.table = s.nodes[1:2], s.contexts[1:2], s.table[1:2]
    out = s.run(token_start=[4, 10])
    assert torch.equal(out[4:10], full[4:10]) and (out[:4] == 7.0).all() and (out[10:] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bad_pages_and_lengths_are_reported(dtype):
    from xinfer_b200 import kernels as k
    s = Step([4, 4], [40, 40], 8, 2, 128, 16, dtype)
    fine = s.run()
    s.table[0, 1] = 10 ** 6
    out = s.run()
    assert int(s.err) == k.ERR_BAD_PAGE and torch.isfinite(out).all() and torch.equal(out[4:], fine[4:])
    s.table[0, 1] = -5
    s.run()
    assert int(s.err) == k.ERR_BAD_PAGE
    s = Step([4], [40], 8, 2, 128, 16, dtype)
    s.contexts = [10 ** 9]
    s.table[0, 2] = s.table[0, 1]
    s.run()
    assert int(s.err) == k.ERR_BAD_PAGE
    s.contexts = [-3]
    assert torch.isfinite(s.run()).all() and int(s.err) == 0


def test_on_another_stream_and_in_a_graph():
    s = Step([30, 64], [700, 90], 32, 8, 128, 16)
    want = s.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = s.run()
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    from xinfer_b200 import kernels as k
    s = Step([4], [40], 8, 2, 128, 16)
    q, kn, vn, kc, vc = (t.to(DEV) for t in (s.q, s.kn, s.vn, s.kc, s.vc))
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    args = dict(out=torch.empty_like(q), q=q, k_new=kn, v_new=vn, k_cache=kc, v_cache=vc, context=i32([40]), token_start=i32([0, 4]), ancestors=s.ancestors.to(DEV),
                block_table=s.table.to(DEV), scale=1.0, err=err, scratch=torch.empty(max(1, k.tree_attention_scratch(4, 8, 2, 128, torch.bfloat16)), device=DEV))
    k.tree_attention(**args)
    for change in (dict(q=s.q), dict(q=q.half()), dict(q=q[:, :7]), dict(out=torch.empty_like(q).transpose(0, 1)), dict(k_new=kn[:3]), dict(v_cache=vc[:1]),
                   dict(k_cache=kc.float()), dict(context=i32([40, 1])), dict(token_start=i32([0])), dict(ancestors=s.ancestors), dict(block_table=i32([0])),
                   dict(window=3), dict(window=0, depth=i32(s.depth)), dict(window=3, depth=i32([1])), dict(context=torch.tensor([40], device=DEV)), dict(err=None)):
        with pytest.raises(k.KernelError):
            k.tree_attention(**{**args, **change})
    assert int(err) == 0


MORE = [  # as above
    ([3, 0, 1, 7, 20] * 20, [0, 50, 130, 64, 9] * 20, 8, 2, 64, 16, None), ([2, 1, 0] * 30, [700, 3, 40] * 30, 4, 4, 128, 32, 33), ([1] * 70, list(range(70)), 4, 1, 32, 8, None),
    ([5, 9], [30, 300], 4, 2, 16, 16, None), ([2, 1], [40, 500], 128, 1, 64, 16, None), ([3], [100], 130, 1, 64, 16, None), ([10, 3], [700, 255], 8, 2, 128, 256, None),
    ([1024], [33], 2, 1, 64, 16, None), ([300, 1], [10, 1000], 8, 4, 64, 16, 40), ([12], [9000], 2, 2, 128, 16, None)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nodes,contexts,nh,nkv,d,ps,window", MORE)
def test_more_against_64_bits(nodes, contexts, nh, nkv, d, ps, window, dtype):
    test_against_64_bits(nodes, contexts, nh, nkv, d, ps, window, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", ["key", "value"])
def test_cached_rows_that_are_not_numbers_reach_every_node(dtype, what):
    s = Step([40, 5], [200, 90], 8, 2, 128, 16, dtype)
    clean = s.run()
    at = s.table[0, 150 // 16], 1, 150 % 16
    (s.kc if what == "key" else s.vc)[at] = float("nan")
    out = s.run()
    assert torch.isnan(out[:40, 4:]).all() and torch.equal(out[:, :4], clean[:, :4]) and torch.equal(out[40:], clean[40:]) and int(s.err) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_that_are_large(dtype):
    """Scores of several hundred, of either sign: the running maximum moves from tile to tile."""
    s = Step([20, 6], [300, 64], 8, 2, 64, 16, dtype, sharp=120.0)
    s.check(s.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_captured_call_follows_its_inputs(dtype):
    """The lengths and masks are the device's: one graph serves other requests of the same shapes."""
    from xinfer_b200 import kernels as k
    steps = [Step(n, c, 8, 2, 128, 16, dtype, seed=i, words=2) for i, (n, c) in enumerate((([30, 2], [300, 40]), ([1, 31], [0, 320]), ([16, 16], [170, 171])))]
    names = ("q", "kn", "vn", "kc", "vc", "ancestors", "table")
    pages, width = max(s.kc.shape[0] for s in steps), max(s.table.shape[1] for s in steps)

    def fitted(s):
        grow = lambda t: torch.cat([t, torch.full((pages - t.shape[0], *t.shape[1:]), float("nan"), dtype=t.dtype)])  # noqa: E731
        table = torch.zeros(2, width, dtype=torch.int32)
        table[:, :s.table.shape[1]] = s.table
        return [s.q, s.kn, s.vn, grow(s.kc), grow(s.vc), s.ancestors, table]

    at = dict(zip(names, (t.to(DEV) for t in fitted(steps[0]))))
    context, start = i32(steps[0].contexts), i32([int(x) for x in steps[0].start])
    out, err = torch.zeros(32, 8, 128, dtype=dtype, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    scratch = torch.empty(k.tree_attention_scratch(32, 8, 2, 128, dtype), device=DEV)
    call = lambda: k.tree_attention(out, at["q"], at["kn"], at["vn"], at["kc"], at["vc"], context, start, at["ancestors"], at["table"],  # noqa: E731
                                    steps[0].scale, err, scratch=scratch)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
        call()                     # one behind another on the same scratch
    for s in steps + steps[:1]:
        for name, t in zip(names, fitted(s)):
            at[name].copy_(t)
        context.copy_(i32(s.contexts))
        start.copy_(i32([int(x) for x in s.start]))
        out.fill_(7.0)
        graph.replay()
        s.check(out)
        assert torch.equal(out, s.run()) and int(err) == 0


def test_more_refusals():
    from xinfer_b200 import kernels as k
    dtype = torch.bfloat16
    q, kn = torch.zeros(4, 8, 64, dtype=dtype, device=DEV), torch.zeros(4, 2, 64, dtype=dtype, device=DEV)
    cache = torch.zeros(2, 2, 16, 64, dtype=dtype, device=DEV)
    need = k.tree_attention_scratch(4, 8, 2, 64, dtype)
    room = torch.empty(need + 4, device=DEV)
    args = dict(out=torch.empty_like(q), q=q, k_new=kn, v_new=kn, k_cache=cache, v_cache=cache, context=i32([20]), token_start=i32([0, 4]), ancestors=i32([[1]] * 4),
                block_table=i32([[0, 1]]), scale=1.0, err=i32([0]), scratch=room[:need])
    k.tree_attention(**args)
    wide = torch.zeros(2, 2, 1 << 20, 64, dtype=dtype, device=DEV)
    for change in (dict(scratch=room[:need - 1]), dict(scratch=room[1:need + 1]), dict(scratch=None), dict(scratch=room.bfloat16()),
                   dict(k_new=kn[:, :0], v_new=kn[:, :0]), dict(context=i32([0] * 8193)),
                   # requests whose tiles together might be more than 32 bits count
                   dict(k_cache=wide, v_cache=wide, context=i32([0] * 4000), token_start=i32([0] * 4001), block_table=torch.zeros(4000, 64, dtype=torch.int32, device=DEV))):
        with pytest.raises(k.KernelError):
            k.tree_attention(**{**args, **change})
    assert int(args["err"]) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window", [None, 30])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-41, -1e-41, 0.125])
def test_any_scale(dtype, window, scale):
    """A factor of zero weighs all keys that are seen alike, one below zero those of opposite queries; what is not seen stays out."""
    s = Step([33, 70, 1], [100, 700, 64], 8, 2, 64, 16, dtype)
    s.scale = scale
    out = s.run(window)
    assert int(s.err) == 0
    if scale < 0:                          # (the bound goes by the products' sizes)
        s.q, s.scale = -s.q, -scale
    s.check(out, window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [0, 2])
def test_a_cache_without_pages(dtype, width):
    """Trees behind nothing at all: no page has been made yet."""
    from xinfer_b200 import kernels as k
    s = Step([20, 70], [0, 0], 8, 2, 64, 16, dtype)
    s.kc, s.vc, s.table = s.kc[:0], s.vc[:0], torch.full((2, width), -1, dtype=torch.int32)
    s.check(s.run())
    assert int(s.err) == 0
    s.contexts = [5, 0]
    assert torch.isfinite(s.run()).all() and int(s.err) == k.ERR_BAD_PAGE
