"""Penalties, biases and grammar masks on logits against 64 bits."""
import numpy as np
import pytest
import torch

from tree_cases import tree, words_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731


def reference(logits, pen, lists, prompt, list_of_row, paths, biases, allowed):
    """Row by row in 64 bits; `bound`: a float32 rounding of every step's result."""
    R, V = logits.shape
    x = logits.astype(np.float64)
    bound = np.zeros_like(x)
    for r in range(R):
        rep, freq, pres = pen[r].astype(np.float64)
        li = list_of_row[r]
        toks = list(lists[li]) if 0 <= li < len(lists) else []
        m = max(0, prompt[li]) if toks else 0
        asked = {t for t in toks[:m]}
        said = toks[m:] + list(paths[r])
        for v in {t for t in asked | set(said) if 0 <= t < V}:
            c = said.count(v)
            x[r, v] = x[r, v] / rep if x[r, v] > 0 else x[r, v] * rep
            size = abs(x[r, v])
            if c:
                x[r, v] -= freq * c + pres
            bound[r, v] += 2.0 ** -23 * (size + abs(freq * c) + abs(pres))
        for v, add in biases[r]:
            if 0 <= v < V:
                bound[r, v] += 2.0 ** -23 * (abs(x[r, v]) + abs(add))
                x[r, v] += add
        if allowed[r] is not None:
            x[r, ~allowed[r]] = -np.inf
    return x, bound


def call(logits, pen, lists, prompt, list_of_row, first, drafted, anc, biases, masks, mask_of_row, out=None):
    from xinfer_b200 import kernels as k
    starts = np.concatenate([[0], np.cumsum([len(t) for t in lists])])
    flat = np.concatenate([np.asarray(t, dtype=np.int64) for t in lists] + [np.zeros(0, np.int64)])
    bias = None
    if biases is not None:
        bs = np.concatenate([[0], np.cumsum([len(b) for b in biases])])
        bias = (i32(bs), i32([v for b in biases for v, _ in b] or np.zeros(0)), torch.tensor([a for b in biases for _, a in b], dtype=torch.float32, device=DEV))
    dev = torch.tensor(logits, device=DEV) if out is None else out
    res = dev if out is not None else torch.full_like(dev, 99.0)
    k.logit_rules(res, dev, torch.tensor(pen, dtype=torch.float32, device=DEV), i32(flat), i32(starts), i32(prompt), list_of_row=i32(list_of_row),
                  tree=(i32(drafted), anc.to(DEV), i32(first)) if drafted is not None else None, bias=bias,
                  mask=masks.to(DEV) if masks is not None else None, mask_of_row=i32(mask_of_row) if mask_of_row is not None else None)
    return res


@pytest.mark.parametrize("vocab", [1, 5, 31, 33, 331, 1023, 5000, 8193, 40001, 151936])
@pytest.mark.parametrize("history", [0, 1, 40, 3000])
def test_against_64_bits(vocab, history):
    rng = np.random.default_rng(vocab + history)
    R, nodes = 7, 6                                        # a tree of six rows and a row by itself
    logits = (rng.normal(size=(R, vocab)) * 3).astype(np.float32)
    lists = [rng.integers(-1, min(vocab, 200) + 2, history).tolist() for _ in range(3)]
    lists.append([])
    prompt = [history // 2, 0, history, 0]
    list_of_row = [0, 0, 0, 1, 2, -1, 3]
    pen = np.stack([rng.choice([1.0, 1.3, 0.8], R), rng.choice([0.0, 0.5, -0.25], R), rng.choice([0.0, 0.7], R)], 1).astype(np.float32)
    _, _, on = tree(rng, nodes)
    drafted = rng.integers(0, min(vocab, 4), R)
    anc = torch.cat([words_of(on, 2), torch.zeros(1, 2, dtype=torch.int32)])
    first = [0] * nodes + [6]
    paths = [[int(drafted[i]) for i in range(nodes) if r < nodes and on[r, i]] for r in range(R)]
    biases = [[(int(v), float(a)) for v, a in zip(rng.integers(-1, vocab + 1, m), np.round(rng.normal(size=m), 3).astype(np.float32))] for m in (0, 1, 5, 0, 40, 3, 2)]
    W = (vocab + 31) // 32 + 1                             # masks may have words to spare
    bits = rng.random((3, W * 32)) < np.array([0.5, 0.02, 0.98])[:, None]
    masks = words_of(bits, W)
    mask_of_row = [0, 1, 2, -1, 1, 1, 9]                   # (a mask that is not there binds nothing)
    allowed = [bits[m, :vocab] if 0 <= m < 3 else None for m in mask_of_row]
    ref, bound = reference(logits, pen, lists, prompt, list_of_row, paths, biases, allowed)
    got = call(logits, pen, lists, prompt, list_of_row, first, drafted, anc, biases, masks, mask_of_row).double().cpu().numpy()
    assert np.array_equal(np.isneginf(got), np.isneginf(ref))
    fin = np.isfinite(ref)
    assert (np.abs(got[fin] - ref[fin]) <= bound[fin]).all()
    same = call(logits, pen, lists, prompt, list_of_row, first, drafted, anc, biases, masks, mask_of_row, out=torch.tensor(logits, device=DEV))
    assert np.array_equal(same.double().cpu().numpy(), got)


@pytest.mark.parametrize("vocab,gap,shift", [(500, 3, 0), (8200, 4, 0), (1000, 8, 1), (1001, 0, 0), (1001, 0, 3)])
def test_rows_that_lie_apart_and_start_anywhere(vocab, gap, shift):
    rng = np.random.default_rng(3)
    R = 5
    wide = torch.zeros(R * (vocab + gap) + 4, device=DEV).normal_()
    rows = wide[shift:shift + R * (vocab + gap)].view(R, vocab + gap)[:, :vocab]
    to = torch.full((R * (vocab + 2) + 4,), 5.0, device=DEV)
    out = to[1:1 + R * (vocab + 2)].view(R, vocab + 2)[:, :vocab]
    from xinfer_b200 import kernels as k
    lists = [rng.integers(0, vocab, 30).tolist() for _ in range(R)]
    pen = np.tile(np.float32([1.5, 0.25, 0.5]), (R, 1))
    bits = rng.random((R, (vocab + 31) // 32 * 32)) < 0.7
    k.logit_rules(out, rows, torch.tensor(pen, device=DEV), i32(np.concatenate(lists)), i32(np.arange(R + 1) * 30), i32([10] * R),
                  mask=words_of(bits, (vocab + 31) // 32).to(DEV))
    ref, bound = reference(rows.cpu().numpy(), pen, lists, [10] * R, list(range(R)), [[]] * R, [[]] * R, [b[:vocab] for b in bits])
    got = out.double().cpu().numpy()
    fin = np.isfinite(ref)
    assert np.array_equal(np.isneginf(got), ~fin) and (np.abs(got[fin] - ref[fin]) <= bound[fin]).all()
    assert int((to == 5.0).sum()) >= 4 + 2 * R


def test_logits_that_are_not_finite():
    """They stay what the formula makes of them; a token that the mask forbids is -inf whatever stood there."""
    from xinfer_b200 import kernels as k
    x = torch.tensor([[float("inf"), float("-inf"), float("nan"), 1.0, -3.4e38, float("nan"), float("inf"), -0.0]], device=DEV)
    out = torch.empty_like(x)
    mask = i32([[0b10011111]])
    k.logit_rules(out, x, torch.tensor([[2.0, 0.5, 0.25]], device=DEV), i32([0, 1, 2, 4, 7]), i32([0, 5]), i32([0]), mask=mask,
                  bias=(i32([0, 2]), i32([5, 3]), torch.tensor([float("inf"), 2.0], device=DEV)))
    got = out[0].tolist()
    assert got[0] == float("inf") and got[1] == float("-inf") and got[2] != got[2] and got[3] == 3.0 and got[4] == float("-inf")
    assert got[5] == got[6] == float("-inf") and got[7] == -0.75


def test_a_token_said_very_often_is_counted():
    from xinfer_b200 import kernels as k
    n = 100_000
    x = torch.ones(1, 9000, device=DEV)
    k.logit_rules(x, x, torch.tensor([[1.0, 0.5, 0.0]], device=DEV), torch.full((n,), 8999, dtype=torch.int32, device=DEV), i32([0, n]), i32([0]))
    assert float(x[0, 8999]) == 1.0 - 0.5 * n and bool((x[0, :8999] == 1.0).all())


def test_refusals():
    from xinfer_b200 import kernels as k
    x = torch.zeros(2, 64, device=DEV)
    args = dict(out=x, logits=x, penalties=torch.ones(2, 3, device=DEV), history=i32([1, 2]), history_start=i32([0, 1, 2]), prompt_len=i32([0, 0]))
    k.logit_rules(**args)
    f = torch.zeros(2, device=DEV)
    for change in (dict(logits=x.cpu()), dict(logits=x.bfloat16()), dict(out=x[:1]), dict(out=x.t().contiguous().t()), dict(penalties=torch.ones(2, 2, device=DEV)),
                   dict(history=torch.zeros(2, device=DEV)), dict(history_start=i32([0, 1])), dict(prompt_len=i32([0])), dict(list_of_row=i32([0])),
                   dict(tree=(i32([1]), i32([[1], [1]]), i32([0, 0]))), dict(tree=(i32([1, 1]), i32([1, 1]), i32([0, 0]))), dict(bias=(i32([0, 1]), i32([1]), f[:1])),
                   dict(bias=(i32([0, 1, 2]), i32([1, 2]), f[:1])), dict(mask=i32([[1, 1]])), dict(mask=i32([[1], [1]])), dict(mask_of_row=i32([0, 0])),
                   dict(mask=i32([[1, 1]]), mask_of_row=i32([0]))):
        with pytest.raises(k.KernelError):
            k.logit_rules(**{**args, **change})


def case_of_rows(rng, R, vocab, lists, list_of_row, paths=None, biases=None):
    logits = (rng.normal(size=(R, vocab)) * 3).astype(np.float32)
    pen = np.stack([rng.choice([1.0, 1.3, 0.8], R), rng.choice([0.0, 0.5], R), rng.choice([0.0, 0.7], R)], 1).astype(np.float32)
    prompt = [len(t) // 3 for t in lists]
    biases = biases or [[] for _ in range(R)]
    ref, bound = reference(logits, pen, lists, prompt, list_of_row, paths or [[]] * R, biases, [None] * R)
    return logits, pen, prompt, ref, bound


@pytest.mark.parametrize("vocab", [600, 5003, 70001])
@pytest.mark.parametrize("counts", [[700, 3], [100] * 20, [384, 1, 385, 0, 384], [0] * 60 + [90] * 9])
def test_many_biases(vocab, counts):
    """More than a block keeps at a time, of one row or of several, with tokens that are named more than once: their sum, in its order."""
    rng = np.random.default_rng(vocab + len(counts))
    R = len(counts)
    biases = [[(int(v), float(a)) for v, a in zip(rng.integers(-1, min(vocab, 2000) + 1, m), np.round(rng.normal(size=m), 2).astype(np.float32))] for m in counts]
    logits, pen, prompt, ref, bound = case_of_rows(rng, R, vocab, [[1, 2, 2, 5]] * R, list(range(R)), biases=biases)
    got = call(logits, pen, [[1, 2, 2, 5]] * R, prompt, list(range(R)), None, None, None, biases, None, None).double().cpu().numpy()
    # (the entries of a token are summed by themselves first: each of its roundings is of a number no larger than all their sizes together)
    for r, row in enumerate(biases):
        for v in {v for v, _ in row if 0 <= v < vocab}:
            mine = [abs(a) for w, a in row if w == v]
            bound[r, v] += 2.0 ** -23 * len(mine) * sum(mine)
    assert (np.abs(got - ref) <= bound).all()


@pytest.mark.parametrize("nodes,vocab", [([60, 60], 3001), ([700], 900), ([1024], 64), ([33, 1, 100], 20000), ([50] * 5, 1024)])
def test_large_trees_of_rows_that_share_a_list(nodes, vocab):
    rng = np.random.default_rng(sum(nodes))
    words = -(-max(nodes) // 32)
    drafted, masks, first, paths, list_of_row = [], [], [], [], []
    for b, n in enumerate(nodes):
        _, _, on = tree(rng, n)
        toks = rng.integers(-1, min(vocab, 6), n)
        paths += [[int(toks[i]) for i in np.flatnonzero(on[r])] for r in range(n)]
        first += [len(drafted)] * n
        drafted += toks.tolist()
        masks.append(words_of(on, words))
        list_of_row += [b] * n
    lists = [rng.integers(0, min(vocab, 10), 50).tolist() for _ in nodes]
    logits, pen, prompt, ref, bound = case_of_rows(rng, len(drafted), vocab, lists, list_of_row, paths)
    got = call(logits, pen, lists, prompt, list_of_row, first, drafted, torch.cat(masks), None, None, None).double().cpu().numpy()
    assert (np.abs(got - ref) <= bound).all()


def test_places_that_make_no_sense_reach_nothing():
    """Starts that do not ascend, lists, rows and masks that are not there: what they name is passed over."""
    from xinfer_b200 import kernels as k
    x = torch.randn(3, 500, device=DEV)
    values = torch.ones(5, device=DEV)
    for starts in ([0, 1000, 5, 5], [0, 5, 0, 0], [-7, 2, 10 ** 9, 2], [5, 0, 0, 0]):
        out = torch.full_like(x, 9.0)
        k.logit_rules(out, x, torch.tensor([[1.0, 0.0, 0.0]] * 3, device=DEV), i32([1, 2]), i32([0, 2 ** 30]), i32([-5]), list_of_row=i32([0, 7, -9]),
                      tree=(i32([1, 2, 3]), i32([[-1], [-1], [-1]]), i32([-3, 2, 10 ** 9])), bias=(i32(starts), i32([0, 1, 2, 3, 4]), values))
        for r in range(3):
            # what lies outside the ascending part is not said by the rule, but every number is the logit or the logit and its bias
            there = (out[r] == x[r]) | (out[r] == x[r] + 1.0)
            assert bool(there.all()) and bool((out[r, 5:] == x[r, 5:]).all())


def edge_tokens(vocab):
    """Tokens around the places where one warp's tokens end and the next one's begin, and those around the chunks' ends."""
    at = [e + i for e in range(128, vocab, 128) for i in range(-2, 4)] + [c + i for c in range(1024, vocab, 1024) for i in range(-4, 1)] + [vocab - 1 - i for i in range(4)]
    return np.array(sorted({t for t in at if 0 <= t < vocab}))


@pytest.mark.parametrize("vocab,gap,trees", [(3001, 0, 2), (3001, 2, 2), (40001, 0, 2), (40001, 1, 2), (50257, 0, 8), (3001, 3, 2), (331, 0, 3)])
def test_paths_of_rows_that_start_at_different_places(vocab, gap, trees):
    """Rows of a tree that start anywhere modulo 16 bytes: a warp's share of the tokens moves from row to row, the counts do not."""
    from xinfer_b200 import kernels as k
    rng = np.random.default_rng(vocab + gap)
    nodes, R = 60, 60 * trees
    few = np.concatenate([np.arange(126, 132), np.arange(254, 260)])
    near = edge_tokens(vocab)
    drafted, masks, paths = [], [], []
    for b in range(trees):
        _, _, on = tree(rng, nodes)
        toks = np.where(rng.random(nodes) < 0.6, rng.choice(few, nodes), rng.choice(near, nodes))
        drafted += toks.tolist()
        paths += [[int(toks[i]) for i in np.flatnonzero(on[r])] for r in range(nodes)]
        masks.append(words_of(on, 2))
    first, list_of_row = np.repeat(np.arange(trees) * nodes, nodes), np.repeat(np.arange(trees) // 2, nodes)
    lists = [rng.choice(near, 40).tolist() for _ in range((trees + 1) // 2)]
    logits, pen, prompt, ref, bound = case_of_rows(rng, R, vocab, lists, list_of_row.tolist(), paths)
    wide = torch.zeros(R, vocab + gap, device=DEV)
    wide[:, :vocab] = torch.tensor(logits, device=DEV)
    x, out = wide[:, :vocab], torch.full((R, vocab), 99.0, device=DEV)
    args = (torch.tensor(pen, device=DEV), i32(np.concatenate(lists)), i32(np.concatenate([[0], np.cumsum([len(t) for t in lists])])), i32(prompt))
    more = dict(list_of_row=i32(list_of_row), tree=(i32(drafted), torch.cat(masks).to(DEV), i32(first)))
    k.logit_rules(out, x, *args, **more)
    assert (np.abs(out.double().cpu().numpy() - ref) <= bound).all()
    again = torch.empty_like(out)
    for _ in range(50):
        k.logit_rules(again, x, *args, **more)
        assert torch.equal(again, out)
    k.logit_rules(x, x, *args, **more)                     # in place
    assert torch.equal(x, out) and bool((wide[:, vocab:] == 0.0).all())


@pytest.mark.parametrize("vocab", [3004, 50_000, 700_001])
@pytest.mark.parametrize("none", [-1, -2, -33, -1025])
def test_rows_whose_tree_begins_before_the_first_row(vocab, none):
    """Node i is row first_row + i where there is one, whatever first_row is; in every chunk of the vocabulary."""
    rng = np.random.default_rng(vocab - none)
    R = 9
    drafted = rng.choice(np.array([1, 5, 1030, 1031, 2050, 3003, vocab // 2, vocab - 1]) % vocab, R)
    first = np.array([none, none, none, 2, 2, none, none, 2 ** 31 - 1, none])
    on = rng.random((R, 64)) < 0.5
    paths = [[int(drafted[first[r] + i]) for i in range(64) if on[r, i] and 0 <= first[r] + i < R] for r in range(R)]
    lists = [rng.integers(0, vocab, 30).tolist()]
    logits, pen, prompt, ref, bound = case_of_rows(rng, R, vocab, lists, [0] * R, paths)
    got = call(logits, pen, lists, prompt, [0] * R, first, drafted, words_of(on, 2), None, None, None).double().cpu().numpy()
    assert (np.abs(got - ref) <= bound).all()
