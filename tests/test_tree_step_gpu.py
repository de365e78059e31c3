"""Acceptance of drafted tokens, slots from lengths on the device and the commit of accepted rows, against plain loops."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tree_cases import tree

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731


def walk(drafted, targets, parents, width):
    path, at, last = [], 0 if len(parents) else None, -1
    while at is not None and len(path) < width:
        path.append(at)
        last = targets[at]
        at = next((i for i in range(len(parents)) if parents[i] == at and drafted[i] == last), None)
    return path, last


@pytest.mark.parametrize("sizes,width", [([1], 1), ([16], 16), ([5, 0, 1, 64, 65, 33], 7), ([200, 1, 31, 32, 96], 40), ([64] * 100, 12), ([1000], 300), ([0, 0], 3)])
@pytest.mark.parametrize("kind", ["mixed", "chain", "star"])
def test_accept(sizes, width, kind):
    from xinfer_b200 import kernels as k
    rng = np.random.default_rng(sum(sizes) + width)
    start = [0] + list(np.cumsum(sizes))
    T = start[-1]
    parents = sum((tree(rng, n, kind)[0] for n in sizes if n), [])
    drafted, targets = rng.integers(0, 5, T), rng.integers(0, 5, T)
    for b, n in enumerate(sizes):
        for i in range(1, n):
            if rng.random() < 0.8:
                targets[start[b] + parents[start[b] + i]] = drafted[start[b] + i]
    B = len(sizes)
    acc, nxt, path = (torch.full(s, 55, dtype=torch.int32, device=DEV) for s in ((B,), (B,), (B, width)))
    k.tree_accept(acc, path, nxt, i32(drafted), i32(targets), i32(parents), i32(start))
    for b, n in enumerate(sizes):
        a = start[b]
        p, last = walk(drafted[a:a + n], targets[a:a + n], parents[a:a + n], width)
        assert acc[b].item() == len(p) and nxt[b].item() == last
        assert path[b].tolist() == [a + i for i in p] + [-1] * (width - len(p))


def test_accept_passes_over_parents_that_make_no_tree():
    from xinfer_b200 import kernels as k
    acc, nxt, path = i32([0]), i32([0]), i32([[0] * 4])
    k.tree_accept(acc, path, nxt, i32([1, 1, 1, 1]), i32([1, 1, 1, 1]), i32([2, 7, 0, 3]), i32([0, 4]))
    assert path.tolist() == [[0, 2, -1, -1]] and acc.tolist() == [2] and nxt.tolist() == [1]


class Cache:
    """The same bookkeeping in plain loops."""

    def __init__(self, rng, lengths, ps, spare, width, ring_more=0):
        self.ps, self.lengths = ps, list(lengths)
        held = [-(-n // ps) for n in lengths]
        total = sum(held) + spare
        ids = rng.permutation(total).tolist()
        self.rows = [[ids.pop() for _ in range(h)] for h in held]
        self.size, self.width = max(1, total + ring_more), width
        self.head = int(rng.integers(0, self.size))
        self.free = ids

    def device(self):
        table = np.full((len(self.lengths), self.width), -1)
        for b, row in enumerate(self.rows):
            table[b, :len(row)] = row
        ring = np.full(self.size, -1)
        for i, p in enumerate(self.free):
            ring[(self.head + i) % self.size] = p
        return i32(table), i32(ring), i32([self.head, len(self.free)])

    def step(self, new):
        """Slots, positions, requests, starts; the state afterwards is this object's."""
        slots, pos, req, start, bad = [], [], [], [0], False
        left, given, taken = len(self.free), [], 0
        asked = 0
        for b, add in enumerate(new):
            n, ps = self.lengths[b], self.ps
            if add < 0:
                given += self.rows[b]
                self.rows[b], self.lengths[b] = [], 0
                start.append(len(slots))
                continue
            fits = -(-(n + add) // ps) <= self.width
            need = -(-(n + add) // ps) - len(self.rows[b]) if fits else 0
            asked += need
            served = fits and (need == 0 or asked <= left)
            bad |= not served
            if served:
                self.rows[b] += self.free[asked - need:asked]
                taken = max(taken, asked) if need else taken
                self.lengths[b] = n + add
            for i in range(n, n + add):
                slots.append(self.rows[b][i // ps] * ps + i % ps if served else -1)
                pos.append(i)
                req.append(b)
            start.append(len(slots))
        self.head = (self.head + taken) % self.size
        self.free = self.free[taken:] + given
        return slots, pos, req, start, bad


def run_slots(c, new, capacity):
    from xinfer_b200 import kernels as k
    B = len(new)
    table, free, ring = c.device()
    lengths = i32(c.lengths)
    slots = torch.full((capacity,), 77, dtype=torch.int64, device=DEV)
    pos, req, start, out, ring_out = (torch.full((n,), 77, dtype=torch.int32, device=DEV) for n in (capacity, capacity, B + 1, B, 2))
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    for _ in range(2):          # a call may be made again
        k.cache_slots(slots, pos, req, start, out, ring_out, table, free, ring, lengths, i32(new), c.ps, err)
    return dict(slots=slots.tolist(), pos=pos.tolist(), req=req.tolist(), start=start.tolist(), lengths=out.tolist(), ring=ring_out.tolist(),
                table=table.tolist(), free=free.tolist(), err=int(err))


def check_slots(c, new, extra=5):
    from xinfer_b200 import kernels as k
    total = sum(max(0, x) for x in new)
    got = run_slots(c, new, total + extra)
    ended = [b for b, x in enumerate(new) if x < 0]
    slots, pos, req, start, bad = c.step(new)
    pad = [-1] * extra
    assert got["slots"] == slots + pad and got["req"] == req + pad and got["pos"][:total] == pos and got["start"] == start
    assert got["lengths"] == c.lengths and got["ring"] == [c.head, len(c.free)] and got["err"] == (k.ERR_NO_PAGE if bad else 0)
    for b, row in enumerate(c.rows):
        assert b in ended or got["table"][b][:len(row)] == row
    assert [got["free"][(c.head + i) % c.size] for i in range(len(c.free))] == c.free
    return got


@pytest.mark.parametrize("ps", [1, 8, 16, 48])
@pytest.mark.parametrize("lengths,new", [([0], [1]), ([0], [0]), ([16], [1]), ([15, 16, 17], [1, 1, 1]), ([0, 5, 40, 100], [300, 0, -1, 7]), ([7] * 40, [3, 0, 17, -1] * 10),
                                         ([33, 0, 1], [2500, 1, 1200]), (list(range(300)), [1, 2] * 150), ([10, 20], [-1, -1])])
def test_slots(lengths, new, ps):
    rng = np.random.default_rng(len(lengths))
    need = sum(-(-(n + max(a, 0)) // ps) - -(-n // ps) for n, a in zip(lengths, new))
    width = max(-(-(n + max(a, 0)) // ps) for n, a in zip(lengths, new)) + 1
    for spare in (need, need + 9):
        check_slots(Cache(rng, lengths, ps, spare, width), new)


def test_slots_of_several_steps_and_no_pages_left():
    rng = np.random.default_rng(5)
    c = Cache(rng, [0] * 12, 8, 60, 12, ring_more=3)
    refused = 0
    for _ in range(40):
        new = [int(x) for x in rng.choice([0, 1, 3, 30, -1, 95], 12, p=[0.2, 0.3, 0.2, 0.15, 0.1, 0.05])]
        refused += check_slots(c, new)["err"] != 0
    assert refused > 3


def test_slots_refuse_rows_that_are_too_short_and_tokens_that_are_too_many():
    from xinfer_b200 import kernels as k
    rng = np.random.default_rng(6)
    check_slots(Cache(rng, [10, 20, 5], 8, 50, 4), [30, 2, 27])      # 40, 22 and 32 tokens in rows of 32
    got = run_slots(Cache(rng, [3], 8, 50, 8), [20], 10)
    assert got["err"] == k.ERR_BAD_ROW and got["req"] == [0] * 10 and got["start"] == [0, 20]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers,nkv,d,ps,accepted", [(1, 1, 16, 16, [1]), (3, 2, 64, 8, [4, 0, 1, 6]), (2, 5, 48, 16, [2] * 30), (2, 3, 7, 16, [3, 5]), (36, 8, 128, 16, [5, 1])])
def test_commit(layers, nkv, d, ps, accepted, dtype):
    from xinfer_b200 import kernels as k
    rng = np.random.default_rng(layers + d)
    g = torch.Generator().manual_seed(layers)
    B, width, T = len(accepted), max(accepted) + 2, 8 * len(accepted)
    total = sum(accepted)
    pages = -(-total // ps) + 2
    kc, vc = ([torch.randn(pages, nkv, ps, d, generator=g).to(dtype) for _ in range(layers)] for _ in range(2))
    kn, vn = ([torch.randn(T, nkv, d, generator=g).to(dtype) for _ in range(layers)] for _ in range(2))
    path = np.full((B, width), -1)
    for b, a in enumerate(accepted):
        path[b, :a] = 8 * b + np.sort(rng.permutation(8)[:a])
    slots = np.concatenate([rng.permutation(pages * ps)[:total], [-1, -1, -1]])
    req = np.concatenate([np.repeat(np.arange(B), accepted), [-1, -1, 0]]).astype(np.int64)
    start = np.concatenate([[0], np.cumsum(accepted)])
    if total > 2:
        slots[2] = -1            # a token that found no page
    dev = lambda ts: [t.to(DEV) for t in ts]  # noqa: E731
    gkc, gvc, gkn, gvn = dev(kc), dev(vc), dev(kn), dev(vn)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    k.cache_commit(k.commit_table(gkc, gvc, gkn, gvn), torch.tensor(slots, device=DEV), i32(req), i32(start), i32(path), err)
    for i in range(total):
        if slots[i] < 0:
            continue
        row = path[req[i], i - start[req[i]]]
        for l in range(layers):
            kc[l][slots[i] // ps, :, slots[i] % ps], vc[l][slots[i] // ps, :, slots[i] % ps] = kn[l][row], vn[l][row]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(gkc + gvc, kc + vc)) and int(err) == 0


def test_commit_reports_what_lies_outside():
    from xinfer_b200 import kernels as k
    kc, vc = (torch.zeros(2, 1, 16, 16, device=DEV) for _ in range(2))
    kn, vn = (torch.ones(4, 1, 16, device=DEV) for _ in range(2))
    table = k.commit_table([kc], [vc], [kn], [vn])
    for slot, row, want in ((32, 0, k.ERR_BAD_PAGE), (0, 4, k.ERR_BAD_ROW), (2 ** 40, 1, k.ERR_BAD_PAGE)):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        k.cache_commit(table, torch.tensor([slot], device=DEV), i32([0]), i32([0, 1]), i32([[row]]), err)
        assert int(err) == want and torch.count_nonzero(kc) + torch.count_nonzero(vc) == 0


def test_refusals():
    from xinfer_b200 import kernels as k
    a = dict(accepted=i32([0]), path=i32([[0]]), next_tokens=i32([0]), drafted=i32([1]), targets=i32([1]), parents=i32([-1]), token_start=i32([0, 1]))
    k.tree_accept(**a)
    for change in (dict(path=i32([0])), dict(next_tokens=i32([0, 0])), dict(targets=i32([1, 1])), dict(parents=torch.tensor([-1], device=DEV)), dict(token_start=i32([0])),
                   dict(drafted=torch.tensor([1], dtype=torch.int32)), dict(path=torch.zeros(1, 0, dtype=torch.int32, device=DEV))):
        with pytest.raises(k.KernelError):
            k.tree_accept(**{**a, **change})
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    s = dict(slots=torch.zeros(2, dtype=torch.int64, device=DEV), positions=i32([0, 0]), request_of=i32([0, 0]), token_start=i32([0, 0]), lengths_out=i32([0]), ring_out=i32([0, 0]),
             block_table=i32([[0, 0]]), free_ring=i32([0, 1]), ring=i32([0, 2]), lengths=i32([0]), new_tokens=i32([1]), page_size=16, err=err)
    k.cache_slots(**s)
    for change in (dict(slots=i32([0, 0])), dict(positions=i32([0])), dict(lengths_out=s["lengths"]), dict(ring_out=s["ring"]), dict(page_size=0), dict(block_table=i32([0])),
                   dict(ring=i32([0])), dict(new_tokens=i32([1, 1])), dict(free_ring=torch.zeros(0, dtype=torch.int32, device=DEV)), dict(err=None)):
        with pytest.raises(k.KernelError):
            k.cache_slots(**{**s, **change})
    big = torch.zeros(k.SLOT_REQUESTS_MAX + 1, dtype=torch.int32, device=DEV)
    with pytest.raises(k.KernelError):
        k.cache_slots(**{**s, "lengths": big})
    c, n = torch.zeros(2, 1, 16, 16, device=DEV), torch.zeros(4, 1, 16, device=DEV)
    for bad in (([], [], [], []), ([c], [c], [n], []), ([c], [c.bfloat16()], [n], [n]), ([c], [c], [n], [n[:2]]), ([c.cpu()], [c], [n], [n]), ([c.half()], [c.half()], [n.half()], [n.half()])):
        with pytest.raises(k.KernelError):
            k.commit_table(*bad)
    with pytest.raises(k.KernelError):
        k.cache_commit(None, s["slots"], s["request_of"], s["token_start"], i32([[0]]), err)


@pytest.mark.parametrize("most", [2 ** 31 - 1, 2 ** 30, 10 ** 6])
def test_slots_for_numbers_of_tokens_that_nobody_has(most):
    """Requests that ask for more than their rows hold get nothing, however much it is together; the one beside them gets its slots
    where the tokens before it leave room."""
    from xinfer_b200 import kernels as k
    rng = np.random.default_rng(9)
    c = Cache(rng, [3, 5, 9, 2], 8, 20, 4)
    pages = [list(row) for row in c.rows]
    got = run_slots(c, [4, most, most, 3], 12)
    assert got["err"] == k.ERR_NO_PAGE | k.ERR_BAD_ROW
    assert got["lengths"] == [7, 5, 9, 5] and got["slots"] == [pages[0][0] * 8 + i for i in range(3, 7)] + [-1] * 8
    assert got["start"] == [0, 4, min(4 + most, 2 ** 31 - 1), min(4 + 2 * most, 2 ** 31 - 1), min(7 + 2 * most, 2 ** 31 - 1)]
    assert got["req"] == [0] * 4 + [1] * 8 and got["ring"][1] == 20


def test_slots_of_the_most_requests():
    rng = np.random.default_rng(10)
    from xinfer_b200 import kernels as k
    B = k.SLOT_REQUESTS_MAX
    new = rng.choice([0, 1, 2, 9, -1], B).tolist()
    lengths = rng.integers(0, 40, B).tolist()
    check_slots(Cache(rng, lengths, 16, 3000, 5), new)


@pytest.mark.parametrize("requests", [4083, 4084, 4095, 4096])
def test_slots_of_as_many_requests_as_fill_the_memory_that_needs_no_asking(requests):
    """In a process of its own: a larger call before it has asked for more shared memory, for all calls after it."""
    code = ("import sys; sys.path[:0] = sys.argv[1:3]\n"
            "import numpy as np, test_tree_step_gpu as t\n"
            f"rng = np.random.default_rng({requests})\n"
            f"lengths, new = rng.integers(0, 40, {requests}).tolist(), rng.choice([0, 1, 2, 9, -1], {requests}).tolist()\n"
            "t.check_slots(t.Cache(rng, lengths, 16, 3000, 5), new)\n")
    here = os.path.dirname(os.path.abspath(__file__))
    done = subprocess.run([sys.executable, "-c", code, here, os.path.dirname(here)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("new", [9, 10, 20, 2 ** 31 - 1])
def test_slots_of_lengths_at_the_end_of_32_bits(new):
    """A length that 32 bits do not hold is refused like one that its row of the table does not hold; the largest one is served."""
    from xinfer_b200 import kernels as k
    rng = np.random.default_rng(11)
    n, ps = 2 ** 31 - 10, 2 ** 30
    c = Cache(rng, [n, 7], ps, 4, 5)
    rows = [list(r) for r in c.rows]
    got = run_slots(c, [new, 2], 24)
    at = [rows[0][1] * ps + i - ps for i in range(n, n + 9)]
    beside = [rows[1][0] * ps + 7, rows[1][0] * ps + 8]
    if new == 9:
        assert got["err"] == 0 and got["lengths"] == [2 ** 31 - 1, 9] and got["slots"] == at + beside + [-1] * 13 and got["pos"][:11] == list(range(n, n + 9)) + [7, 8]
    else:
        mine = min(new, 24)
        assert got["err"] == k.ERR_NO_PAGE | (k.ERR_BAD_ROW if new > 24 else 0) and got["lengths"] == [n, 9]
        assert got["slots"] == ([-1] * mine + beside + [-1] * 24)[:24] and got["pos"][:mine] == [min(i, 2 ** 31 - 1) for i in range(n, n + mine)]
    assert got["ring"][1] == 4 and got["start"] == [0, new, min(new + 2, 2 ** 31 - 1)]
