"""The operators of a decoding step that verifies a tree of drafted tokens, as cases that can be timed and checked.

A case is a dict of plain values; ``kind`` names its operator:

* ``attend``: attention of the drafted tokens over the paged cache and their own ancestors (``kernels.tree_attention``);
* ``rules``: penalties, biases and grammar masks on the logits of every drafted token (``kernels.logit_rules``);
* ``accept``: which drafted tokens the model's own choices confirm (``kernels.tree_accept``);
* ``slots``: block tables and slot maps for tokens whose number is known on the device alone (``kernels.cache_slots``);
* ``commit``: the accepted tokens' keys and values of every layer go to their pages (``kernels.cache_commit``).

How long each request is and how many tokens it brings follow from the case; the values follow from the seed.
"""
import math

import numpy as np
import torch

own = False
DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def listed():
    return [
        # one user of a small model, a narrow tree: launches and latency
        dict(name="attend-1x16", kind="attend", requests=1, nodes=16, context=1024, heads=16, kv_heads=8, dim=128, dtype="bf16", page=16, window=0),
        # eight users at context 4,096 with wide trees: memory and tensor cores both near their limits
        dict(name="attend-8x64", kind="attend", requests=8, nodes=64, context=4096, heads=32, kv_heads=8, dim=128, dtype="bf16", page=16, window=0),
        # many users with long contexts of uneven length: the cache's bytes
        dict(name="attend-48x24-long", kind="attend", requests=48, nodes=24, context=32768, heads=32, kv_heads=8, dim=128, dtype="bf16", page=16, window=0),
        # the float32 engine, as one runs it to check a model: a group of two heads of 48 channels, a window
        dict(name="attend-3x13-f32", kind="attend", requests=3, nodes=13, context=777, heads=10, kv_heads=5, dim=48, dtype="f32", page=16, window=256),
        # one user without a tree whose answer follows a grammar
        dict(name="rules-1x1", kind="rules", requests=1, nodes=1, vocab=151936, history=500, biases=8, masked=True),
        # eight users with wide trees, a mask per drafted token and long histories
        dict(name="rules-8x64", kind="rules", requests=8, nodes=64, vocab=151936, history=4096, biases=16, masked=True),
        # one user
        dict(name="accept-1x16", kind="accept", requests=1, nodes=16, width=16),
        # a full batch of wide trees
        dict(name="accept-256x64", kind="accept", requests=256, nodes=64, width=12),
        # a full batch that took a few tokens each
        dict(name="slots-64x6", kind="slots", requests=64, new=6, length=4096, page=16),
        # prompts that arrive together
        dict(name="slots-32x2048", kind="slots", requests=32, new=2048, length=600, page=16),
        # one user of a small model
        dict(name="commit-1x4", kind="commit", requests=1, accepted=4, layers=28, kv_heads=8, dim=128, dtype="bf16", page=16),
        # a full batch of a large model
        dict(name="commit-128x6", kind="commit", requests=128, accepted=6, layers=36, kv_heads=8, dim=128, dtype="bf16", page=16),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    kind = rng.choices(["attend", "rules", "accept", "slots", "commit"], [50, 20, 8, 10, 12])[0]
    if kind == "attend":
        dtype = rng.choices(["bf16", "f32"], [4, 1])[0]
        kv_heads, group, dim = rng.choice([1, 2, 3, 5, 8]), rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([64, 128, 128, 128, 48, 80, 96] if dtype == "bf16" else [32, 48, 64, 128])
        nodes = _spread(rng, 1, 96)
        context = _spread(rng, 16, 32768 if dtype == "bf16" else 4096)
        most = (1 << 20) if dtype == "bf16" else (1 << 13)      # tokens in the cache
        requests = max(1, min(_spread(rng, 1, 48), most // context))
        page = rng.choice([8, 16, 16, 32, 64])
        case = dict(kind=kind, requests=requests, nodes=nodes, context=context, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    dtype=dtype, page=page, window=rng.choice([0, 0, 0, _spread(rng, 16, 4096)]))
        while case["requests"] > 1 and _cost(case) > 0.9 * max(_cost(c) for c in listed()):
            case["requests"] //= 2
        return case
    if kind == "rules":
        requests, nodes, vocab = _spread(rng, 1, 16), _spread(rng, 1, 64), rng.choice([151936, 32000, _spread(rng, 331, 151936)])
        requests = max(1, min(requests, 512 // nodes))
        return dict(kind=kind, requests=requests, nodes=nodes, vocab=vocab, history=_spread(rng, 1, 8192), biases=rng.choice([0, _spread(rng, 1, 300)]),
                    masked=rng.random() < 0.6)
    if kind == "accept":
        return dict(kind=kind, requests=_spread(rng, 1, 256), nodes=_spread(rng, 2, 128), width=_spread(rng, 3, 24))
    if kind == "slots":
        requests = _spread(rng, 1, 512)
        return dict(kind=kind, requests=requests, new=max(1, min(_spread(rng, 1, 4096), 65536 // requests)), length=_spread(rng, 1, 8192), page=rng.choice([8, 16, 32, 64]))
    requests, accepted = _spread(rng, 1, 128), rng.randint(1, 6)
    return dict(kind=kind, requests=requests, accepted=accepted, layers=rng.choice([2, 12, 28, 36]), kv_heads=rng.choice([1, 4, 5, 8]),
                dim=rng.choice([48, 64, 80, 128]), dtype=rng.choice(["bf16", "bf16", "f32"]), page=rng.choice([8, 16, 64]))


# ---- what follows from the case alone ----------------------------------------------------------------------------------

def _sizes(case):
    """Ragged sizes: the first request has what the case says; of four and more, one has a single token and one has none."""
    rng, n = np.random.default_rng(7), case["requests"]
    nodes = rng.integers(max(1, case["nodes"] // 2), case["nodes"] + 1, n)
    context = np.round(case["context"] * np.exp(rng.uniform(-2.5, 0.0, n))).astype(np.int64)
    nodes[0], context[0] = case["nodes"], case["context"]
    if n >= 4:
        nodes[1], context[2], nodes[n - 1] = 1, 0, 0
    return nodes, context


def _news(case):
    """Tokens that each request brings: of four and more requests one brings none and one ends (-1)."""
    rng, n = np.random.default_rng(8), case["requests"]
    new = rng.integers(max(1, case["new"] // 2), case["new"] + 1, n)
    length = rng.integers(case["length"] // 2, case["length"] + 1, n)
    new[0] = case["new"]
    if n >= 4:
        new[1], new[2], length[3] = 0, -1, 0
    return new, length


def work(case):
    kind = case["kind"]
    if kind == "attend":
        nodes, context = _sizes(case)
        w = case["window"]
        seen = np.minimum(context, w) if w else context             # (no node sees more cached keys than its window)
        t, es = int(nodes.sum()), BYTES[case["dtype"]]
        read = int(seen[nodes > 0].sum()) * case["kv_heads"] * case["dim"] * 2 * es
        rows = t * (2 * case["heads"] + 2 * case["kv_heads"]) * case["dim"] * es
        least = np.minimum(context, np.maximum(0, w - case["nodes"])) if w else context
        return dict(bytes=read + rows + int(-(-seen // case["page"]).sum()) * 4, flops=4 * case["heads"] * case["dim"] * int((nodes * (least + 1)).sum()))
    if kind == "rules":
        rows = case["requests"] * case["nodes"]
        masks = rows * 4 * -(-case["vocab"] // 32) if case["masked"] else 0
        return dict(bytes=rows * case["vocab"] * 8 + masks + case["requests"] * case["history"] * 4 + rows * case["biases"] * 8, flops=rows * case["vocab"])
    if kind == "accept":
        t = case["requests"] * case["nodes"]
        return dict(bytes=12 * t + case["requests"] * (case["width"] + 3) * 4, flops=t)
    if kind == "slots":
        new, _ = _news(case)
        t = int(np.maximum(new, 0).sum())
        return dict(bytes=16 * t + 20 * case["requests"] + 8 * (t // case["page"]), flops=t)
    moved = case["requests"] * case["accepted"] * case["layers"] * case["kv_heads"] * case["dim"] * 2
    return dict(bytes=2 * moved * BYTES[case["dtype"]], flops=moved)


# ---- inputs -----------------------------------------------------------------------------------------------------------------

def _trees(rng, nodes, spine=0.5):
    """Parents (place in the own tree, -1 for the root), depths and which nodes lie on whose path, of trees of so many nodes:
    a node follows the one before it or any earlier one."""
    most = max(1, int(nodes.max()))
    n = len(nodes)
    parents = np.full((n, most), -1, np.int64)
    depth = np.zeros((n, most), np.int64)
    on = np.zeros((n, most, most), bool)
    on[:, 0, 0] = True
    for i in range(1, most):
        p = np.where(rng.random(n) < spine, i - 1, (rng.random(n) * i).astype(np.int64))
        parents[:, i], depth[:, i] = p, depth[np.arange(n), p] + 1
        on[:, i] = on[np.arange(n), p]
        on[:, i, i] = True
    live = np.arange(most)[None] < nodes[:, None]
    words = -(-most // 32)
    bits = np.zeros((n, most, words * 32), np.uint64)
    bits[:, :, :most] = on
    packed = (bits.reshape(n, most, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)
    return parents[live].astype(np.int32), depth[live].astype(np.int32), packed[live]


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    kind = case["kind"]

    def normal(shape, dtype, scale=1.0):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype).mul_(scale)

    s = dict(case=case)
    if kind == "attend":
        nodes, context = _sizes(case)
        t, dt, nkv, d, ps = int(nodes.sum()), TYPES[case["dtype"]], case["kv_heads"], case["dim"], case["page"]
        pages = -(-context // ps)
        total = int(pages.sum()) + 1
        table = np.full((case["requests"], max(1, int(pages.max()))), -1, np.int32)
        ids, at = rng.permutation(total), 0
        for b, m in enumerate(pages):
            table[b, :m] = ids[at:at + m]
            at += m
        _, depth, ancestors = _trees(rng, nodes)
        # queries and keys behind a norm: scores of a few units
        s.update(q=normal((t, case["heads"], d), dt, 1.5), k_new=normal((t, nkv, d), dt), v_new=normal((t, nkv, d), dt),
                 k_cache=normal((total, nkv, ps, d), dt), v_cache=normal((total, nkv, ps, d), dt), context=_dev(context.astype(np.int32)),
                 token_start=_dev(_starts(nodes)), ancestors=_dev(ancestors), depth=_dev(depth), table=_dev(table),
                 out=torch.empty((t, case["heads"], d), device=DEVICE, dtype=dt), scale=1.0 / math.sqrt(d), most=int(nodes.max()))
    elif kind == "rules":
        n, m, v = case["requests"], case["nodes"], case["vocab"]
        rows = n * m
        lists = rng.integers(max(1, case["history"] // 2), case["history"] + 1, n)
        lists[0] = case["history"]
        # token ids as text has them: few of them often
        tokens = np.minimum((v ** rng.random(int(lists.sum()))).astype(np.int64), v - 1)
        _, _, ancestors = _trees(rng, np.full(n, m))
        drafted = np.minimum((v ** rng.random(rows)).astype(np.int64), v - 1)
        penalties = np.stack([rng.choice([1.0, 1.05, 1.2], rows), rng.choice([0.0, 0.4], rows), rng.choice([0.0, 0.6], rows)], 1)
        s.update(logits=normal((rows, v), torch.float32, 3.0), out=torch.empty((rows, v), device=DEVICE), penalties=_dev(penalties.astype(np.float32)),
                 history=_dev(tokens.astype(np.int32)), history_start=_dev(_starts(lists)), prompt_len=_dev((lists // 2).astype(np.int32)),
                 list_of_row=_dev(np.repeat(np.arange(n), m).astype(np.int32)), drafted=_dev(drafted.astype(np.int32)), ancestors=_dev(ancestors),
                 first_row=_dev(np.repeat(np.arange(n) * m, m).astype(np.int32)))
        if case["biases"]:
            per = np.stack([rng.choice(v, min(v, case["biases"]), replace=False) for _ in range(min(rows, 16))])
            per = per[np.arange(rows) % len(per)]
            s.update(bias_start=_dev(np.arange(rows + 1, dtype=np.int32) * per.shape[1]), bias_tokens=_dev(per.reshape(-1).astype(np.int32)),
                     bias_values=_dev(rng.normal(size=per.size).astype(np.float32) * 4))
        if case["masked"]:
            # every third row may say nearly anything, the others a few words of thirty-two
            words = -(-v // 32)
            raw = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=gen, device=DEVICE, dtype=torch.int64)
            thin = raw & torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=gen, device=DEVICE, dtype=torch.int64) & (raw >> 3)
            wide = (torch.arange(rows, device=DEVICE) % 3 == 0)[:, None]
            s.update(mask=torch.where(wide, raw | (raw >> 5), thin).to(torch.int32), mask_of_row=_dev(rng.permutation(rows).astype(np.int32)))
            if rows >= 4:
                s["mask_of_row"][1] = -1           # a row that no grammar binds
    elif kind == "accept":
        n, m = case["requests"], case["nodes"]
        nodes = np.random.default_rng(9).integers(max(1, m // 2), m + 1, n)
        nodes[0] = m
        if n >= 4:
            nodes[2] = 0
        parents, _, ancestors = _trees(rng, nodes, 0.3)
        start = _starts(nodes)
        t = int(nodes.sum())
        base = np.repeat(start[:-1], nodes)
        drafted = rng.integers(0, 24, t)           # few different tokens: siblings that say the same happen
        targets = rng.integers(0, 24, t)
        hit = (parents >= 0) & (rng.random(t) < 0.75)
        targets[(base + parents)[hit]] = drafted[hit]
        s.update(drafted=_dev(drafted.astype(np.int32)), targets=_dev(targets.astype(np.int32)), parents=_dev(parents), ancestors=_dev(ancestors), token_start=_dev(start),
                 accepted=torch.empty(n, dtype=torch.int32, device=DEVICE), next_tokens=torch.empty(n, dtype=torch.int32, device=DEVICE),
                 path=torch.empty((n, case["width"]), dtype=torch.int32, device=DEVICE), most=m)
    elif kind == "slots":
        new, length = _news(case)
        n, ps, t = len(new), case["page"], int(np.maximum(new, 0).sum())
        held = -(-length // ps)
        need = np.where(new < 0, 0, -(-(length + np.maximum(new, 0)) // ps) - held)
        total = int(held.sum() + need.sum()) + 5
        ids = rng.permutation(total).astype(np.int32)
        table, at = np.full((n, int((held + need).max()) + 2), -1, np.int32), 0
        for b, m in enumerate(held):
            table[b, :m] = ids[at:at + m]
            at += m
        ring, head, count = np.full(total, -1, np.int32), int(rng.integers(0, total)), total - at
        ring[(head + np.arange(count)) % total] = ids[at:]
        i32 = lambda *shape: torch.empty(shape, dtype=torch.int32, device=DEVICE)  # noqa: E731
        s.update(new=_dev(new.astype(np.int32)), lengths=_dev(length.astype(np.int32)), table=_dev(table), free_ring=_dev(ring), ring=_dev(np.array([head, count], np.int32)),
                 slots=torch.empty(t + 3, dtype=torch.int64, device=DEVICE), positions=i32(t + 3), request_of=i32(t + 3), token_start=i32(n + 1), lengths_out=i32(n), ring_out=i32(2))
    else:
        n, ps, dt = case["requests"], case["page"], TYPES[case["dtype"]]
        accepted = np.random.default_rng(10).integers(1, case["accepted"] + 1, n)
        accepted[0] = case["accepted"]
        most, t = 2 * case["accepted"], 2 * case["accepted"] * n
        path = np.full((n, case["accepted"] + 1), -1, np.int32)
        for b, a in enumerate(accepted):
            path[b, :a] = b * most + np.concatenate([[0], np.sort(rng.permutation(most - 1)[:a - 1]) + 1])
        start, total = _starts(accepted), int(accepted.sum())
        pages = -(-total // ps) + n
        slots = np.full(total + 2, -1, np.int64)
        slots[:total] = rng.permutation(pages * ps)[:total]
        request_of = np.full(total + 2, -1, np.int32)
        request_of[:total] = np.repeat(np.arange(n), accepted)
        shape, rows = (case["layers"], pages, case["kv_heads"], ps, case["dim"]), (case["layers"], t, case["kv_heads"], case["dim"])
        s.update(k_cache=normal(shape, dt), v_cache=normal(shape, dt), k_new=normal(rows, dt), v_new=normal(rows, dt), path=_dev(path), slots=_dev(slots),
                 request_of=_dev(request_of), token_start=_dev(start))
    if kind in ("attend", "slots", "commit"):
        s["err"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------

def _unpack(words, n):
    """Bits of 32-bit words, lowest first: [..., words] -> [..., n] truth values."""
    bits = (words.unsqueeze(-1) >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return bits.flatten(-2)[..., :n].bool()


def _plain_attend(s):
    c = s["case"]
    nkv, d, most, w = c["kv_heads"], c["dim"], s["most"], c["window"]
    start, context = s["token_start"].long(), s["context"].long()
    t, n = s["q"].shape[0], context.shape[0]
    place = torch.arange(most, device=start.device)
    live = place < (start[1:] - start[:-1])[:, None]
    rows = torch.where(live, start[:-1, None] + place, 0)                                   # [requests, nodes]
    table = s["table"].long().clamp(min=0)
    old = torch.arange(table.shape[1] * c["page"], device=start.device)

    def keys(cache, fresh):
        cached = cache[table].transpose(2, 3).flatten(1, 2)                                 # [requests, cached, kv heads, d]
        return torch.cat([cached, fresh[rows]], 1).permute(0, 2, 1, 3).float()

    depth = s["depth"].long()[rows]
    seen_old = (old < context[:, None])[:, None].expand(n, most, old.shape[0])
    seen_new = _unpack(s["ancestors"][rows], most) & live[:, None]
    if w:
        seen_old = seen_old & (old > (context[:, None] + depth - w)[..., None])
        seen_new = seen_new & (depth[:, :, None] - depth[:, None] < w)
    seen = torch.cat([seen_old, seen_new], 2)[:, None, :, None]                              # [requests, 1, nodes, 1, keys]
    q = s["q"][rows].unflatten(2, (nkv, -1)).permute(0, 2, 1, 3, 4).float()                  # [requests, kv heads, nodes, group, d]
    scores = (q.flatten(2, 3) @ keys(s["k_cache"], s["k_new"]).transpose(2, 3)).mul_(s["scale"]).unflatten(2, (most, -1))
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.flatten(2, 3) @ keys(s["v_cache"], s["v_new"])).unflatten(2, (most, -1)) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 2, 1, 3, 4).flatten(2, 3)[live].reshape(t, c["heads"], d).to(s["q"].dtype)


def _plain_rules(s):
    logits, start, rows_of = s["logits"], s["history_start"].long(), s["list_of_row"].long()
    rows, v = logits.shape
    n = s["prompt_len"].shape[0]
    at = torch.arange(s["history"].shape[0], device=logits.device)
    which = torch.searchsorted(start, at, right=True) - 1
    flat = which * v + s["history"].long()
    prompt = at - start[which] < s["prompt_len"].long()[which]
    made = torch.zeros(n * v, device=logits.device).index_add_(0, flat, (~prompt).float()).view(n, v)
    said = torch.zeros(n * v, device=logits.device).index_add_(0, flat, prompt.float()).view(n, v) > 0
    count = made[rows_of]
    path = _unpack(s["ancestors"], s["ancestors"].shape[1] * 32)
    node = (s["first_row"].long()[:, None] + torch.arange(path.shape[1], device=logits.device)).clamp(max=rows - 1)
    count.view(-1).index_add_(0, (torch.arange(rows, device=logits.device)[:, None] * v + s["drafted"].long()[node]).flatten(), path.float().flatten())
    rep, freq, pres = s["penalties"].unsqueeze(2).unbind(1)
    x = torch.where((count > 0) | said[rows_of], torch.where(logits > 0, logits / rep, logits * rep), logits)
    x = x - freq * count - pres * (count > 0).float()
    if "bias_start" in s:
        bs = s["bias_start"].long()
        which = torch.searchsorted(bs, torch.arange(s["bias_tokens"].shape[0], device=logits.device), right=True) - 1
        x.view(-1).index_add_(0, which * v + s["bias_tokens"].long(), s["bias_values"])
    if "mask" in s:
        m = s["mask_of_row"].long()
        x = torch.where(_unpack(s["mask"][m.clamp(min=0)], v) | (m < 0)[:, None], x, -math.inf)
    return x


def _plain_accept(s):
    start, width = s["token_start"].long(), s["case"]["width"]
    n, most, dev = start.shape[0] - 1, s["most"], start.device
    place = torch.arange(most, device=dev)
    live = place < (start[1:] - start[:-1])[:, None]
    rows = torch.where(live, start[:-1, None] + place, 0)
    tokens, parents = s["drafted"][rows], torch.where(live, s["parents"][rows].long(), -1)
    agrees = (tokens == torch.gather(s["targets"][rows], 1, parents.clamp(min=0))) & (parents >= 0) & live
    twin = (parents[:, :, None] == parents[:, None]) & agrees[:, :, None] & agrees[:, None] & (place[None, None, :] < place[None, :, None])
    good = (agrees & ~twin.any(2)) | ((place == 0) & live)                                   # the first that agrees among its siblings
    on = _unpack(s["ancestors"][rows], most)
    taken = ~(on & ~good[:, None]).any(2) & live
    found = torch.where(taken, place, most).sort(1).values
    found = torch.cat([found, found.new_full((n, max(0, width - most)), most)], 1)[:, :width]
    kept = found < most
    accepted = kept.sum(1)
    path = torch.where(kept, start[:-1, None] + found, -1)
    last = torch.gather(path, 1, (accepted - 1).clamp(min=0)[:, None])[:, 0]
    following = torch.where(accepted > 0, s["targets"][last.clamp(min=0)].long(), -1)
    return dict(accepted=accepted.int(), path=path.int(), next_tokens=following.int())


def _plain_slots(s):
    new, length, ps, size = s["new"].long(), s["lengths"].long(), s["case"]["page"], s["free_ring"].shape[0]
    ended, dev = new < 0, new.device
    new = new.clamp(min=0)
    head, count = s["ring"].long().unbind(0)
    held = (length + ps - 1) // ps
    need = torch.where(ended, 0, (length + new + ps - 1) // ps - held)
    taken = need.cumsum(0)
    column = torch.arange(s["table"].shape[1], device=dev)
    mine = (column >= held[:, None]) & (column < (held + need)[:, None])
    page = s["free_ring"][(head + (taken - need)[:, None] + column - held[:, None]) % size]
    back = torch.where(ended, held, 0)
    give = ended[:, None] & (column < held[:, None])
    to = torch.where(give, (head + count + (back.cumsum(0) - back)[:, None] + column) % size, size)
    s["free_ring"].copy_(torch.cat([s["free_ring"], s["free_ring"][:1]]).scatter_(0, to.flatten(), s["table"].flatten())[:size])
    s["table"].copy_(torch.where(mine, page, s["table"]))
    start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    at = torch.arange(s["slots"].shape[0], device=dev)
    real = at < start[-1]
    which = torch.where(real, torch.searchsorted(start, at, right=True) - 1, 0)
    pos = torch.where(real, length[which] + at - start[which], 0)
    slots = torch.where(real, s["table"][which, pos // ps].long() * ps + pos % ps, -1)
    state = torch.stack([(head + taken[-1]) % size, count - taken[-1] + back.sum()])
    return dict(slots=slots, positions=pos.int(), request_of=torch.where(real, which, -1).int(), token_start=start.int(),
                lengths=torch.where(ended, 0, length + new).int(), ring=state.int(), table=s["table"], free_ring=s["free_ring"])


def _plain_commit(s):
    ps, which = s["case"]["page"], s["request_of"].long()
    at = torch.where(which >= 0, torch.arange(which.shape[0], device=which.device), 0)       # padding does the first token again
    which, slots = which[at], s["slots"][at]
    rows = s["path"].long()[which, at - s["token_start"].long()[which]]
    for cache, fresh in ((s["k_cache"], s["k_new"]), (s["v_cache"], s["v_new"])):
        cache[:, slots // ps, :, slots % ps] = fresh[:, rows].transpose(0, 1)
    return s["k_cache"], s["v_cache"]


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if not own:
        return dict(attend=_plain_attend, rules=_plain_rules, accept=_plain_accept, slots=_plain_slots, commit=_plain_commit)[kind](s)
    from xinfer_b200 import kernels
    if kind == "attend":
        c = s["case"]
        if "scratch" not in s:      # the workspace that a program keeps for its steps
            s["scratch"] = torch.empty(kernels.tree_attention_scratch(s["q"].shape[0], c["heads"], c["kv_heads"], c["dim"], s["q"].dtype), device=DEVICE)
        kernels.tree_attention(s["out"], s["q"], s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], s["context"], s["token_start"], s["ancestors"], s["table"],
                               s["scale"], s["err"], scratch=s["scratch"], depth=s["depth"], window=c["window"] or None)
        return s["out"]
    if kind == "rules":
        bias = (s["bias_start"], s["bias_tokens"], s["bias_values"]) if "bias_start" in s else None
        kernels.logit_rules(s["out"], s["logits"], s["penalties"], s["history"], s["history_start"], s["prompt_len"], list_of_row=s["list_of_row"],
                            tree=(s["drafted"], s["ancestors"], s["first_row"]), bias=bias, mask=s.get("mask"), mask_of_row=s.get("mask_of_row"))
        return s["out"]
    if kind == "accept":
        kernels.tree_accept(s["accepted"], s["path"], s["next_tokens"], s["drafted"], s["targets"], s["parents"], s["token_start"])
        return dict(accepted=s["accepted"], path=s["path"], next_tokens=s["next_tokens"])
    if kind == "slots":
        kernels.cache_slots(s["slots"], s["positions"], s["request_of"], s["token_start"], s["lengths_out"], s["ring_out"], s["table"], s["free_ring"],
                            s["ring"], s["lengths"], s["new"], s["case"]["page"], s["err"])
        return dict(slots=s["slots"], positions=s["positions"], request_of=s["request_of"], token_start=s["token_start"], lengths=s["lengths_out"],
                    ring=s["ring_out"], table=s["table"], free_ring=s["free_ring"])
    if "layers" not in s:           # the addresses of the layers' caches, which a program lays out once
        s["layers"] = kernels.commit_table(list(s["k_cache"]), list(s["v_cache"]), list(s["k_new"]), list(s["v_new"]))
    kernels.cache_commit(s["layers"], s["slots"], s["request_of"], s["token_start"], s["path"], s["err"])
    return s["k_cache"], s["v_cache"]


# ---- the same in 64 bits, request by request ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        nkv, group, w = case["kv_heads"], case["heads"] // case["kv_heads"], case["window"]
        start, context = s["token_start"].tolist(), s["context"].tolist()
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        for b in range(case["requests"]):
            a, z, have = start[b], start[b + 1], context[b]
            if a == z:
                continue
            j = torch.arange(have, device=DEVICE)
            page = s["table"][b].long()[j // case["page"]]
            depth = s["depth"][a:z].long()
            at = torch.cat([j, have + depth])                                        # every key's place in its sequence
            i = torch.arange(z - a, device=DEVICE)
            seen = torch.ones((z - a, have + z - a), dtype=torch.bool, device=DEVICE)
            seen[:, have:] = (s["ancestors"][a:z].long()[:, i // 32] >> (i % 32)) & 1 != 0
            if w:
                seen &= have + depth[:, None] - at < w
            for g in range(nkv):
                k = torch.cat([s["k_cache"][page, g, j % case["page"]], s["k_new"][a:z, g]]).double()
                v = torch.cat([s["v_cache"][page, g, j % case["page"]], s["v_new"][a:z, g]]).double()
                for h in range(g * group, (g + 1) * group):
                    x = (s["q"][a:z, h].double() @ k.T * s["scale"]).masked_fill(~seen, -math.inf)
                    out[a:z, h] = torch.softmax(x, 1).nan_to_num(0.0) @ v
        return out
    if case["kind"] == "rules":
        v, m = case["vocab"], case["nodes"]
        history, start, prompt = s["history"].cpu().numpy(), s["history_start"].tolist(), s["prompt_len"].tolist()
        drafted, words, pen = s["drafted"].cpu().numpy(), s["ancestors"].cpu().numpy().view(np.uint32), s["penalties"].double().cpu().numpy()
        out = s["logits"].double()
        for b in range(case["requests"]):
            own_list = history[start[b]:start[b + 1]]
            base = np.bincount(own_list[prompt[b]:], minlength=v)
            asked = np.bincount(own_list[:prompt[b]], minlength=v) > 0
            for r in range(b * m, (b + 1) * m):
                count = base.copy()
                for i in range(m):
                    if words[r, i // 32] >> (i % 32) & 1:
                        count[drafted[b * m + i]] += 1
                tok = np.nonzero((count > 0) | asked)[0]
                at, many = _dev(tok), _dev(count[tok].astype(np.float64))
                x = out[r, at]
                out[r, at] = torch.where(x > 0, x / pen[r, 0], x * pen[r, 0]) - pen[r, 1] * many - pen[r, 2] * (many > 0)
                if case["biases"]:
                    lo, hi = s["bias_start"][r:r + 2].tolist()
                    out[r, s["bias_tokens"][lo:hi].long()] += s["bias_values"][lo:hi].double()
                if case["masked"] and int(s["mask_of_row"][r]) >= 0:
                    word = s["mask"][int(s["mask_of_row"][r])].long()
                    i = torch.arange(v, device=DEVICE)
                    out[r, (word[i // 32] >> (i % 32)) & 1 == 0] = -math.inf
        return out
    if case["kind"] == "commit":
        ps, k, v = case["page"], s["k_cache"].double(), s["v_cache"].double()
        slots, start, path = s["slots"].tolist(), s["token_start"].tolist(), s["path"].tolist()
        for b in range(case["requests"]):
            for i in range(start[b], start[b + 1]):
                row = path[b][i - start[b]]
                k[:, slots[i] // ps, :, slots[i] % ps] = s["k_new"][:, row].double()
                v[:, slots[i] // ps, :, slots[i] % ps] = s["v_new"][:, row].double()
        return k, v
    return None
