"""The operators of a decoding step whose cache and weights are held in 4 bits, as cases that can be timed and checked.

A case is a dict of plain values; ``kind`` names its operator:

* ``write``: norms and rotation of a step's queries and keys, its keys and values into 4-bit pages (``kernels.cache4_write``);
* ``attend``: attention of a step's tokens, single ones and portions of prompts, over 4-bit pages (``kernels.cache4_attention``);
* ``linear``: products of a step's rows with a weight in 4 bits (``kernels.linear4``).

What is held in 4 bits are groups of consecutive numbers with a scale s and a least value m in bfloat16: a number is m + s * code.
How long each request is and how many tokens it brings follow from the case; the values follow from the seed.
"""
import math

import numpy as np
import torch

own = False
DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}
GROUP = 32                     # channels of a group in the cache
POSITIONS = 40960


def listed():
    return [
        # one user of a small model: a token's heads, launches and latency
        dict(name="write-1", kind="write", tokens=1, heads=16, kv_heads=8, dim=128, dtype="bf16", page=16, norm=True, rot=128, pairs=False),
        # the float32 engine, as one runs it to check a model: heads of 80 channels, half of them rotated in pairs
        dict(name="write-37-f32", kind="write", tokens=37, heads=10, kv_heads=5, dim=80, dtype="f32", page=8, norm=False, rot=40, pairs=True),
        # portions of prompts that fill a step: the rows' bytes
        dict(name="write-8192", kind="write", tokens=8192, heads=32, kv_heads=8, dim=128, dtype="bf16", page=16, norm=True, rot=128, pairs=False),
        # one user of a small model, a token over a short context: latency
        dict(name="attend-1x1", kind="attend", requests=1, new=1, context=1024, heads=16, kv_heads=8, dim=128, dtype="bf16", page=16, window=0),
        # a full batch at the contexts of chats
        dict(name="attend-64x1", kind="attend", requests=64, new=1, context=4096, heads=32, kv_heads=8, dim=128, dtype="bf16", page=16, window=0),
        # long contexts of uneven length: the cache's bytes
        dict(name="attend-24x1-long", kind="attend", requests=24, new=1, context=32768, heads=32, kv_heads=8, dim=128, dtype="bf16", page=16, window=0),
        # portions of prompts over what is cached already, beside requests that bring less: products
        dict(name="attend-4x512", kind="attend", requests=4, new=512, context=4096, heads=32, kv_heads=8, dim=128, dtype="bf16", page=16, window=0),
        # the float32 engine: a group of two heads of 48 channels, a few tokens each, a window
        dict(name="attend-3x13-f32", kind="attend", requests=3, new=13, context=777, heads=10, kv_heads=5, dim=48, dtype="f32", page=16, window=256),
        # one user: the projection to queries, keys and values
        dict(name="linear-1", kind="linear", tokens=1, columns=4096, rows=6144, group=32, dtype="bf16"),
        # eight users: both halves of a gated feed-forward
        dict(name="linear-8", kind="linear", tokens=8, columns=4096, rows=24576, group=128, dtype="bf16"),
        # a full batch: the way back from the feed-forward
        dict(name="linear-64", kind="linear", tokens=64, columns=12288, rows=4096, group=64, dtype="bf16"),
        # the float32 engine, sizes that no tile divides
        dict(name="linear-5-f32", kind="linear", tokens=5, columns=1000, rows=777, group=32, dtype="f32"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / (50 if case["dtype"] == "bf16" else 5))


def draw(rng):
    kind = rng.choices(["write", "attend", "linear"], [25, 45, 30])[0]
    dtype = rng.choices(["bf16", "f32"], [4, 1])[0]
    if kind == "linear":
        case = dict(kind=kind, tokens=_spread(rng, 1, 128 if dtype == "bf16" else 16), columns=_spread(rng, 64, 12288), rows=_spread(rng, 16, 24576),
                    group=rng.choice([32, 64, 128]), dtype=dtype)
        if rng.random() < 0.7:         # layers' sizes are mostly multiples of 64
            case["columns"], case["rows"] = -(-case["columns"] // 64) * 64, -(-case["rows"] // 64) * 64
        return case
    kv_heads, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 5, 8])
    dim = rng.choice([64, 128, 128, 128, 48, 80, 96, 256] if dtype == "bf16" else [32, 48, 64, 128])
    page = rng.choice([8, 16, 16, 32, 64])
    if kind == "write":
        tokens = _spread(rng, 1, 8192 if dtype == "bf16" else 2048)
        rot = rng.choice([0, dim, dim, dim, dim // 2])
        case = dict(kind=kind, tokens=tokens, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, norm=rng.random() < 0.6, rot=rot,
                    pairs=rng.random() < 0.3)
        while case["tokens"] > 1 and _cost(case) > 0.9 * _cost(listed()[2]):
            case["tokens"] //= 2
        return case
    new = rng.choice([1, 1, 1, _spread(rng, 2, 32), _spread(rng, 16, 1024 if dtype == "bf16" else 64)])
    context = _spread(rng, 16, 32768 if dtype == "bf16" else 4096)
    most = (1 << 19) if dtype == "bf16" else (1 << 13)          # tokens in the cache
    case = dict(kind=kind, requests=max(1, min(_spread(rng, 1, 96), most // context)), new=new, context=context, heads=kv_heads * group, kv_heads=kv_heads,
                dim=dim, dtype=dtype, page=page, window=rng.choice([0, 0, 0, _spread(rng, 16, 4096)]))
    top = 0.9 * max(_cost(c) for c in listed() if c["kind"] == "attend")
    while case["requests"] > 1 and (_cost(case) > top or case["requests"] * case["heads"] * new * (context + new) > 4e8):
        case["requests"] //= 2
    while case["new"] > 1 and (_cost(case) > top or case["heads"] * case["new"] * (context + new) > 4e8):
        case["new"] //= 2
    return case


# ---- what follows from the case alone ----------------------------------------------------------------------------------

def _sizes(case):
    """New tokens and lengths with them: the first request has what the case says; of four and more, one brings nothing and one has nothing cached."""
    rng, n = np.random.default_rng(7), case["requests"]
    new = rng.integers(max(1, case["new"] // 2), case["new"] + 1, n)
    context = np.round(case["context"] * np.exp(rng.uniform(-2.5, 0.0, n))).astype(np.int64)
    new[0], context[0] = case["new"], case["context"]
    if n >= 4:
        context[1], new[n - 1] = 0, 0
    return new, context + new


def _padded(tokens):
    """Rows of a step: its tokens and a few behind them that nobody asked for."""
    return tokens + (3 if tokens > 8 else 0)


def _row_bytes(dim):
    return 20 * -(-dim // GROUP)       # codes, scale and least value of every group


def work(case):
    es = BYTES[case["dtype"]]
    if case["kind"] == "linear":
        t, k, n = case["tokens"], case["columns"], case["rows"]
        return dict(bytes=n * k // 2 + n * -(-k // case["group"]) * 4 + t * (k + n) * es, flops=2 * t * n * k)
    nh, nkv, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "write":
        t = _padded(case["tokens"])
        rows = t * (2 * nh + 2 * nkv) * d * es + t * 2 * nkv * d * 2 + t * 12 + t * case["rot"] * 4
        return dict(bytes=rows + case["tokens"] * 2 * nkv * _row_bytes(d), flops=t * (2 * nh + 4 * nkv) * d * 4)
    new, length = _sizes(case)
    w, old = case["window"], length - new
    low = np.maximum(0, old - w + 1) if w else 0 * old               # (the first key that a token sees)
    pairs = 0
    for n, o in zip(new.tolist(), old.tolist()):
        seen = o + 1 + np.arange(n, dtype=np.int64)
        pairs += int((np.minimum(seen, w) if w else seen).sum())
    keys = int((length - low)[new > 0].sum())
    return dict(bytes=keys * nkv * 2 * _row_bytes(d) + 2 * int(new.sum()) * nh * d * es + -(-keys // case["page"]) * 4, flops=4 * nh * d * pairs)


# ---- groups of 4-bit codes ------------------------------------------------------------------------------------------------

def _encode(x, group):
    """Codes, scales and least values of groups of consecutive numbers of the last axis, of x's precision."""
    g = x.unflatten(-1, (-1, group))
    low = g.amin(-1)
    scale = ((g.amax(-1) - low) / 15).to(torch.bfloat16)
    least = low.to(torch.bfloat16)
    s, m = scale.to(x.dtype).unsqueeze(-1), least.to(x.dtype).unsqueeze(-1)
    codes = torch.where(s > 0, torch.round((g - m) / torch.where(s > 0, s, 1.0)), 0.0).clamp(0, 15).to(torch.uint8)
    return codes, scale, least


def _decode(codes, scale, least):
    """[..., groups, numbers of a group] codes -> values in 32 bits."""
    return codes.float().mul_(scale.float().unsqueeze(-1)).add_(least.float().unsqueeze(-1))


def _head_groups(x):
    """Heads [..., d] as [..., d up to a whole group]: what is added repeats the last channel, so that it changes no group's range."""
    d = x.shape[-1]
    more = -d % GROUP
    return torch.cat([x, x[..., -1:].expand(*x.shape[:-1], more)], -1) if more else x


def _words(scale, least):
    return torch.stack([scale, least], -1).contiguous().view(torch.uint8).flatten(-2)      # [..., 4] bytes: scale, least value


def _pages_of(codes, scale, least):
    """[pages, kv heads, slots, groups, 32] codes -> [pages, kv heads, bytes]: the groups' codes slot by slot, then the slots' scales."""
    pages, nkv, ps, groups, _ = codes.shape
    two = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return torch.cat([two.transpose(2, 3).reshape(pages, nkv, -1), _words(scale, least).reshape(pages, nkv, -1)], 2)


def _values_of(page_bytes, ps, dim):
    """[..., bytes of a page] -> [..., slots, dim] values in 32 bits."""
    groups = -(-dim // GROUP)
    codes = page_bytes[..., :groups * ps * 16].unflatten(-1, (groups, ps, 16)).transpose(-3, -2)       # [..., slots, groups, 16]
    words = page_bytes[..., groups * ps * 16:].contiguous().view(torch.bfloat16).unflatten(-1, (ps, groups, 2))
    return _decode(torch.stack([codes & 15, codes >> 4], -1).flatten(-2), words[..., 0], words[..., 1]).flatten(-2)[..., :dim]


def _weight_bytes(w, group):
    """A weight [rows, columns] in tiles of 16 rows and 128 columns [row tiles, column tiles, bytes]: 1,024 bytes of codes, then every row's scales."""
    n, k = w.shape
    rows, cols = -(-n // 16) * 16, -(-k // 128) * 128
    full = torch.zeros((rows, cols), device=w.device)
    full[:n, :k] = w
    codes, scale, least = _encode(full, group)
    codes = codes.view(rows // 16, 2, 8, cols // 128, 4, 4, 4, 2)                 # tile, half, row; tile, 32, 8, pair, place in the pair
    codes = codes.permute(0, 3, 1, 2, 5, 4, 7, 6)                                 # tile, tile, half, row, 8, 32, place, pair
    codes = codes.reshape(rows // 16, cols // 128, -1)
    words = _words(scale, least).view(rows // 16, 16, cols // 128, 128 // group * 4).transpose(1, 2)
    return torch.cat([codes[..., 0::2] | (codes[..., 1::2] << 4), words.reshape(rows // 16, cols // 128, -1)], 2)


def _weight_of(data, group, n, k):
    """The weight's values in 32 bits."""
    rt, ct, _ = data.shape
    two = data[..., :1024]
    codes = torch.stack([two & 15, two >> 4], -1).view(rt, ct, 2, 8, 4, 4, 2, 4).permute(0, 2, 3, 1, 5, 4, 7, 6).reshape(rt * 16, ct * 128 // group, group)
    words = data[..., 1024:].contiguous().view(torch.bfloat16).view(rt, ct, 16, 128 // group, 2).transpose(1, 2).reshape(rt * 16, ct * 128 // group, 2)
    return _decode(codes, words[..., 0], words[..., 1]).flatten(-2)[:n, :k]


# ---- inputs -----------------------------------------------------------------------------------------------------------------

def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    dt = TYPES[case["dtype"]]

    def normal(shape, dtype, scale=1.0):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype).mul_(scale)

    s = dict(case=case)
    if case["kind"] == "linear":
        t, k, n = case["tokens"], case["columns"], case["rows"]
        s.update(x=normal((t, k), dt), weight=_weight_bytes(normal((n, k), torch.float32, 1 / math.sqrt(k)), case["group"]),
                 out=torch.empty((t, n), device=DEVICE, dtype=dt))
        return s
    nh, nkv, d, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "write":
        t, total = case["tokens"], _padded(case["tokens"])
        # a step's tokens are runs of a few requests, each from its own position on
        runs = np.sort(rng.choice(np.arange(1, t), min(t - 1, 7), replace=False)) if t > 1 else np.zeros(0, np.int64)
        first = np.concatenate([[0], runs])
        which = np.searchsorted(runs, np.arange(t), side="right")
        begin = rng.integers(0, POSITIONS - t, len(first))
        place = np.arange(t) - first[which]
        position = begin[which] + place
        counts = -(-np.bincount(which, minlength=len(first)) // ps) + 1                      # (a run begins anywhere in its first page)
        base, pages = np.cumsum(counts) - counts, int(counts.sum())
        page_of = rng.permutation(pages)
        slots = np.full(total, -1, np.int64)
        slots[:t] = page_of[base[which] + (begin[which] % ps + place) // ps] * ps + position % ps
        positions = np.zeros(total, np.int32)
        positions[:t] = position
        rot = case["rot"]
        if rot:
            angle = np.arange(POSITIONS)[:, None] * (1e6 ** (-np.arange(0, rot, 2) / rot))[None]
            s.update(cos=_dev(np.cos(angle).astype(np.float32)), sin=_dev(np.sin(angle).astype(np.float32)))
        if case["norm"]:
            s.update(q_norm=1 + normal((d,), torch.float32, 0.2), k_norm=1 + normal((d,), torch.float32, 0.2))
        bytes_of = ps * _row_bytes(d)
        s.update(qkv=normal((total, (nh + 2 * nkv) * d), dt, 1.5), positions=_dev(positions), slots=_dev(slots), q_out=torch.empty((total, nh, d), device=DEVICE, dtype=dt),
                 k_values=torch.empty((total, nkv, d), device=DEVICE, dtype=torch.bfloat16), v_values=torch.empty((total, nkv, d), device=DEVICE, dtype=torch.bfloat16),
                 k_cache=torch.zeros((pages, nkv, bytes_of), dtype=torch.uint8, device=DEVICE), v_cache=torch.zeros((pages, nkv, bytes_of), dtype=torch.uint8, device=DEVICE),
                 eps=1e-6, err=torch.zeros(1, dtype=torch.int32, device=DEVICE))
        return s
    new, length = _sizes(case)
    t, pages = int(new.sum()), -(-length // ps)
    total = int(pages.sum()) + 1
    table = np.full((case["requests"], max(1, int(pages.max()))), -1, np.int32)
    ids, at = rng.permutation(total), 0
    for b, m in enumerate(pages):
        table[b, :m] = ids[at:at + m]
        at += m

    def cache():
        done = torch.empty((total, nkv, ps * _row_bytes(d)), dtype=torch.uint8, device=DEVICE)
        each = max(1, (1 << 26) // (nkv * ps * d))
        for lo in range(0, total, each):
            rows = normal((min(each, total - lo), nkv, ps, d), torch.float32)
            done[lo:lo + each] = _pages_of(*_encode(_head_groups(rows), GROUP))
        return done

    # queries and keys behind a norm: scores of a few units
    s.update(q=normal((t, nh, d), dt, 1.5), k_cache=cache(), v_cache=cache(), lengths=_dev(length.astype(np.int32)),
             token_start=_dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)), table=_dev(table), out=torch.empty((t, nh, d), device=DEVICE, dtype=dt),
             scale=1.0 / math.sqrt(d), most=int(new.max()), err=torch.zeros(1, dtype=torch.int32, device=DEVICE))
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------

def _rotated(x, cos, sin, pairs):
    """The first channels of heads [tokens, heads, d] rotated by [tokens, rot / 2] angles: in pairs of neighbours or of halves."""
    half = cos.shape[-1]
    c, n = cos.unsqueeze(1), sin.unsqueeze(1)
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if pairs else (x[..., :half], x[..., half:2 * half])
    u, v = a * c - b * n, a * n + b * c
    turned = torch.stack([u, v], -1).flatten(-2) if pairs else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _plain_write(s):
    c = s["case"]
    nh, nkv, d, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    q, k, v = s["qkv"].float().unflatten(1, (-1, d)).split([nh, nkv, nkv], 1)
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + s["eps"]) * s["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + s["eps"]) * s["k_norm"]
    if c["rot"]:
        at = s["positions"].long()
        cos, sin = s["cos"][at], s["sin"][at]
        q, k = _rotated(q, cos, sin, c["pairs"]), _rotated(k, cos, sin, c["pairs"])
    codes, scale, least = _encode(_head_groups(torch.stack([k, v])), GROUP)                  # [2, tokens, kv heads, groups, ...]
    groups = codes.shape[-2]
    slots = torch.where(s["slots"] >= 0, s["slots"], s["slots"][0])                          # padding does the first token again
    at = torch.where(s["slots"] >= 0, torch.arange(slots.shape[0], device=slots.device), 0)
    page, place = slots // ps, slots % ps
    two = (codes[..., 0::2] | (codes[..., 1::2] << 4))[:, at].transpose(2, 3)                # [2, tokens, groups, kv heads, 16]
    words = _words(scale, least)[:, at]                                                      # [2, tokens, kv heads, bytes of a slot]
    grp = torch.arange(groups, device=slots.device)
    pages = s["k_cache"].shape[0], nkv
    k_codes = s["k_cache"][..., :groups * ps * 16].view(*pages, groups, ps, 16)
    v_codes = s["v_cache"][..., :groups * ps * 16].view(*pages, groups, ps, 16)
    k_codes[page[:, None], :, grp, place[:, None]] = two[0]
    v_codes[page[:, None], :, grp, place[:, None]] = two[1]
    s["k_cache"][..., groups * ps * 16:].view(*pages, ps, groups * 4)[page, :, place] = words[0]
    s["v_cache"][..., groups * ps * 16:].view(*pages, ps, groups * 4)[page, :, place] = words[1]
    values = _decode(codes, scale, least).flatten(-2)[..., :d].to(torch.bfloat16)
    return dict(q=q.to(s["qkv"].dtype), k=values[0], v=values[1])


def _plain_attend(s):
    c = s["case"]
    nkv, d, most, w = c["kv_heads"], c["dim"], s["most"], c["window"]
    start, length = s["token_start"].long(), s["lengths"].long()
    t, n = s["q"].shape[0], length.shape[0]
    new = start[1:] - start[:-1]
    place = torch.arange(most, device=start.device)
    live = place < new[:, None]
    rows = torch.where(live, start[:-1, None] + place, 0)                                    # [requests, tokens]
    table = s["table"].long().clamp(min=0)
    key = torch.arange(table.shape[1] * c["page"], device=start.device)

    def values(cache):
        return _values_of(cache[table].transpose(1, 2), c["page"], d).flatten(2, 3)          # [requests, kv heads, keys, d]

    position = (length - new)[:, None] + place
    seen = key <= position[..., None]
    if w:
        seen = seen & (key > position[..., None] - w)
    seen = (seen & live[..., None])[:, None, :, None]                                        # [requests, 1, tokens, 1, keys]
    q = s["q"][rows].unflatten(2, (nkv, -1)).permute(0, 2, 1, 3, 4).float()                  # [requests, kv heads, tokens, group, d]
    scores = (q.flatten(2, 3) @ values(s["k_cache"]).transpose(2, 3)).mul_(s["scale"]).unflatten(2, (most, -1))
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.flatten(2, 3) @ values(s["v_cache"])).unflatten(2, (most, -1)) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 2, 1, 3, 4).flatten(2, 3)[live].reshape(t, c["heads"], d).to(s["q"].dtype)


def _plain_linear(s):
    c = s["case"]
    return (s["x"].float() @ _weight_of(s["weight"], c["group"], c["rows"], c["columns"]).T).to(s["x"].dtype)


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if not own:
        return dict(write=_plain_write, attend=_plain_attend, linear=_plain_linear)[c["kind"]](s)
    from xinfer_b200 import kernels
    if c["kind"] == "write":
        kernels.cache4_write(s["q_out"], s["k_cache"], s["v_cache"], s["qkv"], s["positions"], s["slots"], c["page"], s["err"], q_norm=s.get("q_norm"),
                             k_norm=s.get("k_norm"), eps=s["eps"], cos=s.get("cos"), sin=s.get("sin"), interleaved=c["pairs"], values=(s["k_values"], s["v_values"]))
        return dict(q=s["q_out"], k=s["k_values"], v=s["v_values"])
    if c["kind"] == "attend":
        if "scratch" not in s:         # the workspace that a program keeps for its steps
            s["scratch"] = torch.empty(kernels.cache4_attention_scratch(s["q"].shape[0], c["requests"], c["heads"], c["kv_heads"], c["dim"], s["q"].dtype, s["most"]),
                                       device=DEVICE)
        kernels.cache4_attention(s["out"], s["q"], s["k_cache"], s["v_cache"], s["lengths"], s["token_start"], s["table"], c["page"], s["scale"], s["err"],
                                 scratch=s["scratch"], window=c["window"] or None, longest=s["most"])
        return s["out"]
    if "scratch" not in s:
        s["scratch"] = torch.empty(kernels.linear4_scratch(c["tokens"], c["rows"], c["columns"], s["x"].dtype), device=DEVICE)
    kernels.linear4(s["out"], s["x"], s["weight"], scratch=s["scratch"])
    return s["out"]


# ---- the same in 64 bits, head by head --------------------------------------------------------------------------------------

def _exact_values(x):
    """What 4 bits hold of heads [tokens, kv heads, d] in 64 bits."""
    out = torch.empty_like(x)
    for lo in range(0, x.shape[-1], GROUP):
        g = x[..., lo:lo + GROUP]
        low, high = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        scale, least = ((high - low) / 15).to(torch.bfloat16).double(), low.to(torch.bfloat16).double()
        code = torch.nan_to_num(torch.round((g - least) / scale), nan=0.0).clamp(0, 15)
        out[..., lo:lo + GROUP] = least + scale * code
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        n, k, group = case["rows"], case["columns"], case["group"]
        out = torch.empty((case["tokens"], n), dtype=torch.float64, device=DEVICE)
        x, data = s["x"].double(), s["weight"]
        col = torch.arange(k, device=DEVICE)
        inside = col % 128
        # where a column's code lies in its tile: the byte within a row's, which of its halves
        eight, j, e = inside % 32 // 8, inside // 32, inside % 8
        nibble = (e % 2) * 4 + e // 2
        for lo in range(0, n, 2048):
            row = torch.arange(lo, min(n, lo + 2048), device=DEVICE)[:, None]
            at = (row % 16 // 8) * 512 + (row % 8) * 64 + eight * 16 + j * 4 + nibble // 2
            code = (data[row // 16, col // 128, at].long() >> (4 * (nibble % 2))) & 15
            word = 1024 + (row % 16) * (512 // group) + inside // group * 4
            pick = torch.stack([data[row // 16, col // 128, word + i] for i in range(4)], -1).contiguous().view(torch.bfloat16).double()
            out[:, lo:lo + 2048] = x @ (pick[..., 1] + pick[..., 0] * code).T
        return out
    if case["kind"] == "write":
        x, at = s["qkv"].double(), s["positions"].long()
        nh, d, half = case["heads"], case["dim"], case["rot"] // 2
        heads = []
        for h in range(nh + case["kv_heads"]):
            y = x[:, h * d:(h + 1) * d].clone()
            if case["norm"]:
                y *= (s["q_norm"] if h < nh else s["k_norm"]).double() / ((y * y).sum(1, keepdim=True) / d + s["eps"]).sqrt()
            if half:       # a pair is a complex number
                one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["pairs"] else (slice(0, half), slice(half, 2 * half))
                turned = torch.complex(y[:, one], y[:, two]) * torch.complex(s["cos"][at].double(), s["sin"][at].double())
                y[:, one], y[:, two] = turned.real, turned.imag
            heads.append(y)
        return dict(q=torch.stack(heads[:nh], 1), k=_exact_values(torch.stack(heads[nh:], 1)), v=_exact_values(x.unflatten(1, (-1, d))[:, nh + case["kv_heads"]:]))
    nkv, group, w, ps, d = case["kv_heads"], case["heads"] // case["kv_heads"], case["window"], case["page"], case["dim"]
    groups = -(-d // GROUP)
    start, length = s["token_start"].tolist(), s["lengths"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    channel = torch.arange(d, device=DEVICE)
    for b in range(case["requests"]):
        a, z, have = start[b], start[b + 1], length[b]
        if a == z:
            continue
        j = torch.arange(have, device=DEVICE)
        page, slot = s["table"][b].long()[j // ps][:, None], (j % ps)[:, None]
        p = have - (z - a) + torch.arange(z - a, device=DEVICE)[:, None]
        hidden = (j > p) | (j <= p - w) if w else j > p
        byte = (channel // GROUP * ps + slot) * 16 + channel % GROUP // 2
        word = groups * ps * 16 + (slot * groups + channel // GROUP) * 4
        for g in range(nkv):
            k, v = (torch.stack([cache[page, g, word + i] for i in range(4)], -1).contiguous().view(torch.bfloat16).double() for cache in (s["k_cache"], s["v_cache"]))
            k, v = (x[..., 1] + x[..., 0] * ((cache[page, g, byte].long() >> (channel % 2 * 4)) & 15) for x, cache in ((k, s["k_cache"]), (v, s["v_cache"])))
            for h in range(g * group, (g + 1) * group):
                out[a:z, h] = torch.softmax((s["q"][a:z, h].double() @ k.T * s["scale"]).masked_fill(hidden, -math.inf), 1) @ v
    return out
