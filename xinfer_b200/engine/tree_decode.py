"""Decoding that verifies a tree of drafted tokens per request and step.

A step gives the model every request's last token (the root) and tokens that were guessed to follow it, as a tree: ``draft`` names them.
The model's own choice behind each of them is made exactly as without drafts (the noise of a draw depends on the request's seed and on
how many tokens came before it), the path that these choices confirm is kept, and the choice behind its end is the next root.  The
tokens that come out are therefore those of decoding one by one, a path at a time.

Only the device knows how long the paths are while a step runs: pages, slots and lengths are kept there (``kernels.cache_slots``), the
drafted tokens' keys and values stay outside the cache until the path is known (``kernels.tree_attention``) and then go to their slots
in every layer with one launch (``kernels.cache_commit``).
"""
from __future__ import annotations

import dataclasses
from typing import Callable, Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from .. import kernels
from ..config.generation import join_eos
from ..parts import LayerCache, StepContext, TreeStep
from ..parts.attention import Attention
from ..sampling import SamplingParams
from ..sampling.sampler import Sampler
from .runner import ModelRunner, StepError

Draft = Callable[[List[int]], Tuple[List[int], List[int]]]


@dataclasses.dataclass
class LogitRules:
    """What changes a request's logits before a token is chosen, beside its ``SamplingParams``' frequency and presence penalties (which
    count every token generated so far): ``repetition_penalty`` for the prompt's and the generated tokens, ``bias`` per token id, and
    ``allowed``: given the tokens so far, truth values over the vocabulary (or None: all), for a grammar."""

    repetition_penalty: float = 1.0
    bias: Dict[int, float] = dataclasses.field(default_factory=dict)
    allowed: Optional[Callable[[List[int]], Optional[np.ndarray]]] = None

    def validate(self) -> None:
        tiny, most = np.finfo(np.float32).tiny, np.finfo(np.float32).max      # (logits are divided by it in float32)
        if not tiny <= self.repetition_penalty <= most:
            raise ValueError(f"repetition_penalty must be a number above 0, got {self.repetition_penalty}")
        if any(x != x for x in self.bias.values()):
            raise ValueError("a bias that is no number")

    def active(self) -> bool:
        return self.repetition_penalty != 1.0 or bool(self.bias) or self.allowed is not None


def lookup_draft(most: int, longest: int = 8, match: int = 3) -> Draft:
    """Drafts from the text itself: what followed earlier occurrences of its last tokens (``match`` of them, then fewer), the latest
    first, up to ``longest`` tokens each, merged where they begin alike into one tree of up to ``most`` tokens."""

    def draft(tokens: List[int]) -> Tuple[List[int], List[int]]:
        drafted: List[int] = []
        parents: List[int] = []
        children: Dict[Tuple[int, int], int] = {}
        for n in range(min(match, len(tokens) - 1), 0, -1):
            tail = tokens[-n:]
            for at in range(len(tokens) - n - 1, -1, -1):
                if tokens[at:at + n] != tail:
                    continue
                node = 0
                for t in tokens[at + n:at + n + longest]:
                    if (node, t) not in children:
                        if len(drafted) >= most:
                            return drafted, parents
                        drafted.append(t)
                        parents.append(node)
                        children[node, t] = len(drafted)
                    node = children[node, t]
            if drafted:
                break
        return drafted, parents

    return draft


def tree_facts(parents: Sequence[int]) -> Tuple[np.ndarray, np.ndarray]:
    """Depths, and truth values [n, n]: which nodes lie on whose path, of a tree whose root is node 0 (its parent: -1)."""
    n = len(parents)
    depth = np.zeros(n, dtype=np.int32)
    on = np.eye(n, dtype=bool)
    for i, p in enumerate(parents):
        if i == 0:
            if p != -1:
                raise ValueError("a tree's first node is its root")
            continue
        if not 0 <= p < i:
            raise ValueError(f"node {i} of a tree has the parent {p}: a parent comes before its children")
        depth[i] = depth[p] + 1
        on[i] |= on[p]
    return depth, on


def bit_words(on: np.ndarray, words: int) -> np.ndarray:
    """Truth values [n, m] as int32 words, lowest bit first."""
    bits = np.zeros((on.shape[0], words * 32), dtype=np.uint8)
    bits[:, : on.shape[1]] = on
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32).reshape(on.shape[0], words).view(np.int32)


@dataclasses.dataclass
class _Request:
    tokens: List[int]          # the prompt and what was generated
    prompt: int
    params: SamplingParams
    seed: int
    most: int                  # tokens to generate
    cached: int = 0
    done: bool = False

    def generated(self) -> List[int]:
        return self.tokens[self.prompt:]


class TreeDecoder:
    """Generates with drafted trees over a runner's model and page tensors.  The runner must have no open requests, and none are opened
    while this decoder generates.  Models whose layers all are grouped-query attention (Qwen3's).  Prompts go through the model in steps
    of up to ``max_num_batched_tokens``, in portions of up to ``prefill_chunk_size`` (``EngineConfig``'s limits)."""

    def __init__(self, runner: ModelRunner, *, max_nodes: int = 32, max_depth: int = 12, eos_token_ids=None,
                 max_num_batched_tokens: int = 8192, prefill_chunk_size: int = 8192):
        self.runner, self.max_nodes, self.max_depth = runner, int(max_nodes), int(max_depth)
        if not 1 <= self.max_nodes <= 1024 or not 1 <= self.max_depth:
            raise ValueError("trees of 1 to 1,024 nodes, paths of at least one")
        self.max_batched, self.prefill_chunk = int(max_num_batched_tokens), int(prefill_chunk_size)
        if self.max_batched < 1 or self.prefill_chunk < 1:
            raise ValueError("steps and portions of at least one token")
        plan = runner.plan
        mixers = [runner.model.blocks[run.block].mixer for run in plan.runs]
        if any(type(m) is not Attention for m in mixers) or any(run.cache_from is not None for run in plan.runs) or runner.has_state \
                or len(runner.cache.groups) != 1:
            raise ValueError("drafted trees run on models whose layers all are grouped-query attention over caches of their own")
        if runner.cache.live_requests():
            raise StepError("the runner has open requests: their pages are the host's")
        self.eos_token_ids = tuple(join_eos(plan.eos_token_ids, None) if eos_token_ids is None else eos_token_ids)
        self.page_size = runner.cache.groups[0].page_size
        self.num_pages = runner.cache.groups[0].num_pages
        dev, B, T = runner.device, runner.max_num_seqs, runner.max_num_seqs * self.max_nodes
        self.caches: List[LayerCache] = []
        for cache in runner.layer_caches:
            _, nkv, _, d = cache["k"].shape
            fresh = {name: torch.zeros((T, nkv, d), dtype=cache["k"].dtype, device=dev) for name in ("k_new", "v_new")}
            self.caches.append(LayerCache({**cache.tensors, **fresh}, cache.group, cache.page_size))
        self.commit = kernels.commit_table(*([c[name] for c in self.caches] for name in ("k", "v", "k_new", "v_new")))
        self.width = -(-runner.max_model_len // self.page_size)
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)  # noqa: E731
        self.table, self.free_ring = i32(B, self.width), i32(self.num_pages)
        self.rings, self.lengths = [i32(2), i32(2)], [i32(B), i32(B)]
        self.accepted, self.next_tokens, self.path = i32(B), i32(B), i32(B, self.max_depth)
        self.sampler = Sampler(dev, T)
        self.steps = self.drafted = self.confirmed = 0

    # ---- the device's bookkeeping ----------------------------------------------------------------------------------------
    def _reset(self) -> None:
        self.free_ring.copy_(torch.arange(self.num_pages, dtype=torch.int32))
        self.rings[0].copy_(torch.tensor([0, self.num_pages], dtype=torch.int32))
        self.lengths[0].zero_()

    def _slots(self, new_tokens: torch.Tensor, capacity: int):
        """Pages and slots for so many more tokens of every request; the lengths and the ring are those afterwards."""
        dev, B = self.runner.device, new_tokens.numel()
        slots = torch.empty(max(capacity, 1), dtype=torch.int64, device=dev)
        positions, request_of = (torch.empty(max(capacity, 1), dtype=torch.int32, device=dev) for _ in range(2))
        start = torch.empty(B + 1, dtype=torch.int32, device=dev)
        kernels.cache_slots(slots, positions, request_of, start, self.lengths[1][:B], self.rings[1], self.table[:B], self.free_ring, self.rings[0],
                            self.lengths[0][:B], new_tokens, self.page_size, self.runner.err)
        self.rings.reverse()
        self.lengths.reverse()
        return slots, positions, request_of, start

    def _send(self, *arrays: np.ndarray) -> List[torch.Tensor]:
        """int32 arrays to the device with one copy."""
        flat = [np.ascontiguousarray(a, dtype=np.int32).reshape(-1) for a in arrays]
        dev = torch.from_numpy(np.concatenate(flat)).pin_memory().to(self.runner.device, non_blocking=True)
        out, at = [], 0
        for a, f in zip(arrays, flat):
            out.append(dev[at:at + f.size].view(np.shape(a)))
            at += f.size
        return out

    # ---- one step of the model ------------------------------------------------------------------------------------------
    def _forward(self, token_ids, positions, request_of, start, rows, counts, context: np.ndarray, tree: Optional[TreeStep], starts=None,
                 table=None) -> torch.Tensor:
        """``rows`` None: no logits are wanted."""
        r, B = self.runner, len(counts)
        table = self.table[:B] if table is None else table
        q_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        T = int(q_start[-1])
        ctx = StepContext(
            dtype=r.dtype, device=r.device, num_tokens=T, num_entries=B, token_ids=token_ids, positions=positions[:T], req_of_token=request_of[:T],
            q_start=start, start_pos=starts if starts is not None else tree.context, slots=start,
            logit_rows=start if rows is None else rows, num_logit_rows=0 if rows is None else rows.numel(), tables=[table.reshape(-1)],
            strides=[self.width], err=r.err, workspace=r.workspace, h_q_start=q_start, h_start_pos=context, real_tokens=T,
            real_entries=B, max_context=int((context + counts).max()), tree=tree)
        return r.model.forward(ctx, self.caches, r.layer_states)

    def _choose(self, logits: torch.Tensor, requests: List[_Request], counts, parents, drafted, depth, on, facts, rules: LogitRules) -> torch.Tensor:
        """The model's token behind every row: rules, then the sampler.  ``facts``: the device's (first rows, drafted, ancestors)."""
        row_request = np.repeat(np.arange(len(requests)), counts)
        if rules.active() or any(q.params.has_penalties for q in requests):
            V = logits.shape[1]
            first, tokens_dev, ancestors = facts
            # the rows' own paths count the last token of a request; the lists hold the ones before it
            lists = [q.tokens[:-1] if on is not None else q.tokens for q in requests]
            pen = np.array([[rules.repetition_penalty, q.params.frequency_penalty or 0.0, q.params.presence_penalty or 0.0] for q in requests], np.float32)
            arrays = [np.concatenate([np.asarray(t, np.int32) for t in lists]), np.concatenate([[0], np.cumsum([len(t) for t in lists])]),
                      np.array([min(q.prompt, len(t)) for q, t in zip(requests, lists)]), row_request]
            bias = mask = None
            if rules.bias:
                n = len(rules.bias)
                arrays += [np.arange(len(row_request) + 1) * n, np.tile(np.fromiter(rules.bias.keys(), np.int32, n), len(row_request))]
            if rules.allowed is not None:
                arrays += self._masks(requests, counts, drafted, on, rules.allowed, V)
            sent = self._send(*arrays)
            if rules.bias:
                values = torch.tensor(list(rules.bias.values()), dtype=torch.float32).repeat(len(row_request)).to(logits.device)
                bias = (sent[4], sent[5], values)
            if rules.allowed is not None:
                mask = sent[-2].view(-1, -(-V // 32))
            kernels.logit_rules(logits, logits, torch.from_numpy(pen[row_request]).to(logits.device), sent[0], sent[1], sent[2], list_of_row=sent[3],
                                tree=(tokens_dev, ancestors, first) if on is not None else None, bias=bias, mask=mask,
                                mask_of_row=sent[-1] if mask is not None else None)
        params = [dataclasses.replace(requests[b].params, frequency_penalty=None, presence_penalty=None) for b in range(len(requests))]
        draws = [len(requests[b].generated()) + int(d) for b, d in zip(row_request, depth)]
        return self.sampler.sample(logits, [params[b] for b in row_request], [requests[b].seed for b in row_request], draws)

    @staticmethod
    def _masks(requests, counts, drafted, on, allowed, V: int):
        """The rows' grammar masks as words, and which row has which (-1: none)."""
        words, which, made, at = -(-V // 32), [], [], 0
        for b, (q, n) in enumerate(zip(requests, counts)):
            for i in range(n):
                path = [int(drafted[at + j]) for j in np.nonzero(on[b][i])[0]] if on is not None else []
                ok = allowed((q.tokens[:-1] if on is not None else q.tokens) + path)
                which.append(-1 if ok is None else len(made))
                if ok is not None:
                    made.append(bit_words(np.asarray(ok, bool)[None], words))
            at += n
        return [np.concatenate(made) if made else np.zeros((1, words), np.int32), np.array(which)]

    # ---- generation --------------------------------------------------------------------------------------------------------
    def generate(self, prompts: Sequence[Sequence[int]], params=None, draft: Optional[Draft] = None, rules: Optional[LogitRules] = None) -> List[List[int]]:
        """The tokens generated for every prompt.  ``params``: one ``SamplingParams`` or one per prompt (``seed`` None: the prompt's place).
        ``draft``: given a request's tokens, the tokens guessed behind the last one and their parents in the tree whose root (0) that
        is; default ``lookup_draft``."""
        if self.runner.cache.live_requests():
            raise StepError("the runner has open requests: their pages are the host's")
        rules = rules or LogitRules()
        rules.validate()
        draft = draft or lookup_draft(self.max_nodes - 1, self.max_depth - 1)
        if not prompts:
            return []
        if len(prompts) > self.runner.max_num_seqs:
            raise ValueError(f"{len(prompts)} prompts; the runner takes {self.runner.max_num_seqs} requests")
        per = [params or SamplingParams()] * len(prompts) if params is None or isinstance(params, SamplingParams) else list(params)
        if len(per) != len(prompts):
            raise ValueError(f"{len(per)} sampling params for {len(prompts)} prompts")
        V, limit = self.runner.plan.vocab_size, self.runner.max_model_len
        requests = []
        for b, (p, sp) in enumerate(zip(prompts, per)):
            sp.validate()
            p = [int(t) for t in p]
            if not p or min(p) < 0 or max(p) >= V or len(p) >= limit:
                raise ValueError(f"prompt {b}: 1 to {limit - 1} tokens in [0, {V})")
            requests.append(_Request(p, len(p), sp, (b if sp.seed is None else int(sp.seed)) & 0xFFFFFFFFFFFFFFFF, sp.max_tokens or 16384))
        try:
            self._reset()
            self._prompt_steps(requests, rules)
            while not all(q.done for q in requests):
                self._tree_step(requests, draft, rules)
        except BaseException:
            self.runner.recover()
            self.sampler.reset()
            raise
        return [q.generated() for q in requests]

    def _append(self, q: _Request, tokens: Sequence[int]) -> None:
        """Tokens that the model has chosen, up to a stop or the request's length."""
        stops = [s if isinstance(s, (list, tuple)) else [s] for s in q.params.stop_token_ids] + ([] if q.params.ignore_eos else [[t] for t in self.eos_token_ids])
        for t in tokens:
            q.tokens.append(int(t))
            if any(q.generated()[-len(s):] == list(s) for s in stops if s):
                q.tokens.pop()           # (the token that completes a stop stays out)
                q.done = True
            if len(q.generated()) >= q.most or len(q.tokens) >= self.runner.max_model_len:
                q.done = True
            if q.done:
                return

    def _prompt_steps(self, requests: List[_Request], rules: LogitRules) -> None:
        """Every prompt, in the requests' order, and the first token of each.  A step takes as many whole prompts as it has room for and
        a portion of one that is longer than that."""
        at, B = 0, len(requests)
        while at < B:
            counts: List[int] = []
            room = self.max_batched
            while room and at + len(counts) < B:
                q = requests[at + len(counts)]
                counts.append(min(q.prompt - q.cached, self.prefill_chunk, room))
                room -= counts[-1]
                if q.cached + counts[-1] < q.prompt:
                    break
            at += self._prompt_step(requests, at, np.array(counts, np.int32), rules)

    def _prompt_step(self, requests: List[_Request], at: int, counts: np.ndarray, rules: LogitRules) -> int:
        """The next ``counts`` tokens of the prompts from request ``at`` on; returns how many of them have come to their end."""
        B, n = len(requests), len(counts)
        mine = requests[at:at + n]
        ends = [q.cached + int(c) == q.prompt for q, c in zip(mine, counts)]
        ended = [q for q, e in zip(mine, ends) if e]               # (all of them, or all but the last)
        all_new = np.zeros(B, np.int32)
        all_new[at:at + n] = counts
        context = np.array([q.cached for q in mine], np.int32)
        tokens, new, rows = self._send(np.concatenate([q.tokens[q.cached:q.cached + int(c)] for q, c in zip(mine, counts)]), all_new,
                                       (np.cumsum(counts) - 1)[:len(ended)])
        before = self.lengths[0][at:at + n].clone()
        _, positions, request_of, start = self._slots(new, int(counts.sum()))
        logits = self._forward(tokens, positions, request_of - at, start[at:at + n + 1].clone(), rows if ended else None, counts, context, None, before,
                               self.table[at:at + n])
        got = [self.runner.err]
        if ended:
            got.insert(0, self._choose(logits, ended, np.ones(len(ended), int), None, None, np.zeros(len(ended), int), None, (None, None, None), rules))
        got = torch.cat(got).cpu().numpy()
        self.runner.raise_on(int(got[-1]))
        for q, c in zip(mine, counts):
            q.cached += int(c)
        for q, t in zip(ended, got[:-1]):
            self._append(q, [t])
        return len(ended)

    def _tree_step(self, requests: List[_Request], draft: Draft, rules: LogitRules) -> None:
        B, limit = len(requests), self.runner.max_model_len
        drafted, parents, depth, on, counts = [], [], [], [], []
        for q in requests:
            t: List[int] = []
            p: List[int] = []
            if not q.done:
                t, p = draft(list(q.tokens))
                if len(t) != len(p):
                    raise ValueError(f"{len(t)} drafted tokens with {len(p)} parents")
                if any(not 0 <= x < self.runner.plan.vocab_size for x in t):
                    raise ValueError("a drafted token outside the vocabulary")
                t, p = [q.tokens[-1]] + [int(x) for x in t], [-1] + [int(x) for x in p]
            d, o = tree_facts(p)
            # nodes too many, too deep for a path, or behind the last position are dropped (a node's children come after it)
            keep = (np.arange(len(t)) < self.max_nodes) & (d < self.max_depth) & (q.cached + d < limit)
            place = np.cumsum(keep) - 1
            drafted += [x for x, k in zip(t, keep) if k]
            parents += [int(place[x]) if x >= 0 else -1 for x, k in zip(p, keep) if k]
            depth += d[keep].tolist()
            on.append(o[np.ix_(keep, keep)])
            counts.append(int(keep.sum()))
        starts = np.concatenate([[0], np.cumsum(counts)])
        T = int(starts[-1])
        words = max(1, -(-max(counts) // 32))
        row_request = np.repeat(np.arange(B), counts)
        cached = np.array([q.cached for q in requests], np.int32)
        (tokens, par, dep, anc, start, request_of, positions, rows, first, ended) = self._send(
            np.array(drafted), np.array(parents), np.array(depth), np.concatenate([bit_words(o, words) for o in on]), starts, row_request,
            cached[row_request] + np.array(depth), np.arange(T), starts[row_request], np.array([q.done for q in requests]))
        tree = TreeStep(self.lengths[0][:B], start, anc, dep)
        logits = self._forward(tokens, positions, request_of, start, rows, np.array(counts, np.int32), cached, tree)
        targets = self._choose(logits, requests, counts, parents, drafted, depth, on, (first, tokens, anc), rules)
        kernels.tree_accept(self.accepted[:B], self.path[:B], self.next_tokens[:B], tokens, targets.contiguous(), par, start)
        new = torch.where(ended != 0, -1, self.accepted[:B])                 # (a request that has ended gives its pages back)
        slots, _, of, slot_start = self._slots(new.int(), B * self.max_depth)
        kernels.cache_commit(self.commit, slots, of, slot_start, self.path[:B], self.runner.err)
        got = torch.cat([self.accepted[:B], self.next_tokens[:B], self.path[:B].reshape(-1), self.runner.err]).cpu().numpy()
        self.runner.raise_on(int(got[-1]))
        self.steps += 1
        path = got[2 * B:-1].reshape(B, self.max_depth)
        for b, q in enumerate(requests):
            if q.done:
                continue
            n = int(got[b])
            q.cached += n
            self.drafted += counts[b] - 1
            self.confirmed += n - 1
            self._append(q, [drafted[r] for r in path[b][1:n]] + [int(got[B + b])])
