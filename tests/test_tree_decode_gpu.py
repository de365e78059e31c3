"""Generation with drafted trees: the tokens of decoding one by one, whatever is drafted."""
import dataclasses

import numpy as np
import pytest
import torch

import plain_qwen3 as plain
from helpers import PAGE_SIZE, TINY, prompts_for

pytestmark = pytest.mark.gpu


def runner_of(folder, dtype, name, **kw):
    from xinfer_b200 import ModelRunner
    opts = dict(block_size=PAGE_SIZE[name], num_blocks=64, max_num_seqs=4)
    opts.update(kw)
    return ModelRunner(folder, dtype, **opts)


def oracle_draft(texts, rng, wrong=0.3, width=3):
    """Drafts that know the text to come, with guesses beside it and wrong ones in its place."""
    def draft(tokens):
        want = next(t for t in texts if t[:len(tokens)] == list(tokens))
        drafted, parents, node = [], [], 0
        for t in want[len(tokens):len(tokens) + 6]:
            here = [int(x) for x in rng.integers(0, 200, rng.integers(0, width))]
            if rng.random() > wrong:
                here.insert(int(rng.integers(0, len(here) + 1)), t)
            if not here:
                break
            at = len(drafted)
            drafted += here
            parents += [node] * len(here)
            if t not in here:
                node = at + 1                   # go on below a wrong guess
            else:
                node = at + 1 + here.index(t)
        return drafted, parents
    return draft


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_float32_greedy_equals_plain_whatever_is_drafted(name, model_folders):
    from xinfer_b200 import SamplingParams, TreeDecoder
    folder = model_folders(name, torch.float32)
    cfg, w = plain.load_folder(folder)
    prompts = prompts_for(name, [5, 40, 17, 1])
    want = [plain.generate(cfg, w, p, 24) for p in prompts]
    runner = runner_of(folder, "f32", name)
    decoder = TreeDecoder(runner, max_nodes=16, max_depth=5)
    params = SamplingParams(temperature=0.0, max_tokens=24, ignore_eos=True)
    assert decoder.generate(prompts, params) == want
    assert decoder.generate(prompts, params, draft=lambda t: ([], [])) == want
    before = decoder.steps
    draft = oracle_draft([p + g for p, g in zip(prompts, want)], np.random.default_rng(1))
    assert decoder.generate(prompts, params, draft=draft) == want
    assert decoder.steps - before < 20 and decoder.confirmed > 20
    wild = np.random.default_rng(2)
    assert decoder.generate(prompts[:2], params, draft=lambda t: (wild.integers(0, 200, 30).tolist(), [int(x) for x in [wild.integers(0, i + 1) for i in range(30)]])) == want[:2]


def test_float32_samples_equal_plain(model_folders):
    from xinfer_b200 import SamplingParams, TreeDecoder
    folder = model_folders("B", torch.float32)
    cfg, w = plain.load_folder(folder)
    prompts = prompts_for("B", [1, 7, 23, 40])
    params = [SamplingParams(temperature=0.8, max_tokens=15, ignore_eos=True, seed=50 + i, top_k=20 if i == 2 else None) for i in range(4)]
    want = [plain.generate(cfg, w, p, 15, temperature=0.8, seed=50 + i, **({"top_k": 20} if i == 2 else {})) for i, p in enumerate(prompts)]
    decoder = TreeDecoder(runner_of(folder, "f32", "B"), max_nodes=24)
    assert decoder.generate(prompts, params, draft=oracle_draft([p + g for p, g in zip(prompts, want)], np.random.default_rng(3))) == want
    assert decoder.confirmed > 10


@pytest.mark.parametrize("name", ["A", "C"])
def test_bfloat16_follows_the_plain_logits(name, model_folders):
    from xinfer_b200 import SamplingParams, TreeDecoder
    folder = model_folders(name, torch.bfloat16)
    cfg, w = plain.load_folder(folder)
    prompts = prompts_for(name, [3, 30, 61])
    decoder = TreeDecoder(runner_of(folder, "bf16", name), max_nodes=12)
    outs = decoder.generate(prompts, SamplingParams(max_tokens=40, ignore_eos=True))
    for p, o in zip(prompts, outs):
        ref = plain.forward(cfg, w, p + o)
        assert len(o) == 40
        for i, t in enumerate(o):
            row = ref[len(p) + i - 1]
            assert row[t] >= row.max() - 0.15     # the drift that the step function's bfloat16 tests allow


def test_pages_come_back_and_stops_end_a_request(model_folders):
    from xinfer_b200 import SamplingParams, TreeDecoder
    folder = model_folders("A", torch.float32)
    cfg, w = plain.load_folder(folder)
    prompts = prompts_for("A", [5, 11, 17])
    want = [plain.generate(cfg, w, p, 20) for p in prompts]
    stop = want[1][6]
    runner = runner_of(folder, "f32", "A", num_blocks=9)
    decoder = TreeDecoder(runner, max_nodes=8)
    params = [SamplingParams(max_tokens=n, ignore_eos=True, stop_token_ids=[stop] if i == 1 else []) for i, n in enumerate((20, 20, 3))]
    outs = decoder.generate(prompts, params)
    assert outs[0] == want[0] and outs[2] == want[2][:3]
    assert outs[1] == want[1][:want[1].index(stop)]
    # the requests that ended first have given their pages back: the ring's and the others' are all there are
    lengths, (head, count) = decoder.lengths[0][:3].tolist(), decoder.rings[0].tolist()
    assert lengths[1] == lengths[2] == 0 and lengths[0] > 0
    free = [decoder.free_ring[(head + i) % 9].item() for i in range(count)]
    assert sorted(free + decoder.table[0, : -(-lengths[0] // 16)].tolist()) == list(range(9))


def test_rules_change_the_choices_as_written(model_folders):
    """Greedy with a repetition penalty, a bias, penalties and a grammar, against the plain logits changed in 64 bits."""
    from xinfer_b200 import LogitRules, SamplingParams, TreeDecoder
    folder = model_folders("A", torch.float32)
    cfg, w = plain.load_folder(folder)
    V = cfg["vocab_size"] if isinstance(cfg, dict) else TINY["A"][0]["vocab_size"]
    prompts = prompts_for("A", [6, 21])
    even = np.arange(V) % 2 == 0
    rules = LogitRules(1.3, {3: 0.5, 100: -2.0}, lambda t: even if len(t) % 3 == 0 else None)
    params = SamplingParams(max_tokens=16, ignore_eos=True, frequency_penalty=0.3, presence_penalty=0.2)

    def one_by_one(p):
        seq = list(p)
        for _ in range(16):
            x = np.asarray(plain.forward(cfg, w, seq)[-1], dtype=np.float64).copy()
            made = seq[len(p):]
            for t in set(seq):
                x[t] = x[t] / 1.3 if x[t] > 0 else x[t] * 1.3
            for t in set(made):
                x[t] -= 0.3 * made.count(t) + 0.2
            x[3] += 0.5
            x[100] -= 2.0
            if len(seq) % 3 == 0:
                x[~even] = -np.inf
            seq.append(int(x.argmax()))
        return seq[len(p):]

    want = [one_by_one(p) for p in prompts]
    decoder = TreeDecoder(runner_of(folder, "f32", "A"), max_nodes=16)
    draft = oracle_draft([p + g for p, g in zip(prompts, want)], np.random.default_rng(4), wrong=0.2)
    assert decoder.generate(prompts, params, draft=draft, rules=rules) == want
    assert decoder.confirmed > 8
    assert decoder.generate(prompts, params, rules=rules) == want


def test_refusals(model_folders):
    from xinfer_b200 import SamplingParams, StepError, TreeDecoder
    folder = model_folders("A", torch.float32)
    runner = runner_of(folder, "f32", "A", num_blocks=4)
    slot = runner.open_request()
    with pytest.raises(StepError):
        TreeDecoder(runner)
    runner.close_request(slot)
    decoder = TreeDecoder(runner, max_nodes=8)
    p = SamplingParams(max_tokens=4, ignore_eos=True)
    for bad in ([[]], [[-1]], [[10 ** 6]], [[1]] * 5):
        with pytest.raises(ValueError):
            decoder.generate(bad, p)
    for draft in (lambda t: ([1], []), lambda t: ([10 ** 6], [0]), lambda t: ([1, 2], [0, 2])):
        with pytest.raises(ValueError):
            decoder.generate([[1, 2]], p, draft=draft)
    with pytest.raises(StepError, match="no free pages"):
        decoder.generate([[1] * 60, [2] * 30], p)
    assert len(decoder.generate([[1, 2, 3]], p)[0]) == 4      # it goes on after that
    assert decoder.generate([], p) == []
    for nodes, depth in ((0, 1), (2000, 4), (4, 0)):
        with pytest.raises(ValueError):
            TreeDecoder(runner, max_nodes=nodes, max_depth=depth)


def test_rows_instead_of_pages_hold_the_same_numbers():
    """Heads finished into rows of their own are those that go to pages."""
    from xinfer_b200 import kernels as k
    dev = "cuda:0"
    for dtype, d in ((torch.bfloat16, 64), (torch.float32, 48)):
        g = torch.Generator().manual_seed(d)
        T, nh, nkv = 9, 4, 2
        qkv = torch.randn(T, (nh + 2 * nkv) * d, generator=g).to(dtype).to(dev)
        w = torch.randn(d, generator=g).abs().to(dev)
        cos, sin = torch.randn(40, d // 2, generator=g).to(dev), torch.randn(40, d // 2, generator=g).to(dev)
        pos = torch.tensor([0, 3, 5, 5, 7, 11, 13, 30, 39], dtype=torch.int32, device=dev)
        table = torch.arange(9, dtype=torch.int32, device=dev).view(9, 1)
        req = torch.arange(9, dtype=torch.int32, device=dev)
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        q, q2 = (torch.zeros(T, nh, d, dtype=dtype, device=dev) for _ in range(2))
        kc, vc = (torch.zeros(9, nkv, 64, d, dtype=dtype, device=dev) for _ in range(2))
        k.qk_norm_rope_write(q, kc, vc, qkv, w, w, cos, sin, pos, req, table, 1, nh, nkv, d, d, False, 1e-6, True, err)
        kn, vn = (torch.zeros(T, nkv, d, dtype=dtype, device=dev) for _ in range(2))
        k.qk_norm_rope_rows(q2, kn, vn, qkv, w, w, cos, sin, pos, req, nh, nkv, d, d, False, 1e-6, err)
        at = torch.arange(9), slice(None), pos.long().cpu()
        assert torch.equal(q, q2) and torch.equal(kn.cpu(), kc.cpu()[at]) and torch.equal(vn.cpu(), vc.cpu()[at]) and int(err) == 0


def tokens_of_steps(runner):
    """How many tokens each of the model's steps brings, from now on."""
    counts, forward = [], runner.model.forward
    runner.model.forward = lambda ctx, *a: (counts.append(ctx.num_tokens), forward(ctx, *a))[1]
    return counts


def test_prompts_go_through_the_model_in_steps_of_bounded_size(model_folders):
    from xinfer_b200 import SamplingParams, TreeDecoder
    folder = model_folders("A", torch.float32)
    prompts = prompts_for("A", [430 + i for i in range(20)])
    runner = runner_of(folder, "f32", "A", num_blocks=20 * 32, max_num_seqs=20)
    counts = tokens_of_steps(runner)
    decoder = TreeDecoder(runner, max_nodes=8)
    p = SamplingParams(max_tokens=6, ignore_eos=True, temperature=0.7)
    outs = decoder.generate(prompts, p)
    assert max(counts) <= 8192 and sum(n for n in counts if n > 160) == sum(len(x) for x in prompts)
    one = dataclasses.replace(p, seed=7)
    assert decoder.generate(prompts[7:8], one) == outs[7:8]


@pytest.mark.parametrize("batched,chunk", [(7, 100), (64, 5), (64, 64), (1, 1), (13, 13), (90, 41)])
def test_prompts_in_portions_of_any_size(batched, chunk, model_folders):
    from xinfer_b200 import LogitRules, SamplingParams, TreeDecoder
    folder = model_folders("C", torch.float32)
    cfg, w = plain.load_folder(folder)
    prompts = prompts_for("C", [5, 40, 17, 1])
    want = [plain.generate(cfg, w, p, 8) for p in prompts]
    runner = runner_of(folder, "f32", "C")
    counts = tokens_of_steps(runner)
    decoder = TreeDecoder(runner, max_nodes=4, max_num_batched_tokens=batched, prefill_chunk_size=chunk)
    params = SamplingParams(temperature=0.0, max_tokens=8, ignore_eos=True)
    assert decoder.generate(prompts, params, draft=lambda t: ([], [])) == want
    steps = counts[:len(counts) - decoder.steps]
    assert sum(steps) == 63 and max(steps) <= batched
    rules = LogitRules(1.2, {3: 0.5})
    assert decoder.generate(prompts, params, rules=rules) == TreeDecoder(runner, max_nodes=4).generate(prompts, params, rules=rules)
    for limits in (dict(max_num_batched_tokens=0), dict(prefill_chunk_size=0)):
        with pytest.raises(ValueError):
            TreeDecoder(runner, **limits)


def test_the_command_line_draws_alike_with_and_without_drafts(model_folders, capsys):
    """Every prompt has the seed that the engine gives it, so equal prompts draw different tokens, and drafts change none of them."""
    from xinfer_b200 import cli
    folder = model_folders("A", torch.float32)
    args = ["--m", folder, "--dtype", "f32", "--prompts", "5,17,3,5", "--batch", "3", "--max-tokens", "12", "--ignore-eos", "--temperature", "0.9", "--num-blocks", "64",
            "--max-model-len", "128"]

    def texts(*more):
        assert cli.main(args + list(more)) == 0
        return [line.rsplit(": ", 1)[1] for line in capsys.readouterr().out.splitlines() if line.startswith("[seq ")]

    for seed in ([], ["--seed", "5"]):
        plainly = texts(*seed)
        assert len(plainly) == len(set(plainly)) == 3 and texts("--draft-nodes", "8", *seed) == plainly
