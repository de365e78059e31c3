"""The host's side of drafted trees: drafts from the text, tree facts, words of bits, the command line."""
import numpy as np
import pytest

from xinfer_b200.engine.tree_decode import bit_words, lookup_draft, tree_facts


def test_drafts_follow_earlier_occurrences_latest_first():
    #            0  1  2  3  4  5  6  7  8  9
    text = [1, 2, 3, 7, 1, 2, 3, 8, 1, 2, 3]
    drafted, parents = lookup_draft(10, longest=2)(text)
    assert drafted == [8, 1, 7, 1] and parents == [0, 1, 0, 3]
    drafted, parents = lookup_draft(10, longest=3)(text)
    assert drafted == [8, 1, 2, 7, 1, 2] and parents == [0, 1, 2, 0, 4, 5]
    assert lookup_draft(2)(text) == ([8, 1], [0, 1])
    assert lookup_draft(5)([4]) == ([], []) and lookup_draft(5)([4, 5]) == ([], [])
    assert lookup_draft(0)(text) == ([], [])
    # fewer tokens match where more do not
    assert lookup_draft(5, longest=2)([9, 5, 6, 4, 5]) == ([6, 4], [0, 1])


def test_drafts_that_begin_alike_share_nodes():
    drafted, parents = lookup_draft(20, longest=3, match=1)([5, 1, 2, 3, 5, 1, 2, 4, 5])
    assert drafted == [1, 2, 4, 3] and parents == [0, 1, 2, 2]


def test_tree_facts():
    depth, on = tree_facts([-1, 0, 0, 1, 3, 2])
    assert depth.tolist() == [0, 1, 1, 2, 3, 2]
    assert [np.nonzero(r)[0].tolist() for r in on] == [[0], [0, 1], [0, 2], [0, 1, 3], [0, 1, 3, 4], [0, 2, 5]]
    assert tree_facts([])[0].size == 0
    for bad in ([0], [-1, 1], [-1, -1], [-1, 0, 3]):
        with pytest.raises(ValueError):
            tree_facts(bad)


@pytest.mark.parametrize("n,m,words", [(3, 3, 1), (2, 33, 2), (1, 64, 3), (4, 32, 1)])
def test_bit_words(n, m, words):
    on = np.random.default_rng(m).random((n, m)) < 0.5
    got = bit_words(on, words)
    assert got.shape == (n, words) and got.dtype == np.int32
    for i in range(n):
        for j in range(words * 32):
            assert bool(got[i, j // 32] >> (j % 32) & 1) == (j < m and bool(on[i, j]))


def test_the_command_line_knows_the_options():
    from xinfer_b200.cli import build_parser
    args = build_parser().parse_args(["--m", "x", "--draft-nodes", "8", "--repetition-penalty", "1.1"])
    assert args.draft_nodes == 8 and args.repetition_penalty == 1.1


@pytest.mark.parametrize("rules", [dict(repetition_penalty=0.0), dict(repetition_penalty=-1.5), dict(repetition_penalty=float("nan")), dict(repetition_penalty=float("inf")),
                                   dict(repetition_penalty=1e-45), dict(bias={3: float("nan")})])
def test_rules_that_make_no_sense_are_refused(rules):
    from xinfer_b200.engine.tree_decode import LogitRules
    with pytest.raises(ValueError):
        LogitRules(**rules).validate()
    LogitRules(0.5, {3: -float("inf"), 10 ** 6: 2.0}).validate()


@pytest.mark.parametrize("args", [["--repetition-penalty", "1.1"], ["--repetition-penalty", "0"], ["--draft-nodes", "0"], ["--draft-nodes", "-3"], ["--draft-nodes", "2000"],
                                  ["--draft-nodes", "8", "--repetition-penalty", "0"], ["--draft-nodes", "8", "--repetition-penalty", "-2"]])
def test_the_command_line_refuses_options_before_it_loads_a_model(args):
    from xinfer_b200.cli import main
    with pytest.raises(SystemExit, match="--repetition-penalty|--draft-nodes"):
        main(["--m", "/nowhere", "--prompts", "1,2", *args])
