"""Which rows of a pass predict the scored tokens (`LeanGemma4.token_logprobs`), on the host."""
from types import SimpleNamespace

import pytest

from morj_b200.lean_core import LeanGemma4

# a tree of a shared node (offsets 0..3) and two branches (4..5 and 6..8); sequence 1 ends inside its last node
SLOTS = {0: [0, 1, 2, 3], 1: [4, 5], 2: [6, 7, 8]}
TREE = SimpleNamespace(paths=[[0, 1], [0, 2]], slots=SLOTS.__getitem__, seqs=[[9] * 6, [9] * 6])
REQ = SimpleNamespace(tree=TREE)


def rows(steps, seqs=(0, 1), scored=(None, None)):
    scored = list(scored)
    got = LeanGemma4._scored_rows(None, REQ, list(seqs), dict(steps=[dict(own=own) for own in steps]), scored)
    return got, scored


def test_every_token_after_the_first_is_predicted_by_the_row_before_it():
    got, scored = rows([[0, 1, 2, 3, 4, 5], [6, 7, 8]])
    assert scored == [1, 1]
    assert got == [(0, r) for r in range(5)] + [(0, 0), (0, 1), (0, 2), (0, 3), (1, 0)]


def test_a_given_start_and_the_order_of_the_sequences_are_kept():
    got, scored = rows([[0, 1, 2, 3, 4, 5, 6, 7, 8]], seqs=(1, 0), scored=(5, 4))
    assert scored == [5, 4] and got == [(0, 6), (0, 3), (0, 4)]


def test_without_a_start_scoring_begins_behind_the_rows_of_earlier_passes():
    got, scored = rows([[4, 5, 6, 7, 8]])
    assert scored == [5, 5] and got == [(0, 0), (0, 2)]


@pytest.mark.parametrize('steps,scored,match', [
    ([[4, 5, 6, 7, 8]], (4, None), 'token 4 of sequence 0 is predicted by a row that an earlier pass computed'),
    ([[0, 1, 2, 3, 4, 5, 6, 7, 8]], (0, None), 'tokens 1..5 to score, not from 0'),
    ([[0, 1, 2, 3, 4, 5, 6, 7, 8]], (7, None), 'tokens 1..5 to score, not from 7'),
    ([[5, 8]], (None, None), 'no token to score'),
    ([[0, 1, 2, 3, 4, 5, 6, 7, 8]], (6, 6), 'no token to score'),
])
def test_refusals(steps, scored, match):
    with pytest.raises(ValueError, match=match):
        rows(steps, scored=scored)


def test_with_images_scoring_begins_behind_the_last_block():
    plan = dict(steps=[dict(own=[0, 1, 2, 3, 4, 5, 6, 7, 8])])
    for given, want in [((None, None), [3, 3]), ((3, 5), [3, 5]), ((5, None), [5, 3])]:
        scored = list(given)
        got = LeanGemma4._scored_rows(None, REQ, [0, 1], plan, scored, earliest=3)
        assert scored == want
        assert got == [(0, o) for path, first in zip(([0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 6, 7]), want)
                       for o in path[first - 1:5]]
    for start in (1, 2):
        with pytest.raises(ValueError, match=f'from 3 on, not from {start}: up to there it holds images'):
            LeanGemma4._scored_rows(None, REQ, [0], plan, [start], earliest=3)
    # sequences that end with their images have no token to score
    with pytest.raises(ValueError, match='no token to score'):
        LeanGemma4._scored_rows(None, REQ, [0, 1], plan, [None, None], earliest=7)
