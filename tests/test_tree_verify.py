"""examples/tree_verify.py: what trees, forks and compaction decode is what one pass over
the whole text would.

Two passes differ by bf16 roundings, which move a few of an activation row's 4-bit
codes by one: some hundredths of a logit's standard deviation. A token chosen with a
wrong row, mask or position stands about three under the largest of 512 logits. Half
of one is the line between them.
"""

import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


def test_drafts_without_a_device():
    import tree_verify
    s = tree_verify.Sequence([1, 2, 3, 1, 4, 1])
    tokens, parents = s.draft(6, 2)
    assert tokens == [1, 4, 2, 1, 3, 4] and parents == [-1, 0, 0, 1, 2, 3]
    assert s.draft(1, 2) == ([1], [-1])


@pytest.mark.gpu
@pytest.mark.parametrize("size,width", [(1, 1), (16, 2), (40, 3)])
def test_tokens_are_those_of_one_pass(cuda, size, width):
    import tree_verify
    prompt = [i % 5 + 7 for i in range(33)]
    tokens, passes = tree_verify.generate(60, size, width, prompt)
    assert passes == 61 if size == 1 else passes <= 61
    assert tokens[0][:33] == tokens[1][:33] == prompt and tokens[0][33] != tokens[1][33]
    for t, own in zip(tokens, (32, 33)):  # the fork's first token was not the model's choice
        assert len(t) == 94
        assert float(tree_verify.shortfall(t)[own:].max()) < 0.5
