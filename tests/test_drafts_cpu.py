"""Trees of drafts on the host: masks, depths, which drafts are kept."""
import pytest

from kernite_b200.drafts import accepted, tree_words


def test_tree_words():
    assert tree_words([-1]) == ([1], [0])
    assert tree_words([-1, 0, 1]) == ([1, 3, 7], [0, 1, 2])
    assert tree_words([-1, -1, 0, 1, 2]) == ([1, 2, 5, 10, 21], [0, 0, 1, 1, 2])
    for bad in ([0], [-1, 1], [-2], [-1, 2, 0]):
        with pytest.raises(ValueError):
            tree_words(bad)


def test_accepted():
    parents = [-1, -1, 0, 1, 1, 4]
    tokens = [7, 8, 1, 2, 3, 4]
    assert accepted(tokens, parents, 9, [0] * 6) == ([], 9)
    assert accepted(tokens, parents, 7, [5, 0, 0, 0, 0, 0]) == ([0], 5)
    assert accepted(tokens, parents, 8, [0, 3, 0, 0, 4, 6]) == ([1, 4, 5], 6)
    assert accepted([7, 7], [-1, -1], 7, [1, 2]) == ([0], 1)  # the first of two alike
