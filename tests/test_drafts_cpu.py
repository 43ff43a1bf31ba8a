"""Trees of drafts on the host: masks, depths, which drafts are kept."""
import pytest

from kernite_b200.drafts import DraftStack, accepted, tree_words


def test_tree_words():
    assert tree_words([-1]) == ([1], [0])
    assert tree_words([-1, 0, 1]) == ([1, 3, 7], [0, 1, 2])
    assert tree_words([-1, -1, 0, 1, 2]) == ([1, 2, 5, 10, 21], [0, 0, 1, 1, 2])
    for bad in ([0], [-1, 1], [-2], [-1, 2, 0]):
        with pytest.raises(ValueError):
            tree_words(bad)


@pytest.mark.parametrize("path", [[0, 1], [1], [0, 3], [2, 4], [0, 2, 3], [0, 0], [-1], [0, 9], [4]], ids=str)
def test_only_paths_of_the_tree_are_kept(path):
    """Drafts 0 and 3 continue the context, 1 and 2 draft 0, 4 draft 3."""
    stack = DraftStack.__new__(DraftStack)  # what keep() looks at before it moves anything
    stack.kept, stack.parents = 7, (-1, 0, 0, -1, 3)
    if path == [0, 1]:
        stack.keep(iter(path))
        assert stack.kept == 9 and stack.parents == ()
    else:
        with pytest.raises(ValueError):
            stack.keep(path)
        assert stack.kept == 7


def test_accepted():
    parents = [-1, -1, 0, 1, 1, 4]
    tokens = [7, 8, 1, 2, 3, 4]
    assert accepted(tokens, parents, 9, [0] * 6) == ([], 9)
    assert accepted(tokens, parents, 7, [5, 0, 0, 0, 0, 0]) == ([0], 5)
    assert accepted(tokens, parents, 8, [0, 3, 0, 0, 4, 6]) == ([1, 4, 5], 6)
    assert accepted([7, 7], [-1, -1], 7, [1, 2]) == ([0], 1)  # the first of two alike
