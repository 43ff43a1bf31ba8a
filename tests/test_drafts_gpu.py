"""The stack over trees of drafted tokens on the GPU against the unsharded f64 reference, one token of a
path at a time. Tolerance: the matvec stack's, 1e-3 of sum_k |w_head x| a logit."""
import dataclasses

import numpy as np
import pytest
import torch

import kernite_b200 as kb
from kernite_b200 import stack as st
from kernite_b200.drafts import DraftStack, accepted

pytestmark = pytest.mark.gpu

CFG = dataclasses.replace(st.CONFIGS["tiny"], attention=True, max_pos=40)


class Reference:
    """The reference's logits and bounds after every path, each prefix computed once."""

    def __init__(self, table):
        self.table, self.known = table, {}

    def __call__(self, path):
        path = tuple(path)
        if path not in self.known:
            cache = {}
            for t in path:
                out = st.reference_logits(CFG, self.table[t], with_bound=True, cache=cache)
            self.known[path] = out
        return self.known[path]


@pytest.fixture(scope="module")
def table():
    return np.random.default_rng(8).standard_normal((CFG.vocab, CFG.hidden)).astype(np.float32)


def vectors(table, tokens):
    return torch.from_numpy(table[list(tokens)]).cuda()


@pytest.mark.parametrize("stream", [False, True])
def test_trees_match_the_reference_path_by_path(kernels, table, stream):
    stack = DraftStack(CFG, kernels, cache=kb.CACHE_F16, page_size=16, stream=torch.cuda.Stream() if stream else None)
    ref = Reference(table)

    def check(context, tokens, parents):
        with torch.cuda.stream(stack.stream):
            got = stack.check(vectors(table, tokens), parents).double().cpu().numpy()
        for i in range(len(tokens)):
            path, at = [], i
            while at >= 0:
                path.insert(0, tokens[at])
                at = parents[at]
            want, bound = ref(context + path)
            assert (np.abs(got[i] - want) <= 1e-3 * bound).all()

    context = [3, 900, 17, 44, 45, 46, 3]
    check([], context, list(range(-1, 6)))  # the prompt
    stack.keep(range(7))
    check(context, [5, 6, 7, 8, 9], [-1, -1, 0, 1, 3])
    stack.keep([1, 3, 4])  # rows are moved
    context += [6, 8, 9]
    check(context, [11], [-1])
    stack.keep([0])
    context += [11]
    check(context, [1, 2, 3, 4, 5, 6, 7, 8], [-1, 0, -1, 2, 2, 1, 5, -1])  # over a page's end
    stack.keep([2, 4])
    context += [3, 5]
    check(context, [12, 13], [-1, 0])
    kernels.device_error()


@pytest.mark.parametrize("cache", [kb.CACHE_F16, kb.CACHE_Q8, kb.CACHE_Q4])
def test_greedy_decoding_with_drafts_equals_one_token_at_a_time(kernels, table, cache):
    """Drafts that are sometimes right: the tokens are those of plain decoding (whose choices are well
    apart: the two runs' logits differ by rounding alone, and each checks that its choice leads by more)."""
    plain, trees = (DraftStack(CFG, kernels, cache=cache, page_size=16) for _ in range(2))
    prompt = [1, 2, 3]

    def choose(logits):
        top = torch.topk(logits, 2, dim=1)
        assert bool((top.values[:, 0] > top.values[:, 1]).all())
        return top.indices[:, 0].tolist()

    want = []
    logits = plain.check(vectors(table, prompt), [-1, 0, 1])
    plain.keep(range(3))
    token = choose(logits)[-1]
    for _ in range(24):
        want.append(token)
        token = choose(plain.check(vectors(table, [token]), [-1]))[0]
        plain.keep([0])

    got = []
    rng = np.random.default_rng(4)
    token = choose(trees.check(vectors(table, prompt), [-1, 0, 1]))[-1]
    trees.keep(range(3))
    steps = 0
    while len(got) < 20:
        at = len(got)
        # the token chosen last, and two branches of guesses after it, one of them right for some way
        right = [want[at + 1 + j] if rng.random() < 0.7 else int(rng.integers(CFG.vocab)) for j in range(3)]
        wrong = [int(rng.integers(CFG.vocab)) for _ in range(2)]
        tokens, parents = [token, wrong[0], right[0], wrong[1], right[1], right[2]], [-1, 0, 0, 1, 2, 4]
        choices = choose(trees.check(vectors(table, tokens), parents))
        path, after = accepted(tokens, parents, token, choices)
        trees.keep(path)
        got += [tokens[i] for i in path]
        token = after
        steps += 1
    kernels.device_error()
    assert got[:20] == want[:20]
    assert steps < 20  # some drafts were kept


@pytest.mark.parametrize("own", [False, True], ids=["the caller's stream", "its own"])
@pytest.mark.parametrize("side", [False, True], ids=["default", "side"])
def test_calls_are_ordered_with_the_callers_stream(kernels, table, own, side):
    """x made late on the caller's stream and overwritten right after the call, logits read there at once,
    calls from changing streams: the bits of a run that waits for the GPU after every call."""
    steps = [([3, 900, 17, 44], [-1, 0, 1, 2], [0, 1, 2, 3]), ([5, 6, 7, 8, 9], [-1, -1, 0, 1, 3], [1, 3, 4]),
             ([11, 12], [-1, 0], [0, 1]), ([1, 2, 3], [-1, -1, 1], [1, 2])]
    xs = [vectors(table, tokens) for tokens, _, _ in steps]
    waits = DraftStack(CFG, kernels, page_size=16)
    want = []
    for x, (_, parents, path) in zip(xs, steps):
        want.append(waits.check(x, parents).clone())
        waits.keep(path)
        torch.cuda.synchronize()
    callers = [torch.cuda.Stream() if side else torch.cuda.default_stream() for _ in range(2)]
    torch.cuda.synchronize()
    with torch.cuda.stream(callers[0]):
        stack = DraftStack(CFG, kernels, page_size=16, stream=torch.cuda.Stream() if own else None)
    got = []
    for i, (x, (_, parents, path)) in enumerate(zip(xs, steps)):
        with torch.cuda.stream(callers[i % 2]):
            late = torch.zeros_like(x)
            torch.cuda._sleep(20_000_000)  # some 10 ms
            late.copy_(x)
            out = stack.check(late, parents)
            late.fill_(float("nan"))
            got.append(out.clone())
            stack.keep(path)
    torch.cuda.synchronize()
    kernels.device_error()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_refusals(kernels):
    for bad in (dict(max_drafts=0), dict(max_drafts=9)):
        with pytest.raises(ValueError):
            DraftStack(CFG, kernels, **bad)
    with pytest.raises(kb.Error):
        DraftStack(CFG, kernels, page_size=48)
    s = DraftStack(CFG, kernels, max_drafts=4)
    x = torch.zeros(5, CFG.hidden, device="cuda")
    with pytest.raises(ValueError):
        s.check(x, [-1, 0, 1, 2, 3])
    with pytest.raises(ValueError):
        s.check(x[:2], [-1])
    with pytest.raises(ValueError):
        s.check(x[:1], [0])
    with pytest.raises(ValueError):
        s.keep([0])
    s.kept = CFG.max_pos
    with pytest.raises(ValueError):
        s.check(x[:1], [-1])
