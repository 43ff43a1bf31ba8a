"""Attention of drafted tokens on the GPU (kq_attention_tree) against the f64 restatement in
oracle/kvcache.py, over caches whose every unused byte is noise (stale rows, other pages).

Tolerances, as multiples of W = sum_p w_p |v_p|. An error dS of a logit changes a weight by a factor
1 + dS, and the weighted mean by at most 2 max dS W. f32 activations: q enters as two f16 (2^-22 of an
element, and 2^-32 of the row's largest), the products are exact, a sum of head_dim of them in f32
with truncation errs by at most head_dim 2^-23 of sum |q_e k_e| =: R, taken at 2^-18 R for head_dim
up to 256 (32 more steps of 2^-23 in practice); exp2's argument is rounded at 2^-24 of its size, at
most 2^-16 absolutely for the logits here (below 256 in log2 units), exp2 itself 2^-21. Weights enter
as two f16 (2^-22); a sum of n weighted values in f32 by a tile's 16 positions at a time: n / 16 steps
of 2^-23, n <= 8200: 2^-14. So 2 (2^-18 R + 2^-16) W + (2^-14 + 2^-20) W, and 2^-12 (1 + 2^-5 R) W
covers it. 16-bit activations: the weights are rounded to f16 (2^-11, relative, or 2^-31 of the
largest): 2^-10 W more, and half a step of the result (2^-8 or 2^-11 of it)."""
import numpy as np
import pytest
import torch

import kernite_b200 as kb
from oracle import kvcache as ref

pytestmark = pytest.mark.gpu

TORCH = {kb.TYPE_F32: torch.float32, kb.TYPE_F16: torch.float16, kb.TYPE_BF16: torch.bfloat16}
STEP = {kb.TYPE_F32: 2.0 ** -24, kb.TYPE_F16: 2.0 ** -11, kb.TYPE_BF16: 2.0 ** -8}


def tree_masks(rng, drafts):
    """A random tree's masks: each node sees itself and what its parent sees."""
    words = []
    for t in range(drafts):
        up = int(rng.integers(-1, t)) if t else -1
        words.append((words[up] if up >= 0 else 0) | 1 << t)
    return words


class Case:
    """Sequences of given prefixes and drafts over a paged cache, and both sides' attention."""

    def __init__(self, kind, heads, n_kv, dim, page, prefixes, drafts, masks="tree", type=kb.TYPE_F32, seed=0,
                 gain=1.0):
        self.rng = rng = np.random.default_rng(seed)
        self.args = (kind, heads, n_kv, dim, page)
        self.type, self.prefixes, self.drafts = type, prefixes, drafts
        need = [-(-(p + t) // page) for p, t in zip(prefixes, drafts)]
        self.layout = L = ref.Layout(kind, n_kv, dim, page, sum(need) + 2)
        self.k = rng.integers(0, 256, L.nbytes).astype(np.uint8)  # noise: scales and f16 of all kinds, NaN too
        self.v = rng.integers(0, 256, L.nbytes).astype(np.uint8)
        pool = rng.permutation(L.n_pages)
        self.wide = max(max(need), 1) + 1
        self.table = rng.integers(-5, 1 << 30, (len(prefixes), self.wide)).astype(np.int32)  # unused entries: noise
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = pool[at: at + n]
            at += n
        self.keys, self.values, self.masks = [], [], []
        for s, (p, t) in enumerate(zip(prefixes, drafts)):
            kk = rng.standard_normal((p + t, n_kv, dim)).astype(np.float32) * np.float32(gain)
            vv = rng.standard_normal((p + t, n_kv, dim)).astype(np.float32)
            self.fill(s, kk, vv)
            self.masks.append([(2 << i) - 1 for i in range(t)] if masks in ("chain", "none") else
                              tree_masks(rng, t) if masks == "tree" else list(masks[s]))
        self.no_mask = masks == "none"
        total = sum(drafts)
        self.q = torch.from_numpy(rng.standard_normal((total, heads, dim)).astype(np.float32)).cuda().to(TORCH[type])

    def slot(self, s, p):
        return int(self.table[s, p // self.layout.page]) * self.layout.page + p % self.layout.page

    def fill(self, s, kk, vv):
        """Rows of sequence s into the cache, and what the cache then holds kept for the reference."""
        for p in range(len(kk)):
            self.layout.put(self.k, self.slot(s, p), kk[p])
            self.layout.put(self.v, self.slot(s, p), vv[p])
        self.keys.append(np.stack([self.layout.get(self.k, self.slot(s, p)) for p in range(len(kk))])
                         if len(kk) else np.zeros((0, *self.q_shape())))
        self.values.append(np.stack([self.layout.get(self.v, self.slot(s, p)) for p in range(len(vv))])
                           if len(vv) else np.zeros((0, *self.q_shape())))

    def q_shape(self):
        return self.args[2], self.args[3]

    def desc(self, kernels, **more):
        kind, heads, n_kv, dim, page = self.args
        dev = lambda a, dt: torch.from_numpy(np.ascontiguousarray(a, dtype=dt)).cuda()
        self.kd, self.vd = torch.from_numpy(self.k).cuda(), torch.from_numpy(self.v).cuda()
        cache = kb.KvCache(kind, n_kv, dim, page, self.layout.n_pages, self.kd, self.vd)
        starts = np.cumsum([0] + list(self.drafts))
        words = np.array(sum(self.masks, []), dtype=np.uint64).view(np.int64)
        total = int(starts[-1])
        self.out = torch.full((total, heads, dim), float("nan"), device="cuda", dtype=TORCH[self.type])
        fields = dict(cache=cache, out=self.out, q=self.q, n_heads=heads, starts=dev(starts, np.int32),
                      prefix=dev(self.prefixes, np.int32), pages=dev(self.table, np.int32), max_pages=self.wide,
                      n_seq=len(self.drafts), tokens=total, max_drafts=max(max(self.drafts), 1),
                      max_len=max(max(p + t for p, t in zip(self.prefixes, self.drafts)), 1),
                      mask=None if self.no_mask else dev(words, np.int64), type=self.type)
        fields.update(more)
        d = kb.tree_desc(**fields)
        if "workspace" not in more:
            self.space = torch.full((kernels.tree_workspace(d),), 255, dtype=torch.uint8, device="cuda")
            d.workspace, d.workspace_bytes = self.space.data_ptr(), self.space.numel()
        return d

    def run(self, kernels, **more):
        kernels.attention_tree(self.desc(kernels, **more))
        kernels.device_error()
        return self.out.double().cpu().numpy()

    def check(self, got, scale=None):
        dim, start = self.args[3], 0
        qv = self.q.double().cpu().numpy()
        for s, t in enumerate(self.drafts):
            want, weight, reach = ref.tree_attention(qv[start: start + t], self.keys[s], self.values[s],
                                                     self.prefixes[s], self.masks[s], scale or dim ** -0.5)
            bound = 2.0 ** -12 * (1 + 2.0 ** -5 * reach[..., None]) * weight
            if self.type != kb.TYPE_F32:
                bound += 2.0 ** -10 * weight
            bound += STEP[self.type] * np.abs(want) * (1 + 2.0 ** -6) + 1e-30 + (2.0 ** -24 if self.type == kb.TYPE_F16 else 0)
            err = np.abs(got[start: start + t] - want)
            assert (err <= bound).all(), (s, np.nanmax(err - bound), np.isnan(got[start: start + t]).sum())
            start += t


CASES = [  # kind, heads, n_kv, dim, page, prefixes, drafts
    (ref.Q8, 64, 8, 128, 64, [99], [1]),
    (ref.Q8, 8, 8, 128, 64, [0], [1]),                      # the first token: it sees itself
    (ref.Q8, 8, 2, 128, 16, [0, 1, 127, 128, 129], [1, 2, 1, 3, 7]),
    (ref.Q4, 16, 2, 128, 32, [500, 3, 0, 255], [5, 64, 0, 1]),
    (ref.F16, 4, 1, 128, 128, [1000], [16]),
    (ref.Q4, 8, 1, 64, 16, [77, 300], [9, 2]),
    (ref.Q8, 6, 3, 64, 256, [700, 250], [4, 17]),
    (ref.F16, 16, 2, 64, 64, [63, 64, 65], [1, 1, 1]),
    (ref.Q8, 2, 1, 256, 32, [400], [3]),
    (ref.Q4, 16, 1, 256, 64, [129], [2]),
    (ref.F16, 3, 1, 256, 16, [260], [11]),
    (ref.Q8, 5, 1, 96, 64, [200], [6]),
    (ref.Q4, 4, 2, 160, 16, [90], [3]),
    (ref.F16, 7, 7, 32, 16, [130], [2]),
    (ref.Q8, 64, 1, 128, 64, [140], [2]),                   # 64 query heads share one
    (ref.Q8, 8, 1, 128, 64, [2050], [64]),
    (ref.Q4, 8, 8, 128, 256, [513] * 3, [1] * 3),
    (ref.Q8, 2, 1, 64, 16, list(range(0, 80, 2)), [i % 3 for i in range(40)]),  # more sequences than a warp
]


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_BF16])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_tree_attention(kernels, case, type):
    c = Case(*case, type=type, seed=len(str(case)))
    c.check(c.run(kernels))


@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
def test_f16_activations_and_chains(kernels, kind):
    c = Case(kind, 8, 2, 128, 64, [333, 20], [13, 40], masks="chain", type=kb.TYPE_F16)
    got = c.run(kernels)
    c.check(got)
    c.no_mask = True  # no mask is a chain
    assert np.array_equal(c.run(kernels), got)


def test_a_long_context_split_over_the_gpu_twice_the_same_bits(kernels):
    c = Case(ref.Q4, 8, 1, 64, 64, [8100], [2], seed=4)
    a = c.run(kernels)
    c.check(a)
    assert np.array_equal(c.run(kernels), a)
    c.check(c.run(kernels, max_len=1))  # a bound that is too low costs time only


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_BF16])
@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
def test_rows_that_see_nothing_are_zero(kernels, kind, type):
    """Mask words of zero with nothing before the drafts; and nodes that do not see themselves."""
    c = Case(kind, 8, 2, 128, 16, [0, 0, 200], [3, 1, 4],
             masks=[[0, 1, 0b101], [0], [0, 0b10, 0b1, 0b1111]], type=type, seed=8)
    got = c.run(kernels)
    c.check(got)
    assert (got[0] == 0).all() and (got[3] == 0).all()


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
def test_infinities_and_nan_in_masked_places(kernels, kind, dim, type):
    """Drafts 1 and 3 have keys and values that are not finite. Rows that do not see them are exact;
    rows that do are not finite where the values are not."""
    words = [0b00001, 0b00011, 0b00101, 0b01001, 0b10101]
    c = Case(kind, 8, 2, dim, 16, [150], [5], masks=[words], type=type, seed=2)
    for p, odd in ((151, np.nan), (153, np.inf)):
        kk, vv = np.full((2, dim), odd, np.float32), np.ones((2, dim), np.float32)
        vv[:, 40 % dim] = -odd
        c.layout.put(c.k, c.slot(0, p), kk if odd is np.nan else np.zeros((2, dim)))
        c.layout.put(c.v, c.slot(0, p), vv)
    got = c.run(kernels)
    clean = [0, 2, 4]
    qv = c.q.double().cpu().numpy()
    every = ref.tree_attention(qv, c.keys[0], c.values[0], 150, words, dim ** -0.5)
    want, weight, reach = (a[clean] for a in every)
    err = np.abs(got[clean] - want)
    bound = 2.0 ** -12 * (1 + 2.0 ** -5 * reach[..., None]) * weight + (
        0 if type == kb.TYPE_F32 else 2.0 ** -10 * weight + STEP[type] * 1.02 * np.abs(want))
    assert (err <= bound + 1e-30).all()
    assert np.isnan(got[1]).all()  # a NaN key
    block = slice(32, 64)
    if kind == ref.F16:  # one element of the value is infinite
        assert not np.isfinite(got[3][:, 40]).any() and np.isfinite(np.delete(got[3], 40, axis=1)).all()
    else:  # a block with an infinity reads as NaN
        assert np.isnan(got[3][:, block]).all() and np.isfinite(got[3][:, :32]).all()


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
def test_infinities_and_nan_in_many_short_contexts(kernels, kind, dim, type):
    """Four short contexts, each seen by twenty sequences (the same pages), so that a CTA has several items of
    one or two tiles: every row that sees a draft whose value is infinite or NaN says so, and no other."""
    prefixes, drafts = [20, 70, 20, 70], [5, 25, 25, 9]
    c = Case(kind, 16, 8, dim, 16, prefixes, drafts, type=type, seed=17)
    heads, rng = c.q.shape[1], np.random.default_rng(18)
    for s, t in enumerate(drafts):
        nan, inf = (int(p) for p in rng.permutation(t)[:2])
        for draft, odd, e in ((nan, np.nan, 3), (inf, np.inf, 41), (inf, -np.inf, dim - 1)):
            p = prefixes[s] + draft
            vv = c.values[s][p].astype(np.float32)
            vv[:, e] = odd
            c.layout.put(c.v, c.slot(s, p), vv)
            c.values[s][p] = c.layout.get(c.v, c.slot(s, p))
    with np.errstate(invalid="ignore"):
        rows = np.cumsum([0] + drafts)
        each = [ref.tree_attention(c.q[rows[s]: rows[s + 1]].double().cpu().numpy(), c.keys[s], c.values[s],
                                   prefixes[s], c.masks[s], dim ** -0.5) for s in range(4)]
    many = [s for s in range(4) for _ in range(20)]
    c.table = c.table[many]
    c.q = torch.cat([c.q[rows[s]: rows[s + 1]] for s in many])
    c.prefixes, c.drafts, c.masks = [prefixes[s] for s in many], [drafts[s] for s in many], [c.masks[s] for s in many]
    d = c.desc(kernels)
    first = None
    for _ in range(40):
        c.out.fill_(5.0)
        kernels.attention_tree(d)
        got = c.out.clone()
        first = got if first is None else first
        assert torch.equal(got.nan_to_num(nan=1e4), first.nan_to_num(nan=1e4))
    kernels.device_error()
    got, at = first.double().cpu().numpy(), 0
    for s in many:
        want, weight, reach = each[s]
        mine = got[at: at + drafts[s]]
        at += drafts[s]
        fine = np.isfinite(want)
        assert np.array_equal(np.where(fine, 0.0, want), np.where(fine, 0.0, mine), equal_nan=True)
        bound = 2.0 ** -12 * (1 + 2.0 ** -5 * reach[..., None]) * weight + (
            0 if type == kb.TYPE_F32 else 2.0 ** -10 * weight + STEP[type] * 1.02 * np.abs(want))
        assert (np.abs(mine[fine] - want[fine]) <= bound[fine] + 1e-30).all()
    assert at == len(got) and not np.isfinite(got).all()


def test_extreme_magnitudes(kernels):
    """q of 1e-30 and 1e30 (logits near zero, or one position taking all), rows of zeros, values of very
    different sizes, and keys that give large logits."""
    c = Case(ref.Q8, 4, 1, 128, 64, [700], [4], seed=6)
    c.q[0] *= 1e-30
    c.q[1] = 0
    c.check(c.run(kernels))
    c = Case(ref.Q8, 4, 1, 128, 64, [700], [2], seed=7, gain=8.0)
    for p in range(0, 700, 3):
        c.layout.put(c.v, c.slot(0, p), np.full((1, 128), 1e-3 * (p + 1), np.float32))
    c.values = [np.stack([c.layout.get(c.v, c.slot(0, p)) for p in range(702)])]
    c.check(c.run(kernels))


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_BF16])
@pytest.mark.parametrize("drafts", [1, 9])
def test_one_position_takes_all(kernels, drafts, type):
    """Logits of 1e30: a weight of one, the value itself, in both kernels."""
    c = Case(ref.F16, 2, 1, 64, 16, [300], [drafts], type=type, seed=9)
    c.q *= 1e30
    got = c.run(kernels)
    qv = c.q.double().cpu().numpy()
    for t in range(drafts):
        seen = [p for p in range(300 + drafts) if p < 300 or c.masks[0][t] >> (p - 300) & 1]
        for h in range(2):
            best = seen[int((c.keys[0][seen, 0] @ qv[t, h]).argmax())]
            assert np.abs(got[t, h] - c.values[0][best, 0]).max() <= (2.0 ** -20 + STEP[type]) * 5


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_F16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
@pytest.mark.parametrize("drafts", [[1, 0, 1, 2], [5, 0, 12, 3]], ids=["few", "many"])
def test_every_kind_and_head_size(kernels, kind, dim, drafts, type):
    """Single tokens and small trees of ragged sequences, one of them empty, one without a context."""
    c = Case(kind, 8, 2, dim, 32, [333, 40, 0, 129], drafts, seed=31, type=type)
    c.check(c.run(kernels))


@pytest.mark.parametrize("case", [(ref.F16, 64, 8, 128, 64, [700] * 6, [1] * 6), (ref.Q8, 16, 2, 256, 32, [900] * 4, [3] * 4),
                                  (ref.F16, 16, 2, 128, 16, [1500] * 3, [4] * 3), (ref.Q8, 8, 8, 128, 64, [1100] * 5, [1] * 5),
                                  (ref.Q4, 8, 2, 64, 64, [3000], [1])], ids=str)
def test_rings_go_round_many_times(kernels, case):
    """Several tiles and items a CTA, forty calls one after another: the same bits every time, and right."""
    c = Case(*case, seed=21)
    d = c.desc(kernels)
    first = None
    for _ in range(40):
        kernels.attention_tree(d)
        got = c.out.clone()
        first = got if first is None else first
        assert torch.equal(got, first)
    kernels.device_error()
    c.check(first.double().cpu().numpy())


def test_scale_strides_and_another_stream(kernels):
    c = Case(ref.Q8, 8, 2, 64, 32, [321], [6], seed=12)
    wide = 8 * 64 + 64
    q = torch.zeros(6, wide, device="cuda")
    q[:, : 8 * 64] = c.q.view(6, -1)
    out = torch.full((6, wide + 32), 5.0, device="cuda")
    d = c.desc(kernels, q=q, out=out, q_token=wide, out_token=wide + 32, scale=0.3)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    kernels.attention_tree(d, stream=side)
    side.synchronize()
    kernels.device_error()
    c.check(out[:, : 8 * 64].reshape(6, 8, 64).double().cpu().numpy(), scale=0.3)
    assert (out[:, 8 * 64:] == 5.0).all()


def test_in_a_graph_with_lengths_that_change(kernels):
    """A captured call serves other lengths, pages and masks: they are read on the device."""
    c = Case(ref.Q8, 8, 2, 128, 16, [260, 5], [3, 3], seed=13)
    d = c.desc(kernels)
    cache, out, q, starts, prefix, pages, mask, _ = d._keep
    kernels.attention_tree(d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            kernels.attention_tree(d, stream=side)
    c.prefixes = [77, 5]
    c.keys[0], c.values[0] = c.keys[0][:80], c.values[0][:80]
    prefix.copy_(torch.tensor(c.prefixes, dtype=torch.int32))
    out.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    c.check(out.double().cpu().numpy())
    kernels.device_error()


def test_bad_lengths_and_pages_are_recorded_not_followed(kernels):
    def fresh():
        return Case(ref.Q8, 4, 1, 64, 16, [40, 30], [2, 2], seed=3)

    bad = [("starts", [0, 5, 4]), ("starts", [0, 2, 9]), ("starts", [-1, 2, 4]), ("prefix", [-1, 30]),
           ("prefix", [40, 1 << 30])]
    for name, value in bad:
        c = fresh()
        d = c.desc(kernels, **{name: torch.tensor(value, dtype=torch.int32, device="cuda")})
        kernels.attention_tree(d)
        with pytest.raises(kb.Error) as e:
            kernels.device_error()
        assert e.value.code == kb.KQ_E_DEVICE, name
    c = fresh()
    c.table[0, 1] = c.layout.n_pages
    d = c.desc(kernels)
    kernels.attention_tree(d)
    with pytest.raises(kb.Error):
        kernels.device_error()
    c = fresh()
    d = c.desc(kernels, max_drafts=1)  # sequences with more drafts than said
    kernels.attention_tree(d)
    with pytest.raises(kb.Error):
        kernels.device_error()
    c = fresh()
    c.check(c.run(kernels))  # the next call is fine


# ---------------------------------------------------------------- errors on the mean square
#
# The bounds above add up worst cases; these are for the relative error of a whole output in the mean square,
# |got - want| / |want|, of standard normal queries, keys and values. An error of a weight relative to itself,
# independent of the values, becomes the same relative error of the output, as both add up in squares. f32
# activations: logits are sums of 2 dim / 16 <= 32 products of the tensor core, each cut at 2^-23 (2^-24 in the mean)
# of a partial sum near 0.7: 1.4e-6; exp2's argument (below 16) is rounded at 2^-21: 7e-7; exp2 itself
# 2^-22, the weights' two f16 2^-23: in all below 2^-18 (3.8e-6). The output is a sum of n / 16 products at most, each
# cut at 2^-23 of the sum so far: n / 16 2^-23 at most. What leaving out a second f16 costs is a rounding
# of 2^-11 at most of every weight or query element, 2^-12.3 in the mean (f16's steps are 2^-10 to 2^-11 of a number,
# a rounding is 1 / sqrt(12) of a step): 2e-4, which the bound notices up to 20000 positions.
# f16 activations have that rounding of the weights, and the output's, 2^-11 with both: together below 2^-11 + 2^-18.

def mean_square(got, want):
    return np.sqrt(((got - want) ** 2).sum() / (want ** 2).sum())


def one_f16(c, which):
    """c's first sequence in 64 bits, with the weights or the queries (or both) rounded to f16 once."""
    q, out = c.q.double().cpu().numpy()[: c.drafts[0]], []
    dim, group = c.args[3], c.args[1] // c.args[2]
    for t, row in enumerate(q):
        seen = [p for p in range(c.prefixes[0] + c.drafts[0])
                if p < c.prefixes[0] or c.masks[0][t] >> (p - c.prefixes[0]) & 1]
        for h, x in enumerate(row):
            x = x.astype(np.float16).astype(np.float64) if "q" in which else x
            z = c.keys[0][seen, h // group] @ x * dim ** -0.5
            w = 4 * np.exp(z - z.max())
            v = w.astype(np.float16).astype(np.float64) if "p" in which else w
            out.append(v @ c.values[0][seen, h // group] / w.sum())
    return np.array(out).reshape(q.shape)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
@pytest.mark.parametrize("length,heads,drafts", [(99, 8, 1), (700, 2, 3), (260, 6, 3), (1500, 4, 11)])
def test_f32_activations_have_more_than_16_bits(kernels, kind, dim, length, heads, drafts):
    c = Case(kind, heads, 1, dim, 64, [length], [drafts], masks="chain", seed=41)
    want = ref.tree_attention(c.q.double().cpu().numpy(), c.keys[0], c.values[0], length, c.masks[0], dim ** -0.5)[0]
    bound = 2.0 ** -18 + (length + drafts) / 16 * 2.0 ** -23
    for which in ("p", "q", "pq"):
        assert mean_square(one_f16(c, which), want) > 2 * bound, which
    assert mean_square(c.run(kernels), want) <= bound


@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
@pytest.mark.parametrize("heads,drafts", [(8, 1), (4, 11)])
def test_f16_activations_in_the_mean_square(kernels, kind, heads, drafts):
    c = Case(kind, heads, 1, 128, 64, [900], [drafts], masks="chain", type=kb.TYPE_F16, seed=42)
    want = ref.tree_attention(c.q.double().cpu().numpy(), c.keys[0], c.values[0], 900, c.masks[0], 128 ** -0.5)[0]
    assert mean_square(c.run(kernels), want) <= 2.0 ** -11 + 2.0 ** -18 + 911 / 16 * 2.0 ** -23


def copied(c, n):
    """c's only sequence n times over the same pages, with the same queries: so many items that a CTA does
    whole ones. The expected rows, and the reference's other results, of one."""
    t = c.drafts[0]
    each = ref.tree_attention(c.q.double().cpu().numpy(), c.keys[0], c.values[0], c.prefixes[0], c.masks[0],
                              c.args[3] ** -0.5)
    c.table, c.q = np.repeat(c.table, n, axis=0), c.q.repeat(n, 1, 1)
    c.prefixes, c.drafts, c.masks = c.prefixes * n, [t] * n, c.masks * n
    return each


@pytest.mark.parametrize("heads,drafts", [(2, 3), (2, 9)])
def test_a_long_context_by_one_cta(kernels, heads, drafts):
    """Some 8100 positions added up by one CTA (the warp-MMA kernel's are 296), in the mean square and at the worst."""
    c = Case(ref.Q8, heads, 1, 64, 64, [8100], [drafts], masks="chain", seed=43)
    n = 320 if drafts == 3 else 160
    want, weight, reach = copied(c, n)
    got = c.run(kernels).reshape(n, drafts, heads, 64)
    bound = 2.0 ** -18 + 8111 / 16 * 2.0 ** -23
    assert all(mean_square(g, want) <= bound for g in got)
    assert (np.abs(got - want) <= 2.0 ** -12 * (1 + 2.0 ** -5 * reach[..., None]) * weight).all()


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
@pytest.mark.parametrize("heads,drafts", [(2, 2), (3, 5)], ids=["few", "many"])
def test_logits_that_rise_along_the_context(kernels, kind, dim, type, heads, drafts):
    """Three stretches of a context, the logits of each some 15 log2 units above those before, and values the
    smaller for it (2^10, 2^-5, 2^-17: the smallest a quantised cache holds), so that the first two are a tenth of the
    output each: a maximum is replaced (the kernels rescale what they have by factors near 2^-15) twice in an
    item, and the rescaled part shows."""
    stretches = [(0, 212), (212, 333), (333, 700)]
    c = Case(kind, heads, 1, dim, 32, [700], [drafts], masks="chain", type=type, seed=44)
    c.q[..., 0] = dim ** 0.5
    rng = np.random.default_rng(45)
    kk, vv = (rng.standard_normal((700 + drafts, 1, dim)).astype(np.float32) for _ in range(2))
    for i, (a, b) in enumerate(stretches):
        b = len(kk) if i == 2 else b
        kk[a:b, :, 0] = 15 * np.log(2) * i
        vv[a:b] = vv[a:b] * 2.0 ** (10 - 15 * i) if i < 2 else rng.integers(-1, 2, vv[a:b].shape) * 2.0 ** -17
    c.keys, c.values = [], []
    c.fill(0, kk, vv)
    n = 320 if drafts * heads <= 8 else 160
    want, weight, reach = copied(c, n)
    got = c.run(kernels).reshape(n, drafts, heads, dim)
    bound = 2.0 ** -12 * (1 + 2.0 ** -5 * reach[..., None]) * weight + STEP[type] * np.abs(want) * (1 + 2.0 ** -6)
    if type != kb.TYPE_F32:
        bound += 2.0 ** -10 * weight
    assert (np.abs(got - want) <= bound + 1e-30).all()


@pytest.mark.parametrize("drafts", [1, 9])
def test_a_workspace_serves_any_length(kernels, drafts):
    """Its size does not depend on max_len, n_seq or tokens, and one for many drafts is enough for one."""
    c = Case(ref.Q8, 8, 1, 64, 16, [700, 5], [drafts, 1], seed=5)
    d = c.desc(kernels, max_len=1)
    for fields in (dict(max_len=1 << 20), dict(n_seq=1), dict(n_seq=1 << 16), dict(tokens=1 << 16), dict(max_len=702)):
        for name, value in fields.items():
            was = getattr(d, name)
            setattr(d, name, value)
            assert kernels.tree_workspace(d) == d.workspace_bytes
            setattr(d, name, was)
    d.max_len = 709
    kernels.attention_tree(d)
    kernels.device_error()
    c.check(c.out.double().cpu().numpy())
    for n in range(1, drafts):
        d.max_drafts = n
        assert kernels.tree_workspace(d) <= d.workspace_bytes


def test_scales_past_the_range_are_refused(kernels):
    """Up to 2^127 they are taken: queries of zeros then still give the mean of the values."""
    c = Case(ref.Q8, 4, 2, 64, 16, [40], [1], seed=3)
    c.q.zero_()
    for scale in (3e38, float("inf"), float("-inf"), float("nan")):
        with pytest.raises(kb.Error) as e:
            kernels.attention_tree(c.desc(kernels, scale=scale, workspace=1 << 40, workspace_bytes=1 << 40))
        assert e.value.code == kb.KQ_E_INVALID
    c.check(c.run(kernels, scale=2.0 ** 127))


def test_refusals(kernels):
    c = Case(ref.Q8, 4, 2, 64, 16, [40], [2], seed=3)
    good = c.desc(kernels)
    kernels.attention_tree(good)

    def refused(**fields):
        d = c.desc(kernels)
        for k, v in fields.items():
            setattr(d, k, v)
        with pytest.raises(kb.Error) as e:
            kernels.attention_tree(d)
        assert e.value.code == kb.KQ_E_INVALID, fields

    for fields in (dict(q=0), dict(out=0), dict(starts=0), dict(prefix=0), dict(pages=0), dict(workspace=0),
                   dict(workspace_bytes=16), dict(type=3), dict(n_heads=3), dict(n_heads=0), dict(n_heads=2 * 65),
                   dict(max_drafts=0), dict(max_drafts=65), dict(max_len=0), dict(max_pages=0), dict(max_pages=1 << 30),
                   dict(q=good.q + 4), dict(out=good.out + 4), dict(q_token=4 * 64 - 4), dict(out_token=4 * 64 + 2),
                   dict(mask=good.mask + 4), dict(pages=good.pages + 2), dict(scale=float("nan")), dict(scale=-1.0),
                   dict(workspace=good.workspace + 8), dict(n_seq=1 << 31)):
        refused(**fields)
    d = c.desc(kernels)
    d.tokens = 0
    kernels.attention_tree(d)  # nothing to do
    d.n_heads = 3
    with pytest.raises(kb.Error):
        kernels.tree_workspace(d)
    kernels.device_error()
