"""Rotary positions and the paged cache on the GPU (kq_rope_apply, kq_cache_write, kq_cache_read,
kq_cache_move) against the plain restatements in oracle/kvcache.py.

Tolerances. A rotated element is gain (a cos - b sin): cos and sin carry at most 2 f32 steps (2^-23
each), the f32 rounding of the angle's fraction of a turn 2^-25 turns = 2 pi 2^-25 < 2^-22 radians,
the products and the sum 3 roundings of 2^-24; all times gain (|a| + |b|): 2^-20 gain (|a| + |b|)
covers them. Narrowing to f16 or bf16 adds half a step of the result (2^-11, 2^-8 of it at most,
2^-25 for f16's subnormals). Codes: equal to the restatement's when fed the same f32 rows (values);
for rotated keys, which differ by the above, a code may move by one where the quotient is that near a
tie, and a scale by one step where the largest magnitude is that near a scale's bound, so a key is held
to one scale step plus the rotation's error."""
from fractions import Fraction

import numpy as np
import pytest
import torch

import kernite_b200 as kb
from oracle import kvcache as ref

pytestmark = pytest.mark.gpu

TORCH = {kb.TYPE_F32: torch.float32, kb.TYPE_F16: torch.float16, kb.TYPE_BF16: torch.bfloat16}
STEP = {kb.TYPE_F32: 0.0, kb.TYPE_F16: 2.0 ** -11, kb.TYPE_BF16: 2.0 ** -8}
SCALED = dict(freq_scale=0.25, ext_factor=1.0, orig_ctx=4096)


def _act(rng, type, *shape):
    """Random activations on the GPU in `type`, and the f64 values they are."""
    x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda().to(TORCH[type])
    return x, x.double().cpu().numpy()


def _rope_bound(x, rot, halves, gain, out, type):
    pair = np.abs(x).copy()
    if halves:
        s = pair[..., : rot // 2] + pair[..., rot // 2: rot]
        pair[..., : rot // 2] = pair[..., rot // 2: rot] = s
    else:
        s = pair[..., 0:rot:2] + pair[..., 1:rot:2]
        pair[..., 0:rot:2] = pair[..., 1:rot:2] = s
    pair[..., rot:] = 0
    return 2.0 ** -20 * gain * pair + STEP[type] * np.abs(out) * (1 + 2 ** -10) + (2.0 ** -24 if type == kb.TYPE_F16 else 1e-30)


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_F16, kb.TYPE_BF16])
@pytest.mark.parametrize("tokens,heads,dim,rot,halves,scaling", [
    (1, 72, 128, 128, False, {}), (5, 3, 128, 96, True, SCALED), (1, 1, 2, 2, True, {}),
    (33, 4, 64, 64, True, {}), (7, 8, 256, 256, True, {}), (2, 5, 80, 20, False, {}),
    (3, 2, 100, 6, True, dict(freq_scale=0.5)), (130, 2, 192, 64, False, SCALED), (1, 2, 1024, 256, True, {})])
def test_rope(kernels, type, tokens, heads, dim, rot, halves, scaling):
    rng = np.random.default_rng(tokens * dim + rot)
    x, xv = _act(rng, type, tokens, heads, dim)
    pos = rng.integers(-5, 200000, tokens).astype(np.int32)
    pos[0] = 0 if tokens > 1 else 131071
    factors = rng.uniform(1, 8, rot // 2).astype(np.float32) if dim == 128 else None
    rope = kb.Rope(rot, kb.ROPE_HALVES if halves else kb.ROPE_PAIRS, 500000.0, freq_factors=factors, **scaling)
    angles, gain = ref.rope_angles(rot, 500000.0, freq_factors=factors, **scaling)
    want = ref.rope(xv, pos, rot, halves, angles, gain)
    y = torch.full_like(x, float("nan"))
    d = kb.rope_desc(rope, y, x, torch.from_numpy(pos).cuda(), tokens, heads, dim, type=type)
    kernels.rope(d)
    got = y.double().cpu().numpy()
    assert (np.abs(got - want) <= _rope_bound(xv, rot, halves, gain, want, type)).all()
    # in place, the same bits
    z = x.clone()
    kernels.rope(kb.rope_desc(rope, z, z, torch.from_numpy(pos).cuda(), tokens, heads, dim, type=type))
    assert torch.equal(z, y)
    kernels.device_error()


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("type,offset,token,head", [(kb.TYPE_F32, 0, 3 * 68, 68), (kb.TYPE_F32, 1, 211, 67),
                                                    (kb.TYPE_BF16, 3, 207, 69), (kb.TYPE_F16, 8, 3 * 72, 72),
                                                    (kb.TYPE_F32, 0, 64, 5 * 64)])
def test_rope_strides_and_alignment(kernels, halves, type, offset, token, head):
    """Rows off 16 bytes, padded heads, and heads outermost; nothing outside the rows is written."""
    rng = np.random.default_rng(7)
    tokens, heads, dim, rot = 5, 3, 64, 48
    if head == 5 * 64:
        n = heads * head + offset
    else:
        n = tokens * token + offset + 64
    flat, _ = _act(rng, type, n)
    out = torch.full((n,), 7.0, device="cuda", dtype=TORCH[type])
    pos = rng.integers(0, 5000, tokens).astype(np.int32)
    size = flat.element_size()
    rope = kb.Rope(rot, kb.ROPE_HALVES if halves else kb.ROPE_PAIRS)
    kernels.rope(kb.rope_desc(rope, out.data_ptr() + offset * size, flat.data_ptr() + offset * size,
                              torch.from_numpy(pos).cuda(), tokens, heads, dim, type=type, x_token=token,
                              x_head=head, y_token=token, y_head=head))
    view = lambda a: torch.as_strided(a, (tokens, heads, dim), (token, head, 1), offset)
    xv = view(flat).double().cpu().numpy()
    angles, gain = ref.rope_angles(rot, 10000.0)
    want = ref.rope(xv, pos, rot, halves, angles, gain)
    got = view(out).double().cpu().numpy()
    assert (np.abs(got - want) <= _rope_bound(xv, rot, halves, gain, want, type)).all()
    view(out).fill_(7.0)
    assert (out == 7.0).all()


def test_rope_of_the_negative_position_is_the_gradient(kernels):
    """<g, R x> = <R(-pos) g, x>, and R's difference quotient along a direction is R of it."""
    rng = np.random.default_rng(3)
    shape = (9, 4, 128)
    x, xv = _act(rng, kb.TYPE_F32, *shape)
    g, gv = _act(rng, kb.TYPE_F32, *shape)
    pos = torch.from_numpy(rng.integers(0, 30000, 9).astype(np.int32)).cuda()
    rope = kb.Rope(128, kb.ROPE_HALVES, **SCALED)

    def turn(a, p):
        out = torch.empty_like(a)
        kernels.rope(kb.rope_desc(rope, out, a, p, *shape))
        return out.double().cpu().numpy()

    y, back = turn(x, pos), turn(g, -pos)
    # both sums have 9 * 4 * 128 terms with relative errors of 2^-20
    scale = np.abs(gv * y).sum()
    assert abs((gv * y).sum() - (back * xv).sum()) <= 2.0 ** -18 * scale
    step, h = torch.zeros_like(x), 0.5
    step[3, 1, 17] = h
    slope = (turn(x + step, pos) - y) / h
    assert abs((gv * slope).sum() - back[3, 1, 17]) <= 2.0 ** -17 * np.abs(gv[3, 1]).sum() * np.abs(xv[3, 1]).max()


def _cache(layout, seed=0):
    """Two buffers of noise, on the CPU and the GPU, and the cache over the latter."""
    rng = np.random.default_rng(seed)
    k = rng.integers(0, 256, layout.nbytes).astype(np.uint8)
    v = rng.integers(0, 256, layout.nbytes).astype(np.uint8)
    kd, vd = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    assert kb.cache_bytes(layout.kind, layout.n_kv, layout.dim, layout.page, layout.n_pages) == layout.nbytes
    return k, v, kd, vd, kb.KvCache(layout.kind, layout.n_kv, layout.dim, layout.page, layout.n_pages, kd, vd)


WRITES = [  # kind, heads, n_kv, dim, rot, halves, page, tokens
    (ref.Q8, 64, 8, 128, 128, False, 64, 1), (ref.Q4, 8, 2, 64, 64, True, 16, 7), (ref.F16, 4, 4, 128, 64, True, 32, 9),
    (ref.Q4, 16, 2, 128, 96, True, 64, 33), (ref.Q8, 3, 3, 96, 32, False, 16, 5), (ref.Q4, 5, 1, 256, 256, False, 256, 20),
    (ref.Q8, 2, 2, 256, 256, True, 128, 3), (ref.F16, 6, 2, 32, 20, True, 16, 4), (ref.Q4, 6, 2, 160, 20, False, 16, 4),
    (ref.Q8, 32, 32, 64, 64, True, 16, 70)]


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_F16, kb.TYPE_BF16])
@pytest.mark.parametrize("kind,heads,n_kv,dim,rot,halves,page,tokens", WRITES)
def test_cache_write(kernels, type, kind, heads, n_kv, dim, rot, halves, page, tokens):
    rng = np.random.default_rng(dim + tokens)
    n_pages = tokens // page + 3
    layout = ref.Layout(kind, n_kv, dim, page, n_pages)
    k, v, kd, vd, cache = _cache(layout)
    qkv, x = _act(rng, type, tokens, heads + 2 * n_kv, dim)
    pos = rng.integers(0, 100000, tokens).astype(np.int32)
    slots = rng.permutation(n_pages * page)[:tokens].astype(np.int64)
    if tokens > 2:
        slots[1] = -1  # this token is not kept
    q_out = torch.full((tokens, heads, dim), float("nan"), device="cuda", dtype=TORCH[type])
    rope = kb.Rope(rot, kb.ROPE_HALVES if halves else kb.ROPE_PAIRS, 500000.0)
    kernels.cache_write(kb.cache_write_desc(cache, rope, qkv, q_out, torch.from_numpy(pos).cuda(),
                                            torch.from_numpy(slots).cuda(), tokens, heads, type=type))
    kernels.device_error()
    angles, gain = ref.rope_angles(rot, 500000.0)
    turned = ref.rope(x[:, : heads + n_kv], pos, rot, halves, angles, gain)
    bound = _rope_bound(x[:, : heads + n_kv], rot, halves, gain, turned, kb.TYPE_F32)
    got_q = q_out.double().cpu().numpy()
    assert (np.abs(got_q - turned[:, :heads]) <= _rope_bound(x[:, :heads], rot, halves, gain, turned[:, :heads], type)).all()
    k2, v2 = kd.cpu().numpy(), vd.cpu().numpy()
    # values are not rotated: their bytes are the restatement's, and no other byte changed
    for t in range(tokens):
        if slots[t] >= 0:
            layout.put(v, int(slots[t]), x[t, heads + n_kv:])
    assert np.array_equal(v, v2)
    for t in range(tokens):
        if slots[t] < 0:
            continue
        got, want = layout.get(k2, int(slots[t])), turned[t, heads:]
        if kind == ref.F16:
            step = np.abs(want) * 2.0 ** -11 + 2.0 ** -24
        else:
            most = np.abs(want).reshape(n_kv, -1, 32).max(-1)
            step = np.repeat(ref.scale_value(ref.quantise(want, kind)[1]), 32, axis=-1) * (0.5 + 2 ** -10) + \
                np.repeat(most, 32, axis=-1) * 2.0 ** -4 / ref.TOP[kind]  # the next scale up, half a step of it
        assert (np.abs(got - want) <= step + bound[t, heads:]).all()
        layout.put(k, int(slots[t]), np.zeros((n_kv, dim)))
        layout.put(k2, int(slots[t]), np.zeros((n_kv, dim)))
    assert np.array_equal(k, k2)  # nothing else changed


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_BF16])
@pytest.mark.parametrize("dim,rot,pad", [(128, 128, 0), (128, 64, 1), (96, 48, 0), (64, 20, 0), (160, 160, 3)])
def test_queries_in_place(kernels, dim, rot, pad, type, halves):
    """q_out is q, many tokens, the strides' defaults (or q's own, padded): the bits that a separate q_out gets,
    the cache's too, and k and v as they were. Another stride is refused."""
    tokens, heads, n_kv = 203, 6, 2
    layout = ref.Layout(ref.Q8, n_kv, dim, 32, 8)
    wide = (heads + 2 * n_kv) * dim + pad
    qkv, _ = _act(np.random.default_rng(dim), type, tokens, wide)
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda") * 37
    slots = torch.arange(tokens, device="cuda")
    rope = kb.Rope(rot, kb.ROPE_HALVES if halves else kb.ROPE_PAIRS)
    _, _, kd, vd, cache = _cache(layout)
    apart = torch.empty(tokens, heads * dim, device="cuda", dtype=TORCH[type])
    more = dict(type=type, token_stride=wide if pad else 0)
    kernels.cache_write(kb.cache_write_desc(cache, rope, qkv, apart, pos, slots, tokens, heads, **more))
    k, v, before = kd.clone(), vd.clone(), qkv.clone()
    for stride in (0, wide):
        _, _, kd, vd, cache = _cache(layout)
        qkv.copy_(before)
        kernels.cache_write(kb.cache_write_desc(cache, rope, qkv, qkv, pos, slots, tokens, heads, q_out_token=stride,
                                                **more))
        assert torch.equal(qkv[:, : heads * dim], apart)
        assert torch.equal(qkv[:, heads * dim:], before[:, heads * dim:])
        assert torch.equal(kd, k) and torch.equal(vd, v)
    for stride in (heads * dim, wide + 8):
        with pytest.raises(kb.Error) as e:
            kernels.cache_write(kb.cache_write_desc(cache, rope, qkv, qkv, pos, slots, tokens, heads, q_out_token=stride,
                                                    **more))
        assert e.value.code == kb.KQ_E_INVALID
    kernels.device_error()


@pytest.mark.parametrize("halves", [False, True])
def test_rope_in_the_mean_square(kernels, halves):
    """f32 heads. A rounding to f32 errs by 2.53e-8 of a number in the mean square (half a step of 2^-23 to 2^-24 of
    it, uniform). A rotated pair has one in the cosine or sine (one step more is allowed for below, as sincospi is
    not the nearest number), half of one in the one product that is rounded, one in the sum: sqrt(2.5) 2.53e-8 =
    4.0e-8; an angle of at most an eighth of a turn adds 1e-8 (its steps are 2^-27 half turns and less, uniform),
    4.1e-8 with it. A tenth more for sincospi: 4.5e-8. An angle of up to half a turn in f32 adds 3.9e-8: 5.6e-8."""
    rng = np.random.default_rng(12)
    tokens, heads, rot = 300, 8, 128
    x, xv = _act(rng, kb.TYPE_F32, tokens, heads, rot)
    pos = rng.integers(0, 131072, tokens).astype(np.int32)
    turns = [Fraction(t) for t in ref.rope_turns(rot, 500000.0)]
    y = torch.empty_like(x)
    rope = kb.Rope(rot, kb.ROPE_HALVES if halves else kb.ROPE_PAIRS, 500000.0)
    kernels.rope(kb.rope_desc(rope, y, x, torch.from_numpy(pos).cuda(), tokens, heads, rot))
    got, off, all_ = y.double().cpu().numpy(), 0.0, 0.0
    for i, p in enumerate(pos):
        angles = np.array([float(int(p) * t % 1) * 2 * np.pi for t in turns])
        want = ref.rope(xv[i: i + 1], [1], rot, halves, angles, 1.0)[0]
        off += ((got[i] - want) ** 2).sum()
        all_ += (want ** 2).sum()
    assert np.sqrt(off / all_) <= 4.5e-8


@pytest.mark.parametrize("halves", [False, True])
def test_rope_of_quarter_turns(kernels, halves):
    """Turns of whole quarters and next to them, by a table made by hand: signs and exchanged parts, exactly."""
    rope = kb.Rope(2, kb.ROPE_HALVES if halves else kb.ROPE_PAIRS)
    rope.c.turns[0] = 1 << 62
    pos = [0, 1, 2, 3, 4, -1, -2, -3, 2 ** 31 - 1]
    x = torch.tensor([[3.0, 5.0]], device="cuda").repeat(len(pos), 1)
    y = torch.empty_like(x)
    kernels.rope(kb.rope_desc(rope, y, x, torch.tensor(pos, dtype=torch.int32, device="cuda"), len(pos), 1, 2))
    turned = [[3.0, 5.0], [-5.0, 3.0], [-3.0, -5.0], [5.0, -3.0]]
    assert y.tolist() == [turned[p % 4] for p in pos]
    for eighth in range(8):  # the edges between quarters
        rope.c.turns[0] = (eighth << 61) + 1
        angle = 2 * np.pi * ((eighth << 61) + 1) / 2 ** 64
        kernels.rope(kb.rope_desc(rope, y, x, torch.ones(len(pos), dtype=torch.int32, device="cuda"), len(pos), 1, 2))
        want = [3 * np.cos(angle) - 5 * np.sin(angle), 3 * np.sin(angle) + 5 * np.cos(angle)]
        assert np.abs(np.array(y[0].tolist()) - want).max() <= 2.0 ** -20 * 8


@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("halves", [False, True])
def test_rope_at_the_last_positions(kernels, halves, base):
    """Positions up to 2^31, against turns of 50 digits: the same tolerance as at small ones (the table's error
    times the position is 2^-32 turns)."""
    rot, heads = 128, 3
    pos = [2 ** 31 - 1, -2 ** 31, 2 ** 30 + 7, 10 ** 9, 123456789, -(10 ** 8 + 1)]
    x, xv = _act(np.random.default_rng(6), kb.TYPE_F32, len(pos), heads, rot)
    turns = [Fraction(t) for t in ref.rope_turns(rot, base)]
    y = torch.empty_like(x)
    rope = kb.Rope(rot, kb.ROPE_HALVES if halves else kb.ROPE_PAIRS, base)
    kernels.rope(kb.rope_desc(rope, y, x, torch.tensor(pos, dtype=torch.int32, device="cuda"), len(pos), heads, rot))
    got = y.double().cpu().numpy()
    for i, p in enumerate(pos):
        angles = np.array([float(p * t % 1) * 2 * np.pi for t in turns])
        want = ref.rope(xv[i: i + 1], [1], rot, halves, angles, 1.0)
        assert (np.abs(got[i] - want[0]) <= _rope_bound(xv[i], rot, halves, 1.0, want[0], kb.TYPE_F32)).all()


def test_rope_in_place_with_unlike_strides_is_refused(kernels):
    t = torch.zeros(1 << 10, device="cuda")
    p = torch.zeros(2, dtype=torch.int32, device="cuda")
    args = (kb.Rope(64), t, t, p, 2, 2, 64)
    for strides in (dict(x_token=256), dict(y_token=192), dict(x_head=128, x_token=256, y_token=256)):
        with pytest.raises(kb.Error) as e:
            kernels.rope(kb.rope_desc(*args, **strides))
        assert e.value.code == kb.KQ_E_INVALID
    kernels.rope(kb.rope_desc(kb.Rope(64), t, t, p, 1, 2, 64, x_token=256))  # of one token they do not matter
    kernels.device_error()


@pytest.mark.parametrize("kind", [ref.Q8, ref.Q4])
def test_quantised_blocks_at_the_edges(kernels, kind):
    """Bytes of blocks of zeros, tiny, huge, infinite and NaN values, of exact ties and of magnitudes on
    and next to a scale's bound, equal to the restatement's (no rotation: the rows are the inputs)."""
    top = ref.TOP[kind]
    f = np.float32
    rows = [np.zeros(32), np.full(32, 1e-45), np.full(32, 2.0 ** -18 * top), np.linspace(-3e-6, 3e-6, 32),
            np.full(32, 3.4e38), np.linspace(-1e5, 1e5, 32), np.linspace(-65504, 65504, 32)]
    for b in (1, 7, 8, 9, 0x40, 0x41, 0x77, 0x78, 0x90):
        s = float(ref.SCALES[b])
        rows += [np.where(np.arange(32) == 3, s * top, s * (np.arange(32) % top + 0.5)),
                 np.where(np.arange(32) == 30, np.nextafter(f(s * top), f(1e9)), -s * (np.arange(32) % top + 0.5)),
                 np.where(np.arange(32) == 31, np.nextafter(f(s * top), f(0)), s / 3)]
    for odd in (np.inf, -np.inf, np.nan):
        r = np.linspace(-1, 1, 32)
        r[11] = odd
        rows.append(r)
    rows = np.array(rows, dtype=np.float32)
    n = len(rows) + len(rows) % 2
    rows = np.concatenate([rows, np.ones((n - len(rows), 32), np.float32)]).reshape(-1, 1, 64)
    tokens = len(rows)
    layout = ref.Layout(kind, 1, 64, 16, tokens // 16 + 1)
    k, v, kd, vd, cache = _cache(layout)
    x = torch.from_numpy(np.concatenate([rows, rows[::-1]], axis=1).copy()).cuda()
    slots = torch.arange(tokens, device="cuda")
    kernels.cache_write(kb.cache_write_desc(cache, None, x, None, None, slots, tokens, 0))
    for t in range(tokens):
        layout.put(k, t, rows[t])
        layout.put(v, t, rows[tokens - 1 - t])
    assert np.array_equal(kd.cpu().numpy(), k)
    assert np.array_equal(vd.cpu().numpy(), v)
    # and read back: NaN blocks as NaN, the others exactly
    out = torch.empty(tokens, 64, device="cuda")
    kernels.cache_read(kb.cache_read_desc(cache, out, None, slots, tokens))
    want = np.stack([layout.get(k, t)[0] for t in range(tokens)])
    assert np.array_equal(out.double().cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_F16, kb.TYPE_BF16])
@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
@pytest.mark.parametrize("n_kv,dim,page,count,stride", [(8, 128, 64, 1, 0), (2, 64, 16, 77, 0), (1, 256, 32, 40, 259),
                                                        (3, 96, 16, 33, 3 * 96 + 8), (1, 160, 256, 300, 0), (5, 32, 128, 9, 0)])
def test_cache_read(kernels, type, kind, n_kv, dim, page, count, stride):
    """Every value exactly (f16 holds it; bf16 rounds it), negative slots as zeros, strided rows."""
    layout = ref.Layout(kind, n_kv, dim, page, count // page + 2)
    k, v, kd, vd, cache = _cache(layout, seed=dim)
    if kind == ref.F16:  # noise has f16 NaN and infinities; they come back as they are
        pass
    rng = np.random.default_rng(count)
    slots = rng.integers(0, layout.n_pages * page, count).astype(np.int64)
    slots[count // 2] = -3
    wide = stride or n_kv * dim
    k_out = torch.full((count, wide), 9.0, device="cuda", dtype=TORCH[type])
    v_out = torch.full_like(k_out, 9.0)
    sd = torch.from_numpy(slots).cuda()
    kernels.cache_read(kb.cache_read_desc(cache, k_out, v_out, sd, count, type=type, token_stride=stride))
    kernels.device_error()
    for buf, out in ((k, k_out), (v, v_out)):
        want = np.stack([np.zeros((n_kv, dim)) if s < 0 else layout.get(buf, int(s)) for s in slots])
        want = torch.from_numpy(want.astype(np.float32)).to(TORCH[type]).float().numpy().reshape(count, -1)
        got = out.float().cpu().numpy()
        assert np.array_equal(got[:, : n_kv * dim], want, equal_nan=True)
        assert (got[:, n_kv * dim:] == 9.0).all()
    only = torch.empty_like(v_out)
    kernels.cache_read(kb.cache_read_desc(cache, None, only, sd, count, type=type, token_stride=stride))
    assert torch.equal(only[:, : n_kv * dim].nan_to_num(), v_out[:, : n_kv * dim].nan_to_num())


def test_counts_past_31_bits_are_refused(kernels):
    """Before anything is launched, by every call."""
    t = torch.zeros(1 << 14, device="cuda")
    i = torch.zeros(64, dtype=torch.int64, device="cuda")
    cache, many = kb.KvCache(kb.CACHE_Q8, 1, 64, 16, 4, t, t), 1 << 31
    calls = [lambda n: kernels.rope(kb.rope_desc(kb.Rope(64), t, t, i, n, 1, 64)),
             lambda n: kernels.cache_write(kb.cache_write_desc(cache, None, t, None, None, i, n, 0)),
             lambda n: kernels.cache_read(kb.cache_read_desc(cache, t, t, i, n)),
             lambda n: kernels.cache_move(kb.cache_move_desc(cache, i, i, i, n, 1)),
             lambda n: kernels.cache_move(kb.cache_move_desc(cache, i, i, i, 1, n))]
    for call in calls:
        for n in (many, many + 1, (1 << 32) - 1):
            with pytest.raises(kb.Error) as e:
                call(n)
            assert e.value.code == kb.KQ_E_INVALID
    kernels.device_error()


@pytest.mark.parametrize("type", [kb.TYPE_F32, kb.TYPE_F16, kb.TYPE_BF16])
@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
def test_rows_of_negative_slots_have_no_sign(kernels, kind, type):
    layout = ref.Layout(kind, 2, 64, 16, 1)
    _, _, _, _, cache = _cache(layout)
    out = torch.full((3, 2 * 64), -1.0, device="cuda", dtype=TORCH[type])
    slots = torch.tensor([-1, -(1 << 40), -7], device="cuda")
    kernels.cache_read(kb.cache_read_desc(cache, out, None, slots, 3, type=type))
    kernels.device_error()
    assert (out == 0).all() and not torch.signbit(out).any()


@pytest.mark.parametrize("kind,n_kv,dim,page", [(ref.Q8, 2, 128, 16), (ref.Q4, 3, 64, 32), (ref.F16, 1, 256, 16),
                                                (ref.Q4, 1, 128, 64), (ref.Q8, 1, 96, 16)])
def test_cache_move(kernels, kind, n_kv, dim, page):
    """Rows slide over one another inside a group (every source is read first); a group of 64; an empty
    group; negative slots skipped; other rows untouched."""
    layout = ref.Layout(kind, n_kv, dim, page, 300 // page + 1)
    k, v, kd, vd, cache = _cache(layout, seed=5)
    groups = [([3, 5, 6, 9], [2, 3, 4, 5]), ([], []), ([40, 41, 42], [41, 42, 40]),
              (list(range(101, 165)), list(range(100, 164))), ([200, -1, 202], [210, 211, -1])]
    src = np.array(sum((a for a, _ in groups), []), dtype=np.int64)
    dst = np.array(sum((b for _, b in groups), []), dtype=np.int64)
    starts = np.cumsum([0] + [len(a) for a, _ in groups]).astype(np.int32)
    kernels.cache_move(kb.cache_move_desc(cache, torch.from_numpy(src).cuda(), torch.from_numpy(dst).cuda(),
                                          torch.from_numpy(starts).cuda(), len(groups), len(src)))
    kernels.device_error()
    for buf, dev in ((k, kd), (v, vd)):
        want = buf.copy()
        for s, d in zip(src, dst):
            if s < 0 or d < 0:
                continue
            a, b = divmod(int(s), page), divmod(int(d), page)
            for h in range(n_kv):
                ra = (a[0] * n_kv + h) * layout.record
                rb = (b[0] * n_kv + h) * layout.record
                want[rb + layout.row_bytes(b[1])] = buf[ra + layout.row_bytes(a[1])]
                sa, sb = page * layout.row + a[1] * layout.scales, page * layout.row + b[1] * layout.scales
                want[rb + sb: rb + sb + layout.scales] = buf[ra + sa: ra + sa + layout.scales]
        assert np.array_equal(dev.cpu().numpy(), want)


def test_slots_out_of_range_are_recorded_and_skipped(kernels):
    layout = ref.Layout(ref.Q8, 2, 64, 16, 2)
    k, v, kd, vd, cache = _cache(layout)
    x = torch.randn(3, 4, 64, device="cuda")
    slots = torch.tensor([5, 32, 1 << 40], device="cuda")
    out = torch.full((3, 128), 4.0, device="cuda")
    calls = [lambda: kernels.cache_write(kb.cache_write_desc(cache, None, x, None, None, slots[1:], 2, 0)),
             lambda: kernels.cache_read(kb.cache_read_desc(cache, out, None, slots[1:], 2)),
             lambda: kernels.cache_move(kb.cache_move_desc(cache, slots[1:], slots[:2], torch.tensor(
                 [0, 2], dtype=torch.int32, device="cuda"), 1, 2)),
             lambda: kernels.cache_move(kb.cache_move_desc(cache, slots, slots, torch.tensor(
                 [0, 4], dtype=torch.int32, device="cuda"), 1, 3))]
    for call in calls:
        call()
        with pytest.raises(kb.Error) as e:
            kernels.device_error()
        assert e.value.code == kb.KQ_E_DEVICE and "out of its array" in e.value.message
    assert np.array_equal(kd.cpu().numpy(), k) and np.array_equal(vd.cpu().numpy(), v)
    assert (out == 4.0).all()


def test_refusals(kernels):
    t = torch.zeros(1 << 14, device="cuda")
    p = torch.zeros(64, dtype=torch.int32, device="cuda")
    s = torch.zeros(64, dtype=torch.int64, device="cuda")
    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=258), dict(rot_dim=8, layout=2), dict(rot_dim=8, base=1.0),
                dict(rot_dim=8, freq_scale=0.0), dict(rot_dim=8, ext_factor=1.0), dict(rot_dim=8, ext_factor=-1.0),
                dict(rot_dim=8, attn_factor=0.0), dict(rot_dim=8, freq_factors=[1.0] * 3),
                dict(rot_dim=8, freq_factors=[1.0, 0.0, 1.0, 1.0]), dict(rot_dim=8, base=float("nan"))):
        with pytest.raises(kb.Error) as e:
            kb.Rope(**bad)
        assert e.value.code == kb.KQ_E_INVALID
    rope = kb.Rope(64)
    good = dict(rope=rope, y=t, x=t, positions=p, tokens=2, heads=2, head_dim=64)
    for bad in (dict(head_dim=32), dict(head_dim=2048), dict(x=None), dict(positions=None), dict(type=7),
                dict(x=t.data_ptr() + 2), dict(positions=p.data_ptr() + 1)):
        with pytest.raises(kb.Error) as e:
            kernels.rope(kb.rope_desc(**{**good, **bad}))
        assert e.value.code == kb.KQ_E_INVALID
    kernels.rope(kb.rope_desc(**{**good, "tokens": 0, "x": None}))  # nothing to do
    for bad in ((3, 1, 64, 16, 1), (1, 0, 64, 16, 1), (1, 1, 48, 16, 1), (1, 1, 288, 16, 1), (1, 1, 64, 8, 1),
                (1, 1, 64, 48, 1), (1, 1, 64, 512, 1), (1, 1, 64, 16, 0)):
        with pytest.raises(kb.Error):
            kb.cache_bytes(*bad)
        with pytest.raises(kb.Error):
            kernels.cache_read(kb.cache_read_desc(kb.KvCache(*bad, t, t), t, t, s, 1))
    cache = kb.KvCache(kb.CACHE_Q8, 1, 64, 16, 4, t, t)
    off = kb.KvCache(kb.CACHE_Q8, 1, 64, 16, 4, t.data_ptr() + 8, t)
    write = dict(cache=cache, rope=rope, qkv=t, q_out=t, positions=p, slots=s, tokens=1, n_heads=2)
    for bad in (dict(cache=off), dict(cache=kb.KvCache(kb.CACHE_Q8, 1, 64, 16, 4, None, t)), dict(slots=None),
                dict(positions=None), dict(q_out=None), dict(rope=kb.Rope(128)), dict(type=9),
                dict(slots=s.data_ptr() + 4)):
        with pytest.raises(kb.Error) as e:
            kernels.cache_write(kb.cache_write_desc(**{**write, **bad}))
        assert e.value.code == kb.KQ_E_INVALID
    read = dict(cache=cache, k_out=t, v_out=t, slots=s, count=1)
    for bad in (dict(cache=off), dict(slots=None), dict(type=9), dict(token_stride=63), dict(k_out=t.data_ptr() + 2)):
        with pytest.raises(kb.Error) as e:
            kernels.cache_read(kb.cache_read_desc(**{**read, **bad}))
        assert e.value.code == kb.KQ_E_INVALID
    move = dict(cache=cache, src=s, dst=s, starts=p, groups=1, moves=1)
    for bad in (dict(cache=off), dict(src=None), dict(starts=None), dict(dst=s.data_ptr() + 4)):
        with pytest.raises(kb.Error) as e:
            kernels.cache_move(kb.cache_move_desc(**{**move, **bad}))
        assert e.value.code == kb.KQ_E_INVALID
    kernels.device_error()
