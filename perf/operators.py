"""The operators around a quantised key/value cache, as cases to measure: rotary positions, the
cache's write and read-back, and attention of drafted tokens (a tree, or one token) over it.

`run` computes a case in plain torch operations (32 bits), or, where `own` is true, through the
library's entry points. The cache's format, which both read:

* a page holds `page` positions; K and V are two arrays [pages][kv heads][record];
* a record is the page's codes (rows of `row` bytes, one per position) and then its scale bytes
  (one per 32 elements, [position][head_dim / 32]); an f16 cache has no scales;
* 16-byte units of the codes are permuted inside lines of 128 bytes: logical unit l of position p
  lies at l ^ swizzle(p);
* a scale byte b is the f16 whose bits are b << 7; an 8-bit code is c + 128, a 4-bit one c + 8,
  eight of those in a 32-bit word at nibbles 0,4,1,5,2,6,3,7; the value is c * scale, exact in f16.
"""
import math

import torch

own = False

BITS = {"f16": 16, "q8": 8, "q4": 4}
TOP = {"q8": 127, "q4": 7}  # the largest code
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- the cases

def _rope(name, tokens, heads, dim, rot, layout, act, context, base=10000.0, scale=1.0, ext=0.0):
    return {"op": "rope", "name": name, "tokens": tokens, "heads": heads, "dim": dim, "rot": rot,
            "layout": layout, "act": act, "context": context, "base": base, "scale": scale, "ext": ext}


def _write(name, kind, tokens, heads, kv, dim, page, act, context, layout="pairs", rot=None,
           base=10000.0):
    return {"op": "write", "name": name, "kind": kind, "tokens": tokens, "heads": heads, "kv": kv,
            "dim": dim, "rot": rot or dim, "page": page, "act": act, "context": context,
            "layout": layout, "base": base, "scale": 1.0, "ext": 0.0}


def _read(name, kind, tokens, kv, dim, page, act):
    return {"op": "read", "name": name, "kind": kind, "tokens": tokens, "kv": kv, "dim": dim,
            "page": page, "act": act}


def _tree(name, kind, seqs, drafts, least, most, heads, kv, dim, page, act, chain=False):
    return {"op": "tree", "name": name, "kind": kind, "seqs": seqs, "drafts": drafts, "least": least,
            "most": most, "heads": heads, "kv": kv, "dim": dim, "page": page, "act": act, "chain": chain}


def listed():
    return [
        # one decode step of the 70B stack's shape: its 64 query and 8 key heads rotated (latency)
        _rope("rope_step", 1, 72, 128, 128, "pairs", "f32", 4096),
        # a prompt's heads, halves layout, a quarter of the head left as it is, scaled by parts
        _rope("rope_prompt", 4001, 40, 128, 96, "halves", "bf16", 131072, 500000.0, 0.25, 1.0),
        # one decode step writes its token (and reads it back)
        _write("write_step", "q8", 1, 64, 8, 128, 64, "f32", 4096),
        # a batch of drafted tokens, 4-bit cache
        _write("write_drafts_q4", "q4", 61, 64, 8, 128, 64, "f32", 131072, base=500000.0),
        # a prompt of the 7B stack's shape (as many key as query heads)
        _write("write_prompt", "q8", 6144, 32, 32, 128, 64, "f32", 8192, layout="halves"),
        # a short context read back into 16 bits, small pages
        _read("read_short_q4", "q4", 1001, 8, 128, 16, "f32"),
        # a long context read back for a kernel that wants 16-bit values
        _read("read_long", "q8", 65536, 8, 128, 64, "f16"),
        # the first tokens of a chat, one sequence, one token (latency)
        _tree("decode_short", "q8", 1, 1, 99, 99, 64, 8, 128, 64, "f32"),
        # a serving batch, one token a sequence, ragged contexts
        _tree("decode_batch", "q8", 32, 1, 500, 7900, 64, 8, 128, 64, "f32"),
        # one very long context in 4 bits
        _tree("decode_long_q4", "q4", 1, 1, 131001, 131001, 64, 8, 128, 64, "f32"),
        # a tree of drafts over one conversation
        _tree("tree_one", "q8", 1, 25, 8191, 8191, 64, 8, 128, 64, "f32"),
        # trees of 64 drafts over a few long conversations, 16-bit activations
        _tree("tree_batch", "q8", 4, 64, 6000, 16000, 64, 8, 128, 64, "bf16"),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["rope", "write", "read", "tree", "tree", "tree"])
    act = rng.choice(["f32", "f32", "bf16", "f16"])
    kind = rng.choice(["q8", "q8", "q4", "f16"])
    dim = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    layout = rng.choice(["pairs", "halves"])
    if op == "rope":
        heads = rng.choice([10, 40, 64, 72])
        scale, ext = rng.choice([(1.0, 0.0), (0.25, 0.0), (0.125, 1.0)])
        c = _rope(None, _log(rng, 1, 6000 * 128 // dim), heads, dim, rng.choice([dim, dim, dim // 2]), layout, act,
                  _log(rng, 100, 131072), rng.choice([10000.0, 500000.0]), scale, ext)
    elif op == "write":
        kv = rng.choice([1, 2, 8, 32])
        heads = kv * rng.choice([1, 4, 8]) if kv < 32 else 32
        c = _write(None, kind, min(_log(rng, 1, 6000), 6000 * 128 // dim), heads, kv, dim, page, act,
                   _log(rng, 100, 131072), layout, rng.choice([dim, dim // 2]),
                   rng.choice([10000.0, 500000.0]))
    elif op == "read":
        kv = rng.choice([1, 2, 8, 32])
        c = _read(None, kind, min(_log(rng, 1, 50000), 50000 * 8 * 128 // (kv * dim)), kv, dim, page, act)
    else:
        kv = rng.choice([1, 2, 8, 8, 32])
        heads = kv * rng.choice([1, 4, 8]) if kv < 32 else 32
        seqs = _log(rng, 1, 64)
        drafts = rng.choice([1, 1, _log(rng, 2, 64)])
        # positions of all sequences: bounded by the cache's bytes and by the products
        room = min(2 ** 31 // (BITS[kind] * kv * dim * seqs), 2 ** 34 // (heads * dim * drafts * seqs), 131072)
        most = _log(rng, min(100, room), room)
        c = _tree(None, kind, seqs, drafts, most // 3, most, heads, kv, dim, page, act, rng.random() < 0.2)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _swizzle(pos, row):
    """What position `pos`'s unit indexes are XORed with, in rows of `row` bytes."""
    if row >= 128:
        return pos & 7
    return ((pos >> 1) & 3) << 1 if row == 64 else ((pos >> 2) & 1) << 2


def _order(page, row):
    """order[l]: where logical 16-byte unit l of a page's codes lies."""
    unit = torch.arange(page * row // 16, device="cuda")
    return unit ^ _swizzle(unit // (row // 16), row)


def _quantise(x, kind):
    """(codes, scale bytes) of the 32-element blocks of x's last axis."""
    x = x.unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    want = most / TOP[kind]
    byte = torch.where(want >= 2.0 ** -14, ((want.view(torch.int32) + 0xFFFFF) >> 20) - 896,
                       torch.ceil(want * 2.0 ** 17).int())
    scale = _scale(byte)
    code = torch.round(x / torch.where(scale > 0, scale, 1.0)).clamp(-TOP[kind], TOP[kind])
    return code, byte


def _scale(byte):
    return (byte.to(torch.int16) << 7).view(torch.float16).float()


def _pack(values, kind, page):
    """Values [pages, kv, page, dim] as the records the cache holds, [pages, kv, record] bytes."""
    n, kv, _, dim = values.shape
    if kind == "f16":
        codes = values.half().view(torch.uint8)
        row, scales = 2 * dim, None
    else:
        code, byte = _quantise(values, kind)
        code, scales = code.flatten(-2), byte.to(torch.uint8).reshape(n, kv, -1)
        if kind == "q8":
            row, codes = dim, (code + 128).to(torch.uint8)
        else:
            u = (code + 8).to(torch.uint8).unflatten(-1, (-1, 8))
            lo, hi = u[..., [0, 4, 1, 5]], u[..., [2, 6, 3, 7]]
            row, codes = dim // 2, (lo | (hi << 4)).flatten(-2)
    units = codes.reshape(n, kv, -1, 16)
    put = torch.empty_like(units)
    put[:, :, _order(page, row)] = units
    put = put.reshape(n, kv, -1)
    return put if scales is None else torch.cat([put, scales], -1)


def _cache(g, kind, n_pages, kv, page, dim, key):
    """A pool of pages of normally distributed rows; keys have a few channels that stand out."""
    out = torch.empty(n_pages, kv, page * dim * BITS[kind] // 8 + (0 if kind == "f16" else page * dim // 32),
                      dtype=torch.uint8, device="cuda")
    gain = torch.ones(kv, 1, dim, device="cuda")
    if key:
        gain[..., ::17] = 4.0
    step = max(1, 2 ** 26 // (kv * page * dim))
    for a in range(0, n_pages, step):
        n = min(step, n_pages - a)
        out[a:a + n] = _pack(_randn(g, n, kv, page, dim) * gain, kind, page)
    return out


def prepare(case, seed):
    g = _gen(seed)
    c, s = case, {"case": dict(case)}
    op = c["op"]
    if op in ("rope", "write"):
        s["freq"], s["gain"] = _frequencies(c)
    if op == "rope":
        s["x"] = _randn(g, c["tokens"], c["heads"], c["dim"]).to(TYPES[c["act"]])
        s["y"] = torch.empty_like(s["x"])
        s["pos"] = torch.randint(0, c["context"], (c["tokens"],), device="cuda", generator=g, dtype=torch.int32)
    elif op == "write":
        wide = (c["heads"] + 2 * c["kv"]) * c["dim"]
        s["qkv"] = _randn(g, c["tokens"], wide).to(TYPES[c["act"]])
        s["q_out"] = torch.empty(c["tokens"], c["heads"], c["dim"], dtype=TYPES[c["act"]], device="cuda")
        s["pos"] = torch.randint(0, c["context"], (c["tokens"],), device="cuda", generator=g, dtype=torch.int32)
        pages = -(-c["tokens"] // c["page"]) + 3
        s["slots"] = torch.randperm(pages * c["page"], device="cuda", generator=g)[:c["tokens"]].sort().values
        s["pages"] = pages
        s["k"] = _cache(g, c["kind"], pages, c["kv"], c["page"], c["dim"], True)
        s["v"] = _cache(g, c["kind"], pages, c["kv"], c["page"], c["dim"], False)
        s["k_back"] = torch.empty(c["tokens"], c["kv"], c["dim"], dtype=torch.float16, device="cuda")
        s["v_back"] = torch.empty_like(s["k_back"])
    elif op == "read":
        pages = -(-c["tokens"] // c["page"]) + 1
        s["pages"] = pages
        table = torch.randperm(pages, device="cuda", generator=g)
        at = torch.arange(c["tokens"], device="cuda")
        s["slots"] = table[at // c["page"]] * c["page"] + at % c["page"]
        s["k"] = _cache(g, c["kind"], pages, c["kv"], c["page"], c["dim"], True)
        s["v"] = _cache(g, c["kind"], pages, c["kv"], c["page"], c["dim"], False)
        s["k_out"] = torch.empty(c["tokens"], c["kv"], c["dim"], dtype=TYPES[c["act"]], device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
    else:
        cpu = torch.Generator().manual_seed(seed)
        n, t = c["seqs"], c["drafts"]
        prefix = torch.randint(c["least"], c["most"] + 1, (n,), generator=cpu, dtype=torch.int32)
        each = -(-(prefix + t) // c["page"])  # pages of each sequence
        wide = int(each.max())
        pages = int(each.sum()) + 1
        pool = torch.randperm(pages, generator=cpu, dtype=torch.int64).int()
        first = torch.cumsum(each, 0) - each
        col = torch.arange(wide)
        table = torch.where(col < each[:, None], pool[(first[:, None] + col).clamp(max=pages - 1)], 0)
        # each draft's parent is an earlier one; a node sees itself and the nodes above it
        sees = torch.eye(t, dtype=torch.bool)
        for i in range(1, t):
            up = int(torch.randint(max(0, i - 6), i, (1,), generator=cpu))
            sees[i] |= sees[up]
        if c["chain"]:
            sees = torch.tril(torch.ones(t, t, dtype=torch.bool))
        bits = torch.zeros(t, dtype=torch.int64)
        for i in range(t):
            bits |= sees[:, i].long() << i
        s["sees"] = sees.cuda()
        s["mask"] = bits.repeat(n).cuda()
        s["pages"], s["wide"], s["table"], s["prefix"] = pages, wide, table.int().cuda().contiguous(), prefix.cuda()
        s["starts"] = torch.arange(0, (n + 1) * t, t, dtype=torch.int32, device="cuda")
        s["most"] = int((prefix + t).max())
        s["q"] = _randn(g, n * t, c["heads"], c["dim"]).to(TYPES[c["act"]])
        s["out"] = torch.empty_like(s["q"])
        s["k"] = _cache(g, c["kind"], pages, c["kv"], c["page"], c["dim"], True)
        s["v"] = _cache(g, c["kind"], pages, c["kv"], c["page"], c["dim"], False)
    return s


# ---------------------------------------------------------------- plain forms

def _frequencies(c):
    """(radians per position of each pair, in 64 bits; the gain): base^(-2i/rot), slowed by `scale`
    and, with `ext`, only where a pair turns less than once in the original context (by parts)."""
    rot, base, scale, ext = c["rot"], c["base"], c["scale"], c["ext"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    fast = base ** (-2.0 * i / rot)
    if not ext:
        return fast * scale, 1.0
    orig = ORIGINAL
    where = lambda turns: rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))
    low, high = max(0, math.floor(where(32.0))), min(rot - 1, math.ceil(where(1.0)))
    keep = (1 - ((i - low) / max(0.001, high - low)).clamp(0, 1)) * ext
    return fast * scale * (1 - keep) + fast * keep, 1 + 0.1 * math.log(1 / scale)


ORIGINAL = 8192  # the context a scaled model was trained on


def _rotate(x, pos, freq, gain, layout):
    """x [tokens, heads, dim] in 32 bits, its first 2 * len(freq) elements rotated. The angles are
    taken in 64 bits: at position 100000 a 32-bit angle is off by 0.004."""
    angle = pos.double()[:, None] * freq
    cos, sin = (angle.cos() * gain).float()[:, None], (angle.sin() * gain).float()[:, None]
    half = len(freq)
    y = x.clone()
    if layout == "pairs":
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2] = a * cos - b * sin
        y[..., 1:2 * half:2] = a * sin + b * cos
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half] = a * cos - b * sin
        y[..., half:2 * half] = a * sin + b * cos
    return y


def _unpack(records, kind, page, dim):
    """Records [..., kv, record] as values [..., kv, page, dim] in 32 bits."""
    row = dim * BITS[kind] // 8
    lead = records.shape[:-1]
    units = records[..., :page * row].unflatten(-1, (-1, 16))
    codes = units.index_select(-2, _order(page, row)).reshape(*lead, page, row)
    if kind == "f16":
        return codes.view(torch.float16).float()
    scale = _scale(records[..., page * row:]).reshape(*lead, page, dim // 32, 1)
    if kind == "q8":
        code = codes.float() - 128
    else:
        word = codes.unflatten(-1, (-1, 4))
        lo, hi = word & 15, word >> 4
        code = torch.stack([lo[..., 0], lo[..., 2], hi[..., 0], hi[..., 2], lo[..., 1], lo[..., 3],
                            hi[..., 1], hi[..., 3]], -1).flatten(-2).float() - 8
    return (code.unflatten(-1, (-1, 32)) * scale).flatten(-2)


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "rope":
        return _rotate(s["x"].float(), s["pos"], s["freq"], s["gain"], c["layout"]).to(s["x"].dtype)
    if op == "write":
        t, d, heads, kv = c["tokens"], c["dim"], c["heads"], c["kv"]
        x = s["qkv"].float().view(t, heads + 2 * kv, d)
        qk = _rotate(x[:, :heads + kv], s["pos"], s["freq"], s["gain"], c["layout"])
        kept = torch.cat([qk[:, heads:], x[:, heads + kv:]], 1)
        if c["kind"] != "f16":
            code, byte = _quantise(kept, c["kind"])
            kept = (code * _scale(byte)).flatten(-2)
        kept = kept.half()
        return {"q": qk[:, :heads].to(s["qkv"].dtype), "k": kept[:, :kv], "v": kept[:, kv:]}
    if op == "read":
        row, page = torch.div(s["slots"], c["page"], rounding_mode="floor"), s["slots"] % c["page"]
        back = lambda a: _unpack(a, c["kind"], c["page"], c["dim"])[row, :, page].to(TYPES[c["act"]])
        return {"k": back(s["k"]), "v": back(s["v"])}
    n, t, kv, d, heads = c["seqs"], c["drafts"], c["kv"], c["dim"], c["heads"]
    flat = lambda a: _unpack(a[s["table"].long()], c["kind"], c["page"], d).transpose(1, 2).flatten(2, 3)
    key, value = flat(s["k"]), flat(s["v"])  # [sequence, kv head, position, dim]
    q = s["q"].float().view(n, t, kv, heads // kv, d).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, d)
    logit = (q @ key.transpose(2, 3)).view(n, kv, t, heads // kv, -1) / math.sqrt(d)
    at = torch.arange(key.shape[2], device="cuda") - s["prefix"][:, None]  # draft's number, or < 0
    seen = (at < 0)[:, None] | (s["sees"][:, at.clamp(0, t - 1)].transpose(0, 1) & ((at >= 0) & (at < t))[:, None])
    logit = logit.masked_fill(~seen[:, None, :, None], -math.inf)
    weight = torch.exp(logit - logit.amax(-1, keepdim=True))
    weight = weight / weight.sum(-1, keepdim=True)
    out = (weight.view(n, kv, -1, key.shape[2]) @ value).view(n, kv, t, heads // kv, d)
    return out.permute(0, 2, 1, 3, 4).reshape(n * t, heads, d).to(s["q"].dtype)


# ---------------------------------------------------------------- the library's operators

_loaded = []


def _kernels():
    if not _loaded:
        import kernite_b200 as kb

        _loaded.append((kb, kb.Kernels.load(0)))
    return _loaded[0]


def _plan(s):
    """The descriptors (and the workspace) a program keeps beside its buffers."""
    kb, kernels = _kernels()
    c = s["case"]
    act = {"f32": kb.TYPE_F32, "f16": kb.TYPE_F16, "bf16": kb.TYPE_BF16}
    plan = {"kernels": kernels}
    if c["op"] in ("rope", "write"):
        rope = kb.Rope(c["rot"], layout={"pairs": kb.ROPE_PAIRS, "halves": kb.ROPE_HALVES}[c["layout"]],
                       base=c["base"], freq_scale=c["scale"], ext_factor=c["ext"], orig_ctx=ORIGINAL)
    if c["op"] == "rope":
        plan["rope"] = kb.rope_desc(rope, s["y"], s["x"], s["pos"], c["tokens"], c["heads"], c["dim"],
                                    type=act[c["act"]])
        return plan
    kind = {"f16": kb.CACHE_F16, "q8": kb.CACHE_Q8, "q4": kb.CACHE_Q4}[c["kind"]]
    cache = kb.KvCache(kind, c["kv"], c["dim"], c["page"], s["pages"], s["k"], s["v"])
    if c["op"] == "write":
        plan["write"] = kb.cache_write_desc(cache, rope, s["qkv"], s["q_out"], s["pos"], s["slots"],
                                            c["tokens"], c["heads"], type=act[c["act"]])
        plan["read"] = kb.cache_read_desc(cache, s["k_back"], s["v_back"], s["slots"], c["tokens"],
                                          type=kb.TYPE_F16)
    elif c["op"] == "read":
        plan["read"] = kb.cache_read_desc(cache, s["k_out"], s["v_out"], s["slots"], c["tokens"],
                                          type=act[c["act"]])
    else:
        plan["tree"] = kb.tree_desc(cache, s["out"], s["q"], c["heads"], s["starts"], s["prefix"], s["table"],
                                    s["wide"], c["seqs"], c["seqs"] * c["drafts"], c["drafts"], s["most"],
                                    mask=s["mask"], type=act[c["act"]])
        plan["space"] = torch.empty(kernels.tree_workspace(plan["tree"]), dtype=torch.uint8, device="cuda")
        plan["tree"].workspace, plan["tree"].workspace_bytes = plan["space"].data_ptr(), plan["space"].numel()
    return plan


def _library(s):
    if "plan" not in s:
        s["plan"] = _plan(s)
    p, op = s["plan"], s["case"]["op"]
    kernels = p["kernels"]
    if op == "rope":
        kernels.rope(p["rope"])
        return s["y"]
    if op == "write":
        kernels.cache_write(p["write"])
        kernels.cache_read(p["read"])
        return {"q": s["q_out"], "k": s["k_back"], "v": s["v_back"]}
    if op == "read":
        kernels.cache_read(p["read"])
        return {"k": s["k_out"], "v": s["v_out"]}
    kernels.attention_tree(p["tree"])
    return s["out"]


def run(state):
    return _library(state) if own else _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without

def _kept(c, rows):
    """Bytes the cache holds for `rows` positions, keys and values."""
    return 2 * rows * c["kv"] * c["dim"] * (BITS[c["kind"]] / 8 + (0 if c["kind"] == "f16" else 1 / 32))


def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}[c["act"]]
    if c["op"] == "rope":
        n = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * size + 4 * c["tokens"], "flops": 3 * n}
    if c["op"] == "write":
        t, d = c["tokens"], c["dim"]
        q, k = t * c["heads"] * d, t * c["kv"] * d
        # q|k|v in, q out, the cache written and read once, 16-bit keys and values out
        return {"bytes": (2 * q + 2 * k) * size + 2 * _kept(c, t) + 4 * k + 12 * t, "flops": 3 * (q + k) + 8 * k}
    if c["op"] == "read":
        n = c["tokens"] * c["kv"] * c["dim"]
        return {"bytes": _kept(c, c["tokens"]) + 2 * n * size + 8 * c["tokens"], "flops": 2 * n}
    mean = (c["least"] + c["most"]) / 2 + c["drafts"]
    rows = c["seqs"] * c["drafts"]
    return {"bytes": _kept(c, c["seqs"] * mean) + 2 * rows * c["heads"] * c["dim"] * size,
            "flops": 4 * rows * c["heads"] * c["dim"] * mean}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_angles(c, pos):
    rot = c["rot"]
    rate = []
    for i in range(rot // 2):
        f = c["base"] ** (-2.0 * i / rot)
        if c["ext"]:
            edge = [rot / 2 * math.log(ORIGINAL / (2 * math.pi * b), c["base"]) for b in (32.0, 1.0)]
            low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
            slow = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            f = f * (c["scale"] * slow + (1 - slow))
        else:
            f = f * c["scale"]
        rate.append(f)
    gain = 1 + 0.1 * math.log(1 / c["scale"]) if c["ext"] else 1.0
    return torch.outer(pos.double(), torch.tensor(rate, dtype=torch.float64, device=pos.device)), gain


def _exact_rotate(c, x, pos):
    """The rotation as a product of complex numbers."""
    angle, gain = _exact_angles(c, pos)
    turn = torch.polar(torch.full_like(angle, gain), angle)[:, None]
    x = x.double()
    rot = c["rot"]
    if c["layout"] == "pairs":
        z = torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * turn
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, x[..., rot:]], -1)


def _exact_kept(x, kind):
    """x as the cache holds it: the smallest scale of four significant bits that covers a block."""
    if kind == "f16":
        return x
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    least = blocks.abs().max(-1, keepdim=True).values / TOP[kind]
    power = torch.floor(torch.log2(least.clamp(min=2.0 ** -14)))
    step = torch.exp2(power - 3)
    scale = torch.ceil(least / step) * step
    code = torch.where(scale > 0, torch.round(blocks / scale.clamp(min=2.0 ** -30)), 0.0)
    return (code * scale).reshape(x.shape)


def _exact_rows(raw, c, slots):
    """Rows of the cache in 64 bits, [slots, kv, dim], by the address of every element."""
    kind, page, dim, kv = c["kind"], c["page"], c["dim"], c["kv"]
    row = dim * BITS[kind] // 8
    flat = raw.reshape(-1)
    size = raw.shape[-1]
    e = torch.arange(dim, device=raw.device)
    where = (slots // page)[:, None] * kv + torch.arange(kv, device=raw.device)
    where = where[..., None] * size
    p = (slots % page)[:, None, None]
    at = lambda byte: where + ((p * row + byte) ^ (_swizzle(p, row) << 4))
    if kind == "f16":
        low, high = flat[at(2 * e)].int(), flat[at(2 * e + 1)].int()
        sign, power, part = high >> 7, (high >> 2) & 31, ((high & 3) << 8) | low
    else:
        b = flat[where + page * row + p * (dim // 32) + e // 32].int()
        sign, power, part = torch.zeros_like(b), b >> 3, (b & 7) << 7
    size64 = torch.where(power > 0, (1024 + part).double() * torch.exp2(power.double() - 25),
                         part.double() * 2.0 ** -24)
    unit = torch.where(sign > 0, -size64, size64)
    if kind == "f16":
        return unit
    if kind == "q8":
        return (flat[at(e)].double() - 128) * unit
    place = (e % 8) // 2 + 4 * (e % 2)  # the element's nibble in its word
    byte = flat[at(e // 8 * 4 + place // 2)].int()
    return (((byte >> (4 * (place % 2))) & 15).double() - 8) * unit


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rope":
        return _exact_rotate(c, s["x"], s["pos"])
    if c["op"] == "write":
        x = s["qkv"].double().view(c["tokens"], -1, c["dim"])
        h, kv = c["heads"], c["kv"]
        return {"q": _exact_rotate(c, x[:, :h], s["pos"]),
                "k": _exact_kept(_exact_rotate(c, x[:, h:h + kv], s["pos"]), c["kind"]),
                "v": _exact_kept(x[:, h + kv:], c["kind"])}
    if c["op"] == "read":
        return {"k": _exact_rows(s["k"], c, s["slots"]), "v": _exact_rows(s["v"], c, s["slots"])}
    t, group, d = c["drafts"], c["heads"] // c["kv"], c["dim"]
    out = torch.empty(c["seqs"] * t, c["heads"], d, dtype=torch.float64, device="cuda")
    for n in range(c["seqs"]):
        length = int(s["prefix"][n])
        p = torch.arange(length + t, device="cuda")
        slots = s["table"][n].long()[p // c["page"]] * c["page"] + p % c["page"]
        open_ = torch.ones(t, length + t, dtype=torch.bool, device="cuda")
        open_[:, length:] = s["sees"]
        keys, values = _exact_rows(s["k"], c, slots), _exact_rows(s["v"], c, slots)
        for h in range(c["heads"]):
            logit = s["q"][n * t:(n + 1) * t, h].double() @ keys[:, h // group].T * d ** -0.5
            out[n * t:(n + 1) * t, h] = torch.softmax(logit.masked_fill(~open_, -math.inf), 1) @ values[:, h // group]
    return out
