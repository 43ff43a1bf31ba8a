"""Plain f64 / integer restatements, in numpy, of the operators on drafted tokens: rotary positions, the
paged cache's quantisation and byte layout, and the attention of a tree of drafts. Written from the
definitions in include/kq.h, one element at a time where it matters; test infrastructure only."""
from __future__ import annotations

import math
from decimal import Decimal, localcontext

import numpy as np

F16, Q8, Q4 = 0, 1, 2
TOP = {Q8: 127, Q4: 7}
LAST = {Q8: 0xA6, Q4: 0xC6}  # the largest scale byte
NAN_SCALE = 0xFF


def scale_value(byte) -> np.ndarray:
    """A scale byte as the f16 with bits byte << 7, in f64."""
    return (np.asarray(byte, dtype=np.uint16) << 7).view(np.float16).astype(np.float64)


# every finite scale, ascending
SCALES = scale_value(np.arange(0xF8))


# ---------------------------------------------------------------- rotary positions

def rope_angles(rot: int, base: float, freq_scale: float = 1.0, ext_factor: float = 0.0,
                attn_factor: float = 1.0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                orig_ctx: int = 0, freq_factors=None):
    """(radians per position of each pair, gain)."""
    out = []
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if freq_factors is not None:
            f /= float(np.float32(freq_factors[i]))
        if ext_factor:
            # the pair that turns b times over the original context: base^(-2i/rot) * ctx = 2 pi b
            edge = [rot * math.log(orig_ctx / (2 * math.pi * b)) / (2 * math.log(base))
                    for b in (beta_fast, beta_slow)]
            low, high = max(0.0, math.floor(edge[0])), min(rot - 1.0, math.ceil(edge[1]))
            ramp = min(1.0, max(0.0, (i - low) / max(0.001, high - low)))
            mix = (1 - ramp) * ext_factor
            f *= freq_scale * (1 - mix) + mix
        else:
            f *= freq_scale
        out.append(f)
    gain = attn_factor * (1 + 0.1 * math.log(1 / freq_scale) if ext_factor else 1.0)
    return np.array(out), gain


def rope_turns(rot: int, base: float, freq_scale: float = 1.0, ext_factor: float = 0.0, beta_fast: float = 32.0,
               beta_slow: float = 1.0, orig_ctx: int = 0, freq_factors=None) -> list:
    """Turns per position of each pair, to 50 digits."""
    with localcontext() as ctx:
        ctx.prec = 60
        two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
        big = Decimal(base)
        out = []
        for i in range(rot // 2):
            f = big ** (Decimal(-2 * i) / rot)
            if freq_factors is not None:
                f /= Decimal(float(np.float32(freq_factors[i])))
            slow = Decimal(freq_scale)
            if ext_factor:
                edge = [rot * (orig_ctx / (two_pi * Decimal(b))).ln() / (2 * big.ln()) for b in (beta_fast, beta_slow)]
                low, high = max(0, math.floor(edge[0])), min(rot - 1, math.ceil(edge[1]))
                ramp = min(Decimal(1), max(Decimal(0), (i - low) / max(Decimal(0.001), Decimal(high - low))))
                mix = (1 - ramp) * Decimal(ext_factor)
                slow = slow * (1 - mix) + mix
            out.append(f * slow / two_pi)
        return out


def rope(x, positions, rot: int, halves: bool, angles, gain: float) -> np.ndarray:
    """x (tokens, heads, dim), its first rot elements rotated, f64."""
    y = np.array(x, dtype=np.float64)
    a = np.asarray(positions, dtype=np.float64)[:, None] * angles
    c, s = gain * np.cos(a)[:, None], gain * np.sin(a)[:, None]
    if halves:
        u, v = y[..., : rot // 2].copy(), y[..., rot // 2: rot].copy()
        y[..., : rot // 2], y[..., rot // 2: rot] = u * c - v * s, u * s + v * c
    else:
        u, v = y[..., 0:rot:2].copy(), y[..., 1:rot:2].copy()
        y[..., 0:rot:2], y[..., 1:rot:2] = u * c - v * s, u * s + v * c
    return y


# ---------------------------------------------------------------- the cache's blocks

def quantise(x, kind: int):
    """f32 rows (..., dim), dim a multiple of 32 -> (codes, scale bytes): the smallest scale that covers
    the block, codes the nearest integers (f32 quotients, ties to even)."""
    x = np.asarray(x, dtype=np.float32)
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore"):
        most = np.abs(blocks).max(-1)
    bad = ~np.isfinite(blocks).all(-1)
    most = np.where(bad, 0, most)
    # most / top rounded to f32 first, as the definition's quotient is
    want = (most.astype(np.float32) / np.float32(TOP[kind])).astype(np.float64)
    byte = np.searchsorted(SCALES, want, side="left").clip(max=LAST[kind])
    scale = scale_value(byte)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        code = np.rint(blocks / np.where(scale > 0, scale, 1)[..., None].astype(np.float32))
    code = np.clip(np.where((scale > 0)[..., None], code, 0), -TOP[kind], TOP[kind])
    code = np.where(bad[..., None], 0, code).astype(np.int64)
    byte = np.where(bad, NAN_SCALE, byte).astype(np.uint8)
    return code.reshape(x.shape), byte


def kept(x, kind: int) -> np.ndarray:
    """x as the cache holds it, f64."""
    if kind == F16:
        with np.errstate(over="ignore"):
            return np.asarray(x, dtype=np.float32).astype(np.float16).astype(np.float64)
    code, byte = quantise(x, kind)
    with np.errstate(invalid="ignore"):
        return code * np.repeat(scale_value(byte), 32, axis=-1)


# ---------------------------------------------------------------- the cache's bytes

class Layout:
    def __init__(self, kind: int, n_kv: int, dim: int, page: int, n_pages: int):
        self.kind, self.n_kv, self.dim, self.page, self.n_pages = kind, n_kv, dim, page, n_pages
        self.pitch = 64 if dim <= 64 else 128 if dim <= 128 else 256
        self.row = {F16: 2 * self.pitch, Q8: self.pitch, Q4: self.pitch // 2}[kind]
        self.scales = 0 if kind == F16 else self.pitch // 32
        self.record = page * (self.row + self.scales)

    @property
    def nbytes(self) -> int:
        return self.n_pages * self.n_kv * self.record

    def swizzle(self, p: int) -> int:
        return p % 8 if self.row >= 128 else 2 * (p // 2 % 4) if self.row == 64 else 4 * (p // 4 % 2)

    def row_bytes(self, p: int) -> np.ndarray:
        """Where each byte of position p's row of codes lies in a record."""
        at = p * self.row + np.arange(self.row)
        return (at // 16 ^ self.swizzle(p)) * 16 + at % 16

    def put(self, buf: np.ndarray, slot: int, rows: np.ndarray) -> None:
        """f32 rows (n_kv, dim) into slot `slot` of the buffer (nbytes bytes)."""
        full = np.zeros((self.n_kv, self.pitch), dtype=np.float32)
        full[:, : self.dim] = rows
        page, p = divmod(slot, self.page)
        for h in range(self.n_kv):
            rec = buf[(page * self.n_kv + h) * self.record:][: self.record]
            if self.kind == F16:
                with np.errstate(over="ignore"):
                    rec[self.row_bytes(p)] = full[h].astype(np.float16).view(np.uint8)
                continue
            code, byte = quantise(full[h], self.kind)
            at = self.page * self.row + p * self.scales
            rec[at: at + self.scales] = byte
            if self.kind == Q8:
                rec[self.row_bytes(p)] = (code + 128).astype(np.uint8)
            else:
                u = (code + 8).reshape(-1, 8)
                word = sum(u[:, e] << (4 * (e // 2 + 4 * (e % 2))) for e in range(8)).astype(np.uint32)
                rec[self.row_bytes(p)] = word.view(np.uint8)

    def get(self, buf: np.ndarray, slot: int) -> np.ndarray:
        """Slot's values, f64 (n_kv, dim)."""
        page, p = divmod(slot, self.page)
        out = np.empty((self.n_kv, self.pitch))
        for h in range(self.n_kv):
            rec = buf[(page * self.n_kv + h) * self.record:][: self.record]
            raw = rec[self.row_bytes(p)]
            if self.kind == F16:
                out[h] = raw.view(np.float16)
                continue
            at = self.page * self.row + p * self.scales
            with np.errstate(invalid="ignore"):
                scale = np.repeat(scale_value(rec[at: at + self.scales]), 32)
                if self.kind == Q8:
                    out[h] = (raw.astype(np.float64) - 128) * scale
                else:
                    word = raw.view(np.uint32)
                    code = np.stack([(word >> (4 * (e // 2 + 4 * (e % 2)))) & 15 for e in range(8)], -1)
                    out[h] = (code.reshape(-1).astype(np.float64) - 8) * scale
        return out[:, : self.dim]


# ---------------------------------------------------------------- attention of drafted tokens

def tree_attention(q, keys, values, prefix: int, masks, scale: float):
    """One sequence's drafts q (drafts, heads, dim) over its positions keys, values (prefix + drafts,
    n_kv, dim), f64. masks: a word a draft (bit u: it sees draft u). Returns (out, sum_p w_p |v_p|, the
    largest sum_e |q_e k_e| * scale over the positions a row sees)."""
    q = np.asarray(q, dtype=np.float64)
    drafts, heads, dim = q.shape
    group = heads // keys.shape[1]
    out, weight, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    for t in range(drafts):
        seen = [p for p in range(prefix + drafts) if p < prefix or masks[t] >> (p - prefix) & 1]
        if not seen:
            continue
        for h in range(heads):
            k, v = keys[seen, h // group], values[seen, h // group]
            logit = k @ q[t, h] * scale
            w = np.exp(logit - logit.max())
            w /= w.sum()
            out[t, h], weight[t, h] = w @ v, w @ np.abs(v)
            reach[t, h] = (np.abs(k) @ np.abs(q[t, h])).max() * scale
    return out, weight, reach
