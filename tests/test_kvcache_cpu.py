"""What the calls on drafted tokens check and make on the host, without a GPU: the descriptors' layout, the
rotation's table, a cache's size, refusals; and the f64 restatement against the definitions it restates."""
import ctypes
import os
import subprocess
from fractions import Fraction

import numpy as np
import pytest

import kernite_b200 as kb
from oracle import kvcache as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"kq_rope_params": kb.KqRopeParams, "kq_rope": kb.KqRope, "kq_rope_desc": kb.KqRopeDesc,
           "kq_cache": kb.KqCache, "kq_cache_write_desc": kb.KqCacheWriteDesc,
           "kq_cache_read_desc": kb.KqCacheReadDesc, "kq_cache_move_desc": kb.KqCacheMoveDesc,
           "kq_tree_desc": kb.KqTreeDesc}


def test_descriptor_layouts_match_the_header(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {field[0]}));' for field in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "kq.h"\nint main(void){' + "\n".join(lines)
                   + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in STRUCTS.values():
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, field[0]).offset for field in cls._fields_]
    assert got == want


def test_entry_points_reject_null_ctx():
    L = kb.lib()
    for name, cls in (("kq_rope_apply", kb.KqRopeDesc), ("kq_cache_write", kb.KqCacheWriteDesc),
                      ("kq_cache_read", kb.KqCacheReadDesc), ("kq_cache_move", kb.KqCacheMoveDesc),
                      ("kq_attention_tree", kb.KqTreeDesc)):
        assert getattr(L, name)(None, ctypes.byref(cls()), None) == kb.KQ_E_INVALID, name
        assert name in kb.last_error()
    assert L.kq_tree_workspace(None, ctypes.byref(kb.KqTreeDesc())) == 0


@pytest.mark.parametrize("rot,kw", [(2, {}), (128, {}), (64, dict(base=500000.0)), (256, dict(freq_scale=0.25)),
                                    (96, dict(base=500000.0, freq_scale=0.25, ext_factor=1.0, orig_ctx=8192)),
                                    (16, dict(freq_factors=[1, 2, 3, 4, 5, 6, 7, 8]))], ids=str)
def test_rope_table(rot, kw):
    """Turns modulo 1, times 2^64. A table in f64 arithmetic is right to a few 2^-53 of a pair's turns."""
    table = kb.Rope(rot, **kw).c
    angles, gain = ref.rope_angles(rot, kw.get("base", 10000.0), **{k: v for k, v in kw.items() if k != "base"})
    assert abs(table.gain - gain) <= 2.0 ** -23 * gain
    pi2 = Fraction(884279719003555, 2 ** 47)  # 2 pi to f64
    for i, a in enumerate(angles):
        want = Fraction(float(a)) / pi2 % 1
        off = abs(Fraction(table.turns[i], 2 ** 64) - want)
        assert min(off, 1 - off) <= Fraction(1, 2 ** 48)


@pytest.mark.parametrize("rot,kw", [(2, {}), (256, {}), (128, dict(base=500000.0)), (96, dict(base=1e8)),
                                    (64, dict(base=10000.0, freq_scale=0.3)),
                                    (96, dict(base=500000.0, freq_scale=0.25, ext_factor=0.7, orig_ctx=8192)),
                                    (16, dict(freq_factors=[1, 2, 3.7, 4, 5, 6, 7, 8]))], ids=str)
def test_rope_table_to_its_last_bits(rot, kw):
    """The table against 50 digits: the nearest 2^-64 is 2^-65 away at most, and 64-bit significands add a few
    2^-67 (turns are below 1/6, each of five operations errs by 2^-65 of the result), 2^-63 in all; so a position
    of 2^31 is 2^-32 turns off at most."""
    table = kb.Rope(rot, **kw).c
    for i, want in enumerate(ref.rope_turns(rot, kw.get("base", 10000.0),
                                            **{k: v for k, v in kw.items() if k != "base"})):
        off = abs(Fraction(table.turns[i], 2 ** 64) - Fraction(want) % 1)
        assert min(off, 1 - off) <= Fraction(1, 2 ** 63), i


@pytest.mark.parametrize("rot,kw", [(0, {}), (3, {}), (258, {}), (64, dict(layout=7)), (64, dict(base=1.0)),
                                    (64, dict(base=float("nan"))), (64, dict(freq_scale=0.0)),
                                    (64, dict(freq_scale=float("inf"))), (64, dict(ext_factor=1.0)),
                                    (4, dict(freq_factors=[1, 0])), (4, dict(freq_factors=[1]))], ids=str)
def test_rope_refusals(rot, kw):
    with pytest.raises(kb.Error):
        kb.Rope(rot, **kw)


@pytest.mark.parametrize("kind,n_kv,dim,page,pages", [(ref.F16, 1, 32, 16, 1), (ref.Q8, 8, 128, 64, 129),
                                                      (ref.Q4, 3, 96, 256, 7), (ref.Q4, 2, 64, 32, 5),
                                                      (ref.Q8, 32, 256, 128, 1 << 16)])
def test_cache_bytes(kind, n_kv, dim, page, pages):
    assert kb.cache_bytes(kind, n_kv, dim, page, pages) == ref.Layout(kind, n_kv, dim, page, pages).nbytes


@pytest.mark.parametrize("kind,n_kv,dim,page,pages", [(3, 1, 64, 16, 1), (1, 0, 64, 16, 1), (1, 1, 0, 16, 1),
                                                      (1, 1, 48, 16, 1), (1, 1, 288, 16, 1), (1, 1, 64, 24, 1),
                                                      (1, 1, 64, 512, 1), (1, 1, 64, 8, 1), (1, 1, 64, 16, 0)])
def test_cache_refusals(kind, n_kv, dim, page, pages):
    with pytest.raises(kb.Error):
        kb.cache_bytes(kind, n_kv, dim, page, pages)


# ---------------------------------------------------------------- the restatement

def test_scales_are_f16_with_three_fraction_bits():
    assert ref.SCALES[0] == 0 and ref.SCALES[1] == 2.0 ** -17 and ref.SCALES[0x78] == 1.0
    assert (np.diff(ref.SCALES) > 0).all()
    assert ref.scale_value(ref.LAST[ref.Q8]) * 127 == 7112 and ref.scale_value(ref.LAST[ref.Q4]) * 7 == 6272


@pytest.mark.parametrize("kind", [ref.Q8, ref.Q4])
def test_blocks_take_the_smallest_scale_and_the_nearest_code(kind):
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((400, 32)) * 10.0 ** rng.uniform(-6, 3, (400, 1))).astype(np.float32)
    code, byte = ref.quantise(x, kind)
    top = ref.TOP[kind]
    for row, c, b in zip(x.astype(np.float64), code, byte[:, 0]):
        most = np.abs(row).max()
        assert np.abs(c).max() <= top
        if b < ref.LAST[kind]:
            assert ref.SCALES[b] * top >= most * (1 - 2.0 ** -24)
        assert b == 0 or ref.SCALES[b - 1] * top < most
        if b and most <= ref.SCALES[b] * top:
            assert (np.abs(row - c * ref.SCALES[b]) <= ref.SCALES[b] * (0.5 + 2.0 ** -15)).all()
    values = ref.kept(x, kind)
    assert (values == values.astype(np.float16)).all()  # exact in f16


@pytest.mark.parametrize("kind", [ref.F16, ref.Q8, ref.Q4])
@pytest.mark.parametrize("dim,page", [(32, 16), (64, 32), (96, 64), (128, 16), (256, 128)])
def test_records_hold_every_row_apart(kind, dim, page):
    layout = ref.Layout(kind, 2, dim, page, 2)
    rng = np.random.default_rng(4)
    buf = rng.integers(0, 256, layout.nbytes).astype(np.uint8)
    rows = rng.standard_normal((2 * page, 2, dim)).astype(np.float32)
    order = rng.permutation(2 * page)
    for slot in order:
        layout.put(buf, int(slot), rows[slot])
    for slot in range(2 * page):
        assert (layout.get(buf, slot) == ref.kept(rows[slot], kind)).all()
    every = np.concatenate([layout.row_bytes(p) for p in range(page)])
    assert (np.sort(every) == np.arange(page * layout.row)).all()


def test_attention_of_hand_sized_trees():
    q = np.zeros((2, 2, 4))
    q[:, :, 0] = 1.0
    keys, values = np.zeros((3, 1, 4)), np.arange(12.0).reshape(3, 1, 4)
    out, weight, _ = ref.tree_attention(q, keys, values, 1, [0b01, 0b10], 1.0)
    assert (out[0, 0] == [2, 3, 4, 5]).all() and (out[1, 1] == [4, 5, 6, 7]).all() and (weight == out).all()
    keys[1, 0, 0] = np.log(3.0)
    out, _, _ = ref.tree_attention(q, keys, values, 1, [0b01, 0b10], 1.0)
    assert np.allclose(out[0, 0], (values[0, 0] + 3 * values[1, 0]) / 4, rtol=1e-15)
    out, _, _ = ref.tree_attention(q, keys[:2], values[:2], 0, [0, 0], 1.0)
    assert (out == 0).all()
