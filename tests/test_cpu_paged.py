"""The paged cache's calls without a GPU: what they refuse, the rotary
frequencies, and the bounds of the index arithmetic that the kernels share."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT
from paged_model import ACCURATE, attend_cut, decode, encode, off_by

P = ctypes.c_void_p
AT = 4096  # an aligned address that no refused call reads


def _pages(rai, **kw):
    a = dict(k=AT, v=AT, layers=2, pages=8, page_size=16, kv_heads=2, head_dim=64, type=rai.CACHE_F32)
    a.update(kw)
    return rai.Pages(*a.values())


def _batch(rai, **kw):
    a = dict(tables=AT, table_stride=4, q_start=AT, kv_len=AT, seqs=2, tokens=5, max_q=3, max_kv=64)
    a.update(kw)
    return rai.PageBatch(*a.values())


def _refused(rai, rc, status, text):
    with pytest.raises(rai.RaiError) as e:
        rai._check(rc)
    assert e.value.status == status and text in str(e.value)


BAD_PAGES = [
    (dict(k=None), "RAI_E_ARG", "null"), (dict(v=None), "RAI_E_ARG", "null"), (dict(type=3), "RAI_E_ARG", "cache type"),
    (dict(type=-1), "RAI_E_ARG", "cache type"), (dict(page_size=8), "RAI_E_SHAPE", "page_size"),
    (dict(page_size=24), "RAI_E_SHAPE", "page_size"), (dict(page_size=2048), "RAI_E_SHAPE", "page_size"),
    (dict(page_size=0), "RAI_E_SHAPE", "page_size"), (dict(head_dim=0), "RAI_E_SHAPE", "head_dim"),
    (dict(head_dim=12), "RAI_E_SHAPE", "head_dim"), (dict(head_dim=264), "RAI_E_SHAPE", "head_dim"),
    (dict(layers=0), "RAI_E_SHAPE", "empty"), (dict(pages=0), "RAI_E_SHAPE", "empty"),
    (dict(kv_heads=0), "RAI_E_SHAPE", "empty"), (dict(kv_heads=4097), "RAI_E_SHAPE", "overflow"), (dict(pages=1 << 31), "RAI_E_SHAPE", "overflow"),
    (dict(k=AT + 8), "RAI_E_ARG", "aligned"), (dict(v=AT + 2), "RAI_E_ARG", "aligned"),
]
BAD_BATCH = [
    (dict(tables=None), "RAI_E_ARG", "null"), (dict(q_start=None), "RAI_E_ARG", "null"),
    (dict(kv_len=None), "RAI_E_ARG", "null"), (dict(table_stride=0), "RAI_E_SHAPE", "table_stride"),
    (dict(seqs=65536), "RAI_E_SHAPE", "65535"), (dict(tokens=1 << 31), "RAI_E_SHAPE", "overflow"),
    (dict(tokens=1 << 24), "RAI_E_SHAPE", "2^24"), (dict(max_kv=1 << 31), "RAI_E_SHAPE", "overflow"), (dict(table_stride=1 << 31), "RAI_E_SHAPE", "overflow"),
]


def _store(rai, pages=None, layer=0, batch=None, rope="ok", q_out=AT, qo_ld=256, q=AT, q_ld=256, heads=4, k=AT,
           k_ld=128, v=AT, v_ld=128):
    rope = rai.Rope(AT, 64, 0, 1.0) if rope == "ok" else rope
    return rai.lib().rai_paged_store_dev(pages or _pages(rai), layer, batch or _batch(rai), rope, q_out, qo_ld, q, q_ld,
                                         heads, k, k_ld, v, v_ld, None)


def _attend(rai, pages=None, layer=0, batch=None, opts=None, out=2 * AT, o_ld=256, q=AT, q_ld=256, heads=4, work=None, n=0):
    opts = opts or rai.AttentionOptions(0.125, 0.0, 0, None)
    return rai.lib().rai_paged_attention_dev(out, o_ld, q, q_ld, heads, pages or _pages(rai), layer,
                                             batch or _batch(rai), opts, work, n, None)


@pytest.mark.parametrize("kw,status,text", BAD_PAGES)
def test_refused_pages(rai, kw, status, text):
    _refused(rai, _store(rai, _pages(rai, **kw)), status, text)
    _refused(rai, _attend(rai, _pages(rai, **kw)), status, text)
    _refused(rai, rai.lib().rai_paged_fork_dev(_pages(rai, **kw), AT, 4, AT, 2, AT, AT, 2, 2 * AT, 2 * AT, AT, None),
             status, text)
    _refused(rai, rai.lib().rai_paged_move_dev(_pages(rai, **kw), AT, AT, 1, None, 0, None), status, text)


@pytest.mark.parametrize("kw,status,text", BAD_BATCH)
def test_refused_batches(rai, kw, status, text):
    _refused(rai, _store(rai, batch=_batch(rai, **kw)), status, text)
    _refused(rai, _attend(rai, batch=_batch(rai, **kw)), status, text)


def test_refused_stores(rai):
    R = rai.Rope
    _refused(rai, _store(rai, layer=2), "RAI_E_RANGE", "layer")
    _refused(rai, _store(rai, rope=R(None, 64, 0, 1.0)), "RAI_E_ARG", "null")
    for rot in (0, 7, 66):
        _refused(rai, _store(rai, rope=R(AT, rot, 0, 1.0)), "RAI_E_SHAPE", "rot_dim")
    _refused(rai, _store(rai, rope=R(AT, 64, 0, math.inf)), "RAI_E_ARG", "gain")
    for name in ("q", "q_out", "k", "v"):
        _refused(rai, _store(rai, **{name: None}), "RAI_E_ARG", "null")
    for name, n in (("q_ld", 255), ("qo_ld", 255), ("k_ld", 127), ("v_ld", 127)):
        _refused(rai, _store(rai, **{name: n}), "RAI_E_SHAPE", "overlap")
    _refused(rai, _store(rai, q_ld=300), "RAI_E_SHAPE", "in place")
    _refused(rai, _store(rai, pages=None, batch=None, heads=16385), "RAI_E_SHAPE", "overflow")


def test_refused_attention(rai):
    O = rai.AttentionOptions
    _refused(rai, _attend(rai, layer=2), "RAI_E_RANGE", "layer")
    for heads in (0, 3, 16386):
        _refused(rai, _attend(rai, heads=heads, q_ld=1 << 24, o_ld=1 << 24), "RAI_E_SHAPE", "heads")
    for scale in (math.nan, math.inf):
        _refused(rai, _attend(rai, opts=O(scale, 0.0, 0, None)), "RAI_E_ARG", "scale")
    for cap in (-1.0, math.nan, math.inf, 1e-31, 1e31):
        _refused(rai, _attend(rai, opts=O(1.0, cap, 0, None)), "RAI_E_ARG", "softcap")
    _refused(rai, _attend(rai, out=AT), "RAI_E_ARG", "out must not be q")
    _refused(rai, _attend(rai, batch=_batch(rai, tokens=1 << 22)), "RAI_E_SHAPE", "rows x heads")
    _refused(rai, _attend(rai, out=None), "RAI_E_ARG", "null")
    _refused(rai, _attend(rai, q=None), "RAI_E_ARG", "null")
    _refused(rai, _attend(rai, q_ld=255), "RAI_E_SHAPE", "overlap")
    _refused(rai, _attend(rai, o_ld=255), "RAI_E_SHAPE", "overlap")
    _refused(rai, _attend(rai, n=64), "RAI_E_ARG", "null")
    _refused(rai, _attend(rai, work=AT + 4, n=64), "RAI_E_ARG", "aligned")
    with pytest.raises(rai.RaiError):
        rai.attention_workspace(3, _pages(rai), _batch(rai), O(1.0, 0.0, 0, None))
    assert rai.attention_workspace(4, _pages(rai), _batch(rai, seqs=0, tables=None), O(1.0, 0.0, 0, None)) == 0


def test_refused_forks_and_moves(rai):
    L, pg = rai.lib(), _pages(rai)
    good = [pg, AT, 4, AT, 2, AT, AT, 2, 2 * AT, 2 * AT, AT, None]

    def fork(**kw):
        a = list(good)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return L.rai_paged_fork_dev(*a)

    for i in (1, 3, 5, 6, 8, 9, 10):
        _refused(rai, fork(**{f"a{i}": None}), "RAI_E_ARG", "null")
    _refused(rai, fork(a2=0), "RAI_E_SHAPE", "empty")
    _refused(rai, fork(a4=0), "RAI_E_SHAPE", "empty")
    _refused(rai, fork(a7=65536), "RAI_E_SHAPE", "65535")
    _refused(rai, fork(a8=AT + 28), "RAI_E_ARG", "tables_out overlaps")
    _refused(rai, fork(a9=AT + 4), "RAI_E_ARG", "lengths_out overlaps")
    assert fork(a7=0) == 0
    _refused(rai, L.rai_paged_move_dev(pg, None, AT, 1, None, 0, None), "RAI_E_ARG", "null")
    _refused(rai, L.rai_paged_move_dev(pg, AT, None, 1, None, 0, None), "RAI_E_ARG", "null")
    _refused(rai, L.rai_paged_move_dev(pg, AT, AT, 1, None, 3, None), "RAI_E_ARG", "null")
    _refused(rai, L.rai_paged_move_dev(pg, AT, AT, 65536, None, 0, None), "RAI_E_SHAPE", "65535")
    assert L.rai_paged_move_dev(pg, None, None, 0, None, 0, None) == 0


def test_limits_of_forks_and_moves(rai):
    """Pages x layers of a launch, in parts of 32 KB: of 2 KB (one part) and of 64 MB pages (2048)."""
    L, small, large = rai.lib(), dict(page_size=16, kv_heads=1, head_dim=32), dict(page_size=1024, kv_heads=64, head_dim=256)
    for n, layers, kw in [(65535, 129, small), (1, 4096, large), (2, 2048, large)]:
        _refused(rai, L.rai_paged_move_dev(_pages(rai, layers=layers, **kw), AT, AT, n, None, 0, None), "RAI_E_SHAPE",
                 "pages x layers")
    _refused(rai, L.rai_paged_fork_dev(_pages(rai, layers=4097, **large), AT, 4, AT, 2, AT, AT, 2, 2 * AT, 2 * AT, AT, None),
             "RAI_E_SHAPE", "overflow")
    _refused(rai, L.rai_paged_fork_dev(_pages(rai), AT, 4, AT, 65536, AT, AT, 2, 2 * AT, 2 * AT, AT, None), "RAI_E_SHAPE",
             "65535")


def test_refused_selections(rai):
    L, need = rai.lib(), rai.beam_workspace(100, 2, 3, 6)
    good = [AT, 100, 100, AT, AT, 5, 2, 3, 6, AT, AT, AT, AT, need, None]

    def select(**kw):
        a = list(good)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return L.rai_beam_select_dev(*a)

    for i in (0, 3, 9, 10, 11, 12):
        _refused(rai, select(**{f"a{i}": None}), "RAI_E_ARG", "null")
    _refused(rai, select(a1=99), "RAI_E_SHAPE", "overlap")
    _refused(rai, select(a2=0), "RAI_E_SHAPE", "empty")
    for n in (0, 65):
        _refused(rai, select(a7=n), "RAI_E_SHAPE", "beams")
        _refused(rai, select(a8=n), "RAI_E_SHAPE", "take")
    for t in (-1, 100):
        _refused(rai, select(a5=t), "RAI_E_RANGE", "end_token")
    _refused(rai, select(a12=AT + 8), "RAI_E_ARG", "aligned")
    _refused(rai, select(a13=need - 1), "RAI_E_SHAPE", "workspace")
    assert select(a6=0) == 0


def test_nothing_to_do(rai):
    """No sequences, rows or new tokens: done, whatever else is given."""
    for kw in (dict(seqs=0), dict(tokens=0), dict(max_q=0)):
        b = _batch(rai, tables=None, q_start=None, kv_len=None, **kw)
        assert _store(rai, batch=b, q=None, k=None, v=None) == 0
        assert _attend(rai, batch=b, q=None, out=None) == 0


def test_rope_frequencies(rai):
    """Against the rules written per pair: f64 powers and logs agree to some ulps."""
    near = dict(rtol=1e-13, atol=0)
    base = np.array([1e4 ** (-2 * i / 96) for i in range(48)])
    inv, gain = rai.rope_frequencies(rai.ROPE_NONE, 1e4, 96)
    assert gain == 1.0 and np.allclose(inv, base, **near)
    inv, gain = rai.rope_frequencies(rai.ROPE_LINEAR, 1e4, 96, 4.0)
    assert gain == 1.0 and np.allclose(inv, base / 4, **near)
    inv, gain = rai.rope_frequencies(rai.ROPE_LLAMA3, 1e4, 96, 8.0, 8192.0, 1.0, 4.0)
    for i, f in enumerate(base):
        wave = 2 * math.pi / f
        if wave < 8192 / 4:
            want = f
        elif wave > 8192:
            want = f / 8
        else:
            mix = (8192 / wave - 1.0) / 3.0
            want = (1 - mix) * f / 8 + mix * f
        assert math.isclose(inv[i], want, rel_tol=1e-12), i
    assert gain == 1.0 and inv[0] == 1.0 and math.isclose(inv[47], base[47] / 8, rel_tol=1e-12)
    inv, gain = rai.rope_frequencies(rai.ROPE_YARN, 1e4, 96, 16.0, 4096.0)
    at = [96 * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(1e4)) for n in (32, 1)]
    lo, hi = math.floor(at[0]), math.ceil(at[1])
    for i, f in enumerate(base):
        r = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        assert math.isclose(inv[i], f * (1 - r) + f / 16 * r, rel_tol=1e-12), i
    assert gain == np.float32(0.1 * math.log(16.0) + 1.0)


def test_refused_frequencies(rai):
    ok = dict(scaling=rai.ROPE_LLAMA3, theta=1e4, rot_dim=64, factor=8.0, trained_context=8192.0, low_freq=1.0,
              high_freq=4.0)
    for kw, text in [(dict(scaling=4), "scaling"), (dict(scaling=-1), "scaling"), (dict(theta=0.0), "theta"),
                     (dict(theta=math.inf), "theta"), (dict(theta=math.nan), "theta"), (dict(rot_dim=0), "rot_dim"),
                     (dict(rot_dim=63), "rot_dim"), (dict(factor=0.5), "factor"), (dict(factor=math.nan), "factor"),
                     (dict(trained_context=0.0), "trained"), (dict(low_freq=0.0), "low_freq"),
                     (dict(low_freq=4.0), "low_freq"), (dict(high_freq=math.inf), "low_freq"),
                     (dict(scaling=rai.ROPE_YARN, theta=1.0), "theta 1")]:
        with pytest.raises(rai.RaiError) as e:
            rai.rope_frequencies(**{**ok, **kw})
        assert text in str(e.value)


def test_index_bounds(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "rai_amd", "csrc"), os.path.join(ROOT, "tests", "paged_index_check.cpp"),
                    "-o", exe], check=True)
    assert subprocess.run([exe], capture_output=True, text=True, check=True).stdout == "ok\n"


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_parts_of_matrix_operands(cache, hd):
    """The parts that the attention's 16-bit operands are cut into leave f32 accuracy; with a part less in any
    operand, or fewer products, attention is off by several times what its tests on the GPU allow."""
    r = np.random.default_rng(hd)
    q = r.standard_normal((32, hd)).astype(np.float32)
    k, v = (decode(encode(r.standard_normal((900, hd)), cache), cache) for _ in range(2))
    s = q.astype(np.float64) @ k.T.astype(np.float64) / np.sqrt(hd)
    p = np.exp(s - s.max(1, keepdims=True))
    want = p @ v.astype(np.float64) / p.sum(1, keepdims=True)
    whole = {"f32": dict(query_parts=3, weight_parts=3, key_parts=3, value_parts=3, products=3),
             "f16": dict(query_parts=2, weight_parts=2), "bf16": dict(query_parts=3, weight_parts=3)}[cache]
    assert off_by(attend_cut(q, k, v, cache, **whole), want)[0] < 3
    for name, n in whole.items():
        assert off_by(attend_cut(q, k, v, cache, **{**whole, name: n - 1}), want)[0] > 4 * ACCURATE, name
