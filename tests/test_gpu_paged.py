"""The paged cache's calls on the GPU against their definitions in 64 bits
(paged_model.py).  Slots that hold no position are NaN throughout, so that a read
of one shows."""
import ctypes
import gc

import numpy as np
import pytest

from paged_model import ACCURATE, EPS32, Pool, attend, decode, encode, off_by, rotate, spans, store_dtype

pytestmark = pytest.mark.gpu

CACHES = ["f32", "f16", "bf16"]
SENTINEL = np.float32(-12345.0)


class Dev:
    """Device arrays of one test, alive until it ends."""

    def __init__(self, rai):
        self.rai, self.keep = rai, []

    def up(self, a):
        self.keep.append(self.rai.DeviceArray.from_host(a))
        return self.keep[-1]

    def pages(self, pool):
        t = dict(f32=self.rai.CACHE_F32, f16=self.rai.CACHE_F16, bf16=self.rai.CACHE_BF16)[pool.cache]
        self.k, self.v = self.up(pool.k), self.up(pool.v)
        return self.rai.Pages(self.k.ptr, self.v.ptr, pool.layers, pool.pages, pool.page, pool.kv_heads, pool.hd, t)

    def batch(self, pool, q_start, kv_len, tokens, max_q, max_kv):
        return self.rai.PageBatch(self.up(pool.tables).ptr, pool.tables.shape[1], self.up(np.int32(q_start)).ptr,
                                  self.up(np.int32(kv_len)).ptr, len(kv_len), tokens, max_q, max_kv)

    def pool_back(self, pool):
        return (self.k.to_host(pool.k.dtype, pool.k.size).reshape(pool.k.shape),
                self.v.to_host(pool.v.dtype, pool.v.size).reshape(pool.v.shape))


def _starts(news, front=0):
    return np.concatenate([[0], np.cumsum(news)]) + front


def _claims(cut, tokens):
    """How many sequences have each row: row starts that do not ascend give a row to two, and then it holds
    either's result."""
    n = np.zeros(tokens, int)
    for q0, nq, _ in cut:
        n[q0:q0 + nq] += 1
    return n


def _run_attention(rai, dev, pg, batch, q, heads, hd, opts, layer=0, ld=None, out_ld=None, work=None, stream=None):
    """q [tokens][heads][hd]; rows lie `ld` floats apart on the device, NaN between them."""
    tokens, wide = q.shape[0], heads * hd
    ld, out_ld = ld or wide, out_ld or wide
    rows = np.full((tokens, ld), np.nan, np.float32)
    rows[:, :wide] = q.reshape(tokens, wide)
    dq, do = dev.up(rows), dev.up(np.full((tokens, out_ld), SENTINEL, np.float32))
    n = rai.attention_workspace(heads, pg, batch, opts) if work is None else work
    # Scratch that holds NaN, and a guard behind it.
    dw = dev.up(np.full(n // 4 + 64, np.nan, np.float32))
    rai._check(rai.lib().rai_paged_attention_dev(do.ptr, out_ld, dq.ptr, ld, heads, pg, layer, batch, opts,
                                                 dw.ptr if n else None, n, stream))
    rai._check(rai.lib().rai_device_synchronize())
    assert np.isnan(dw.to_host(np.float32, n // 4 + 64)[n // 4:]).all()
    out = do.to_host(np.float32, tokens * out_ld).reshape(tokens, out_ld)
    assert (out[:, wide:] == SENTINEL).all()
    return out[:, :wide].reshape(tokens, heads, hd)


def _check_attention(rai, pool, news, lengths, heads, scale, softcap=0.0, window=0, slopes=None, front=0, back=0,
                     layer=0, ld=None, out_ld=None, q=None, q_start=None, max_q=None, max_kv=None, works=(None, 0)):
    dev, hd = Dev(rai), pool.hd
    tokens = front + sum(news) + back
    if q is None:
        q = np.random.default_rng(len(news)).standard_normal((tokens, heads, hd)).astype(np.float32)
    q_start = _starts(news, front) if q_start is None else q_start
    max_q = max(news) if max_q is None else max_q
    max_kv = max(lengths) if max_kv is None else max_kv
    pg = dev.pages(pool)
    batch = dev.batch(pool, q_start, lengths, tokens, max_q, max_kv)
    opts = rai.AttentionOptions(scale, softcap, window, dev.up(np.float32(slopes)).ptr if slopes is not None else None)
    cut = spans(q_start, lengths, tokens, max_q, min(max_kv, pool.tables.shape[1] * pool.page))
    want = [attend(pool, layer, sp, s, q, heads, scale, softcap, window, slopes) for s, sp in enumerate(cut)]
    for work in works:
        got = _run_attention(rai, dev, pg, batch, q, heads, hd, opts, layer, ld, out_ld, work)
        mine = _claims(cut, tokens)
        for (q0, nq, _), (w, tol) in zip(cut, want):
            g = got[q0:q0 + nq].astype(np.float64)
            bad = ~(np.abs(g - w) <= tol + 1e-30)
            bad[mine[q0:q0 + nq] > 1] = False
            assert not bad.any(), (work, np.argwhere(bad)[:4], g[bad][:4], w[bad][:4], tol[bad][:4])
        assert (got[mine == 0] == SENTINEL).all()
    return got


# Heads, kv heads, head size: groups of one to twelve, sizes on both sides of whole tiles.
LAYOUTS = [(4, 4, 64), (8, 1, 128), (6, 2, 80), (32, 8, 128), (3, 3, 8), (5, 1, 256), (12, 1, 96), (32, 4, 64),
           (2, 1, 40), (34, 2, 72), (2, 2, 160)]
# New tokens and lengths: one token, none, lengths on both sides of a page and of a tile, longer chunks.
BATCHES = [
    ([1], [1]),
    ([1, 1, 1, 1], [17, 16, 300, 33]),
    ([0, 3, 0, 9], [40, 3, 0, 77]),
    ([37, 1, 130], [37, 64, 200]),
    ([5, 2], [3, 0]),  # fewer positions than rows: the first rows see nothing
]


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("news,lengths", BATCHES)
def test_attention(rai, cache, heads, kv_heads, hd, news, lengths):
    page = 16 << (heads + len(news)) % 4
    pool = Pool(cache, page, kv_heads, hd, lengths, seed=hd + heads)
    pool.fill(0, lengths)
    _check_attention(rai, pool, news, lengths, heads, hd ** -0.5, front=len(news) % 2, back=1 + heads % 3,
                     ld=heads * hd + 12, out_ld=heads * hd + 1)


OPTIONS = [dict(softcap=5.0), dict(window=1), dict(window=50), dict(window=129, softcap=30.0), dict(slopes=True),
           dict(slopes=True, window=70, softcap=20.0)]


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("opt", range(len(OPTIONS)))
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 64), (4, 1, 128)])
def test_attention_options(rai, cache, opt, heads, kv_heads, hd):
    o = dict(OPTIONS[opt])
    if o.get("slopes"):
        o["slopes"] = 2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)
    news, lengths = [1, 70, 9], [260, 200, 33]
    pool = Pool(cache, 32, kv_heads, hd, lengths, seed=opt, layers=2)
    pool.fill(1, lengths)
    _check_attention(rai, pool, news, lengths, heads, 0.2, layer=1, **o)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("news,lengths", [([1], [3001]), ([1, 2], [2500, 700]), ([40], [2100])])
def test_attention_long(rai, cache, news, lengths):
    """Long axes, split where scratch is given and in one pass where it is not."""
    pool = Pool(cache, 64, 2, 64, lengths, seed=3)
    pool.fill(0, lengths)
    _check_attention(rai, pool, news, lengths, 8, 0.3, works=(None, 0, 4096, 20000))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("news,lengths", [([1, 1], [90, 300]), ([33, 70], [90, 260])])
def test_attention_large_scores(rai, cache, news, lengths):
    """Scores of some hundreds: one key takes nearly all the weight, and the running maximum rises often."""
    pool = Pool(cache, 16, 1, 64, lengths, seed=4)
    pool.fill(0, lengths, std=6.0)
    q = 8.0 * np.random.default_rng(2).standard_normal((sum(news), 4, 64)).astype(np.float32)
    _check_attention(rai, pool, news, lengths, 4, 0.3, q=q)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4])
def test_attention_sizes_of_values(rai, cache, size):
    """Queries far from one: small ones, and large ones against small scales."""
    lengths = [100, 50]
    pool = Pool(cache, 16, 2, 64, lengths, seed=5)
    pool.fill(0, lengths)
    q = size * np.random.default_rng(2).standard_normal((21, 4, 64)).astype(np.float32)
    _check_attention(rai, pool, [20, 1], lengths, 4, 0.125 / max(size, 1.0), q=np.float32(q))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("nq,n", [(1, 200), (40, 200)])
def test_attention_infinities_in_masked_places(rai, cache, value, which, nq, n):
    """Keys that only some rows see: the others are as if those were not there."""
    heads, hd, window = 4, 64, 100
    pool = Pool(cache, 16, 2, hd, [n], seed=6)
    pool.fill(0, [n])
    clean = np.array(pool.k if which == "k" else pool.v)
    mine = pool.k if which == "k" else pool.v
    spots = [n - nq - window, n - nq - window + 3, n - 2]  # behind every window, behind some, in front of some
    for p in spots:
        pg, slot = pool.place(0, p)
        if which == "k":
            mine[0, pg, :, slot, 5] = encode(np.float32([value]), cache)[0]
        else:
            mine[0, pg, :, 5, slot] = encode(np.float32([value]), cache)[0]
    dev = Dev(rai)
    q = np.abs(np.random.default_rng(1).standard_normal((nq, heads, hd))).astype(np.float32)
    pg, batch = dev.pages(pool), dev.batch(pool, [0, nq], [n], nq, nq, n)
    opts = rai.AttentionOptions(0.125, 0.0, window, None)
    mine[:] = clean
    want, tol = attend(pool, 0, (0, nq, n), 0, q, heads, 0.125, window=window)
    # -inf in a key, seen with positive queries: weight zero, as if the key were not there.
    for work in (None, 0):
        got = _run_attention(rai, dev, pg, batch, q, heads, hd, opts, work=work)
        for j in range(nq):
            pos = n - nq + j
            seen = any(pos - window < p <= pos for p in spots)
            if not seen:
                assert (np.abs(got[j] - want[j]) <= tol[j]).all(), j
            elif which == "v":
                others = np.arange(hd) != 5
                assert (np.abs(got[j] - want[j]) <= tol[j])[:, others].all(), j
                ok = np.isnan(got[j][:, 5]) if np.isnan(value) else got[j][:, 5] == value
                assert ok.all(), (j, got[j][:, 5])
            elif value == -np.inf:
                assert np.isfinite(got[j]).all(), j
            else:
                assert np.isnan(got[j]).all(), j


@pytest.mark.parametrize("cache", CACHES)
def test_attention_bad_entries(rai, cache):
    """Page ids outside the pool, row starts and lengths past their bounds: cut, as documented."""
    lengths = [150, 90, 200]
    pool = Pool(cache, 16, 2, 64, lengths, seed=7)
    pool.fill(0, lengths)
    pool.tables[0, 2], pool.tables[0, 5], pool.tables[2, 0] = -7, pool.pages, 1 << 30
    pool.tables[1, :] = np.iinfo(np.int32).min  # a sequence without pages
    _check_attention(rai, pool, [3, 2, 40], lengths, 4, 0.125)
    pool.tables[1, :] = pool.tables[2, :]
    _check_attention(rai, pool, [3, 2, 40], [150, 10 ** 9, -4], 4, 0.125, max_kv=180)
    _check_attention(rai, pool, [3, 2, 40], lengths, 4, 0.125, q_start=[-5, 3, 2, 10 ** 9], max_q=20)


@pytest.mark.parametrize("seed", range(24))
def test_attention_random_batches(rai, seed):
    """Head layouts, sizes, lengths, options, strides, layers and broken tables, drawn."""
    r = np.random.default_rng(seed)
    hd, kv_heads, per = 8 * r.integers(1, 33), int(r.choice([1, 2, 3, 5])), int(r.choice([1, 2, 3, 4, 7, 8, 33]))
    heads, seqs = kv_heads * per, r.integers(1, 6)
    news = [int(r.choice([0, 1, 1, 2, 9, 40])) for _ in range(seqs)] + [1]
    lengths = [max(0, m + int(r.choice([-3, 0, 1, 15, 63, 200, 500]))) for m in news]
    pool = Pool(CACHES[seed % 3], 16 << r.integers(5), kv_heads, int(hd), lengths, seed=seed, layers=2)
    pool.fill(1, lengths, std=float(r.choice([0.3, 1.0, 3.0])))
    for _ in range(seed % 4):
        pool.tables[r.integers(seqs), r.integers(pool.tables.shape[1])] = int(r.choice([-1, pool.pages, 1 << 30]))
    slopes = 2.0 ** (-8.0 * np.arange(1, heads + 1) / heads) if r.random() < 0.3 else None
    _check_attention(rai, pool, news, lengths, heads, float(r.choice([hd ** -0.5, -0.2, 0.5, 0.0])),
                     softcap=float(r.choice([0.0, 3.0, 25.0])), window=int(r.choice([0, 1, 7, 64, 301])), slopes=slopes,
                     front=int(r.integers(3)), back=int(r.integers(3)), layer=1, ld=int(heads * hd + r.choice([0, 1, 4])),
                     out_ld=int(heads * hd + r.choice([0, 3, 4])), works=(None, 0, int(4096 * r.integers(1, 40))))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("news,lengths,split", [([1, 1], [200, 180], False), ([1, 3], [2000, 900], False),
                                                ([1, 3], [2000, 900], True), ([90], [700], False), ([90], [1800], True)])
def test_attention_is_as_accurate_as_f32(rai, cache, hd, news, lengths, split):
    """Normal inputs, by norms: few rows and chunks, in one pass and in splits."""
    heads, kv_heads, tokens = 4, 2, sum(news)
    pool = Pool(cache, 32, kv_heads, hd, lengths, seed=hd + tokens)
    pool.fill(0, lengths)
    q = np.random.default_rng(hd).standard_normal((tokens, heads, hd)).astype(np.float32)
    dev, starts = Dev(rai), _starts(news)
    pg, batch = dev.pages(pool), dev.batch(pool, starts, lengths, tokens, max(news), max(lengths))
    opts = rai.AttentionOptions(hd ** -0.5, 0.0, 0, None)
    assert not split or rai.attention_workspace(heads, pg, batch, opts) > 0
    got = _run_attention(rai, dev, pg, batch, q, heads, hd, opts, work=None if split else 0)
    want = np.concatenate([attend(pool, 0, (int(a), m, n), s, q, heads, hd ** -0.5)[0]
                           for s, (a, m, n) in enumerate(zip(starts, news, lengths))])
    total, row = off_by(got, want)
    assert total <= ACCURATE and row <= 2 * ACCURATE, (total, row)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("nq", [1, 40])
def test_attention_of_a_wide_range(rai, cache, nq):
    """A query element of 2^30 that meets zeros beside normal ones, and a key of weight 2^-29 that alone has
    values in one dimension: f32's accuracy, or with f16 what the header says."""
    heads, hd, n, scale = 4, 64, 200, 0.125
    pool = Pool(cache, 16, 1, hd, [n], seed=12)
    pool.fill(0, [n])
    q = np.random.default_rng(3).standard_normal((nq, heads, hd)).astype(np.float32)
    q[:, :, 5], q[:, :, 9] = 2.0 ** 30, 8.0
    for p in range(n):
        pg, slot = pool.place(0, p)
        pool.k[0, pg, :, slot, 5] = encode(np.float32([0.0]), cache)[0]
        pool.v[0, pg, :, 7, slot] = encode(np.float32([1.0 if p == 3 else 0.0]), cache)[0]
        pool.k[0, pg, :, slot, 9] = encode(np.float32([-20.0 if p == 3 else 0.0]), cache)[0]
    want, tol = attend(pool, 0, (0, nq, n), 0, q, heads, scale)
    if cache == "f16":
        k, v, _ = pool.rows(0, 0, np.arange(n))
        for j in range(nq):
            seen = n - nq + j + 1
            kk, vv = np.abs(k[:seen, 0]), np.abs(v[:seen, 0])
            for h in range(heads):
                s = k[:seen, 0] @ q[j, h].astype(np.float64) * scale
                w = np.exp(s - s.max())
                x = np.abs(q[j, h].astype(np.float64))
                off = kk @ np.maximum(2.0 ** -22 * x, 2.0 ** -39 * x.max()) * scale
                tol[j, h] += (w / w.sum() * np.expm1(2 * off.max())) @ vv + np.maximum(2.0 ** -22 * w, 2.0 ** -39) / w.sum() @ vv
    dev = Dev(rai)
    pg, batch = dev.pages(pool), dev.batch(pool, [0, nq], [n], nq, nq, n)
    got = _run_attention(rai, dev, pg, batch, q, heads, hd, rai.AttentionOptions(scale, 0.0, 0, None))
    assert (np.abs(got - want) <= tol).all()


def test_attention_calls_on_two_streams_and_in_a_graph(rai):
    """Two calls in flight with scratch of their own; a captured call replayed on new lengths and queries."""
    L, P, heads, hd = rai.lib(), ctypes.c_void_p, 8, 64
    lengths = [1500, 900, 40]
    pool = Pool("bf16", 32, 2, hd, lengths, seed=8)
    pool.fill(0, lengths)
    dev = Dev(rai)
    pg = dev.pages(pool)
    tables, starts = dev.up(pool.tables), dev.up(np.int32([0, 1, 3, 4]))
    opts = rai.AttentionOptions(0.125, 0.0, 0, None)
    rng = np.random.default_rng(0)
    lens = [np.int32([1500, 900, 40]), np.int32([700, 2, 39]), np.int32([33, 800, 1])]
    qs = [rng.standard_normal((4, heads, hd)).astype(np.float32) for _ in lens]

    def call(dl, dq, do, dw, n, stream):
        batch = rai.PageBatch(tables.ptr, pool.tables.shape[1], starts.ptr, dl.ptr, 3, 4, 2, 1500)
        rai._check(L.rai_paged_attention_dev(do.ptr, heads * hd, dq.ptr, heads * hd, heads, pg, 0, batch, opts, dw.ptr,
                                             n, stream))

    batch = rai.PageBatch(tables.ptr, pool.tables.shape[1], starts.ptr, starts.ptr, 3, 4, 2, 1500)
    n = rai.attention_workspace(heads, pg, batch, opts)
    sets = [(dev.up(l), dev.up(q), dev.up(np.zeros_like(q)), rai.DeviceArray(max(n, 16))) for l, q in zip(lens, qs)]
    want = []
    for s in sets:
        call(*s, n, None)
        rai._check(L.rai_device_synchronize())
        want.append(s[2].to_host(np.float32, 4 * heads * hd))
    for (l, q, w) in zip(lens, qs, want):  # and those are right
        for i, sp in enumerate(spans([0, 1, 3, 4], l, 4, 2, 1500)):
            r, tol = attend(pool, 0, sp, i, q, heads, 0.125)
            assert (np.abs(w.reshape(4, heads, hd)[sp[0]:sp[0] + sp[1]] - r) <= tol).all()
    streams = [P(), P()]
    for s in streams:
        rai._check(L.rai_stream_create(ctypes.byref(s)))
    for _ in range(3):
        for s in sets:
            rai._check(L.rai_memcpy_h2d(s[2].ptr, np.zeros(4 * heads * hd, np.float32).ctypes.data, 16 * heads * hd))
        for s, st in zip(sets, [streams[0], streams[1], streams[0]]):
            call(*s, n, st)
        rai._check(L.rai_device_synchronize())
        for s, w in zip(sets, want):
            assert np.array_equal(s[2].to_host(np.float32, 4 * heads * hd).view(np.uint32), w.view(np.uint32))
    graph, ex = P(), P()
    gc.collect()
    gc.disable()
    try:
        assert L.hipStreamBeginCapture(streams[0], 1) == 0
        call(*sets[0], n, streams[0])
        assert L.hipStreamEndCapture(streams[0], ctypes.byref(graph)) == 0
    finally:
        gc.enable()
    assert L.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in (1, 2, 0, 1):
        rai._check(L.rai_memcpy_h2d(sets[0][0].ptr, lens[i].ctypes.data, 12))
        rai._check(L.rai_memcpy_h2d(sets[0][1].ptr, qs[i].ctypes.data, qs[i].nbytes))
        assert L.hipGraphLaunch(ex, streams[0]) == 0
        rai._check(L.rai_stream_synchronize(streams[0]))
        assert np.array_equal(sets[0][2].to_host(np.float32, 4 * heads * hd).view(np.uint32), want[i].view(np.uint32))
        call(*sets[1], n, None)
        rai._check(L.rai_device_synchronize())
    assert L.hipGraphExecDestroy(ex) == 0 and L.hipGraphDestroy(graph) == 0
    for s in streams:
        rai._check(L.rai_stream_destroy(s))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("news,lengths", [([1], [1]), ([1, 2], [0, 0]), ([3, 200], [0, 0])])
def test_attention_nothing_cached(rai, cache, news, lengths):
    """Lengths of zero and one; a table of one page."""
    pool = Pool(cache, 16, 1, 64, lengths, seed=1)
    pool.fill(0, lengths)
    _check_attention(rai, pool, news, lengths, 2, 0.125)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("nq", [1, 5, 9, 40])
def test_attention_many_heads_on_one(rai, cache, nq):
    """70 query heads on a kv head: one token is more rows than the kernel of few rows takes."""
    pool = Pool(cache, 32, 1, 64, [300, 90], seed=2)
    pool.fill(0, [300, 90])
    _check_attention(rai, pool, [nq, 1], [300, 90], 70, 0.125)


@pytest.mark.parametrize("cache", ["f32", "bf16"])
@pytest.mark.parametrize("nq,n", [(1, 900), (70, 900)])
def test_attention_values_near_the_type_s_largest(rai, cache, nq, n):
    """Means of values near 3e38 stay finite, split or not."""
    pool = Pool(cache, 16, 1, 64, [n], seed=3)
    pool.fill(0, [n])
    top = encode(np.float32([3e38]), cache)[0]
    pool.v[:, pool.tables[0]] = top
    pool.v[:, pool.tables[0], :, ::2] = encode(np.float32([-3e38]), cache)[0]
    want = decode(np.array([top]), cache)[0]
    dev, q = Dev(rai), np.random.default_rng(1).standard_normal((nq, 4, 64)).astype(np.float32)
    pg, batch = dev.pages(pool), dev.batch(pool, [0, nq], [n], nq, nq, n)
    for work in (None, 0):
        got = _run_attention(rai, dev, pg, batch, q, 4, 64, rai.AttentionOptions(0.125, 0.0, 0, None), work=work)
        # The weights' sum is off by a half step a key at most, and so is their weighted sum.
        assert (np.abs(got[:, :, 1::2].astype(np.float64) / want - 1) <= 2 * (n + 16) * EPS32).all()
        assert (np.abs(got[:, :, ::2].astype(np.float64) / -want - 1) <= 2 * (n + 16) * EPS32).all()


@pytest.mark.parametrize("cache", CACHES)
def test_chunk_attention_in_a_graph(rai, cache):
    """A chunk's kernels, their scratch and more than 64 KB of LDS captured; replays on other queries with
    eager calls between them."""
    L, P, heads, hd, nq, n = rai.lib(), ctypes.c_void_p, 4, 128, 70, 1300
    pool = Pool(cache, 64, 2, hd, [n], seed=9)
    pool.fill(0, [n])
    dev, rng = Dev(rai), np.random.default_rng(0)
    pg, batch = dev.pages(pool), dev.batch(pool, [0, nq], [n], nq, nq, n)
    opts = rai.AttentionOptions(0.1, 0.0, 0, None)
    qs = [rng.standard_normal((nq, heads, hd)).astype(np.float32) for _ in range(3)]
    size = rai.attention_workspace(heads, pg, batch, opts)
    dq, do, dw = dev.up(qs[0]), dev.up(np.zeros_like(qs[0])), rai.DeviceArray(max(size, 16))
    stream, graph, ex = P(), P(), P()
    rai._check(L.rai_stream_create(ctypes.byref(stream)))
    gc.collect()
    gc.disable()
    try:
        assert L.hipStreamBeginCapture(stream, 1) == 0
        rc = L.rai_paged_attention_dev(do.ptr, heads * hd, dq.ptr, heads * hd, heads, pg, 0, batch, opts, dw.ptr, size,
                                       stream)
        assert L.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    finally:
        gc.enable()
    rai._check(rc)
    assert L.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in (0, 1, 2, 0):
        want, tol = attend(pool, 0, (0, nq, n), 0, qs[i], heads, 0.1)
        rai._check(L.rai_memcpy_h2d(dq.ptr, qs[i].ctypes.data, qs[i].nbytes))
        assert L.hipGraphLaunch(ex, stream) == 0
        rai._check(L.rai_stream_synchronize(stream))
        got = do.to_host(np.float32, qs[i].size).reshape(qs[i].shape)
        assert (np.abs(got - want) <= tol).all()
        eager = _run_attention(rai, dev, pg, batch, qs[i], heads, hd, opts)
        assert np.array_equal(eager.view(np.uint32), got.view(np.uint32))
    assert L.hipGraphExecDestroy(ex) == 0 and L.hipGraphDestroy(graph) == 0
    rai._check(L.rai_stream_destroy(stream))


def test_offsets_past_32_bits(rai):
    """Pages whose elements lie past 2^32 of the pool: stored, attended, forked and moved there."""
    heads, kv_heads, hd, page, n, high = 4, 2, 64, 64, 150, (1 << 32) // (2 * 64 * 64) + 3
    small = Pool("bf16", page, kv_heads, hd, [n], seed=4)
    rng = np.random.default_rng(6)
    k, v = rng.standard_normal((2, n, kv_heads * hd)).astype(np.float32)
    q = rng.standard_normal((n, heads, hd)).astype(np.float32)
    for p in range(n):
        small.put(0, 0, p, k[p].reshape(kv_heads, hd), v[p].reshape(kv_heads, hd))
    count = high + 8
    dk, dv = (rai.DeviceArray(2 * count * kv_heads * page * hd) for _ in range(2))
    pg = rai.Pages(dk.ptr, dv.ptr, 1, count, page, kv_heads, hd, rai.CACHE_BF16)
    dev, L = Dev(rai), rai.lib()
    tables = dev.up(np.int32([[high, high + 2, high + 1]]))
    batch = rai.PageBatch(tables.ptr, 3, dev.up(np.int32([0, n])).ptr, dev.up(np.int32([n])).ptr, 1, n, n, n)
    rai._check(L.rai_paged_store_dev(pg, 0, batch, None, None, 0, None, 0, 0, dev.up(k).ptr, kv_heads * hd, dev.up(v).ptr,
                                     kv_heads * hd, None))
    opts = rai.AttentionOptions(0.125, 0.0, 0, None)
    want, tol = attend(small, 0, (0, n, n), 0, q, heads, 0.125)
    got = _run_attention(rai, dev, pg, batch, q, heads, hd, opts)
    assert (np.abs(got - want) <= tol).all()
    # Two children of a sequence of 150 positions, the second's last page to high + 5, then that to high + 7.
    out = [dev.up(np.zeros(m, np.int32)) for m in (6, 2, 2)]
    rai._check(L.rai_paged_fork_dev(pg, tables.ptr, 3, dev.up(np.int32([n])).ptr, 1, dev.up(np.int32([0, 0])).ptr,
                                    dev.up(np.int32([high + 4, high + 5])).ptr, 2, *[o.ptr for o in out], None))
    rai._check(L.rai_paged_move_dev(pg, dev.up(np.int32([high + 5])).ptr, dev.up(np.int32([high + 7])).ptr, 1, out[0].ptr,
                                    6, None))
    rai._check(L.rai_device_synchronize())
    assert out[0].to_host(np.int32, 6).tolist() == [high, high + 2, high + 1, high, high + 2, high + 7]
    for nq in (1, n):
        two = rai.PageBatch(out[0].ptr, 3, dev.up(np.int32([0, nq, 2 * nq])).ptr, out[1].ptr, 2, 2 * nq, nq, n)
        got = _run_attention(rai, dev, pg, two, np.concatenate([q[n - nq:]] * 2), heads, hd, opts)
        for half in (got[:nq], got[nq:]):
            assert (np.abs(half - want[n - nq:]) <= tol[n - nq:]).all()


# ------------------------------------------------------------------- store --

def _check_store(rai, cache, page, heads, kv_heads, hd, news, lengths, rot, interleaved, gain=1.0, front=0, back=0,
                 in_place=False, inv=None, pool=None, q_start=None, max_q=None, max_kv=None, extra=5):
    pool = pool or Pool(cache, page, kv_heads, hd, lengths, seed=hd + len(news), layers=2)
    dev, rng, tokens = Dev(rai), np.random.default_rng(hd), front + sum(news) + back
    q_start = _starts(news, front) if q_start is None else q_start
    max_q = max(news) if max_q is None else max_q
    max_kv = max(lengths) if max_kv is None else max_kv
    inv = 1e4 ** (-2.0 * np.arange(rot // 2) / rot) if inv is None and rot else inv
    wide, kw = heads * hd, kv_heads * hd
    q, k, v = (rng.standard_normal((tokens, n + e)).astype(np.float32) for n, e in ((wide, extra), (kw, extra + 2), (kw, 0)))
    pg, batch = dev.pages(pool), dev.batch(pool, q_start, lengths, tokens, max_q, max_kv)
    dq = dev.up(q)
    do = dq if in_place else dev.up(np.full((tokens, wide + 3), SENTINEL, np.float32))
    o_ld = q.shape[1] if in_place else wide + 3
    rope = rai.Rope(dev.up(np.asarray(inv, np.float64)).ptr, rot, interleaved, gain) if rot else None
    rai._check(rai.lib().rai_paged_store_dev(pg, 1, batch, rope, do.ptr, o_ld, dq.ptr, q.shape[1], heads,
                                             dev.up(k).ptr, k.shape[1], dev.up(v).ptr, v.shape[1], None))
    rai._check(rai.lib().rai_device_synchronize())
    got_q = do.to_host(np.float32, tokens * o_ld).reshape(tokens, o_ld)
    gk, gv = dev.pool_back(pool)
    want_k, want_v = decode(pool.k, cache).astype(np.float64), decode(pool.v, cache).astype(np.float64)
    mag = np.zeros_like(want_k)  # magnitude of what was rotated, for the bound
    cut = spans(q_start, lengths, tokens, max_q, min(max_kv, pool.tables.shape[1] * pool.page))
    mine = _claims(cut, tokens)
    for s, (q0, nq, n) in enumerate(cut):
        for j in range(nq):
            pos, r = n - nq + j, q0 + j
            turn = lambda x, h: rotate(x.reshape(h, hd), pos, inv, rot, interleaved, gain) if rot else np.float64(x.reshape(h, hd))
            # Each of the two products of a rotation: the half steps of the function's value (a few), of
            # the gain, the product and the sum.
            if heads and mine[r] == 1:
                w = turn(q[r, :wide], heads)
                tol = 8 * EPS32 * 2 * gain * np.abs(q[r, :wide]).max()
                assert (np.abs(got_q[r, :wide].reshape(heads, hd) - w) <= tol).all(), (s, j)
            where = pool.place(s, pos)
            if where:
                want_k[1, where[0], :, where[1]] = turn(k[r, :kw], kv_heads)
                mag[1, where[0], :, where[1]] = np.abs(k[r, :kw]).max() * max(gain, 1.0)
                want_v[1, where[0], :, :, where[1]] = decode(encode(v[r], cache), cache).reshape(kv_heads, hd)
    step = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[cache]
    tiny = 2.0 ** -25 if cache == "f16" else 0.0  # half a step of f16's subnormals
    with np.errstate(invalid="ignore"):
        far = np.abs(decode(gk, cache) - want_k)
        near = far <= (1 + step) * 16 * EPS32 * mag + step * np.abs(want_k) + tiny
    assert (near | (np.isnan(want_k) & np.isnan(decode(gk, cache)))).all()
    assert np.array_equal(decode(gv, cache), want_v, equal_nan=True)
    if not in_place:
        assert (got_q[:, wide:] == SENTINEL).all()
        if heads:
            assert (got_q[mine == 0] == SENTINEL).all()
    else:
        assert np.array_equal(got_q[mine == 0], q[mine == 0]) and np.array_equal(got_q[:, wide:], q[:, wide:])


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,kv_heads,hd,rot", [(4, 2, 64, 64), (32, 8, 128, 128), (3, 1, 80, 32), (5, 5, 8, 2),
                                                   (2, 1, 256, 96), (0, 2, 64, 64), (4, 4, 96, 0)])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("news,lengths", BATCHES)
def test_store(rai, cache, heads, kv_heads, hd, rot, interleaved, news, lengths):
    page = 16 << (heads + len(news)) % 4
    _check_store(rai, cache, page, heads, kv_heads, hd, news, lengths, rot, interleaved, gain=1.0 + 0.25 * interleaved,
                 front=heads % 2, back=2, in_place=(heads + len(news)) % 2 == 1 and heads > 0)


@pytest.mark.parametrize("news,lengths", [([1, 1], [20001, 1000001]), ([100, 300], [131072, 40000])])
def test_store_far_positions(rai, news, lengths):
    """Angles of positions up to a million, where an f32 product would be off by 0.06."""
    inv, gain = rai.rope_frequencies(rai.ROPE_LLAMA3, 5e5, 64, 8.0)
    _check_store(rai, "f32", 1024, 4, 2, 64, news, lengths, 64, 0, gain=gain, inv=inv)


@pytest.mark.parametrize("cache", CACHES)
def test_store_bad_entries(rai, cache):
    lengths = [40, 70, 90]
    pool = Pool(cache, 16, 2, 64, lengths, seed=1, layers=2)
    pool.tables[0, 2], pool.tables[1, :], pool.tables[2, 4] = pool.pages, -1, -(1 << 31)
    _check_store(rai, cache, 16, 4, 2, 64, [20, 10, 50], lengths, 64, 0, pool=pool)
    _check_store(rai, cache, 16, 4, 2, 64, [20, 10, 50], [40, 10 ** 9, -3], 64, 0, pool=pool, max_kv=65)
    _check_store(rai, cache, 16, 4, 2, 64, [20, 10, 50], lengths, 64, 0, pool=pool, q_start=[-9, 25, 20, 10 ** 9], max_q=30)


@pytest.mark.parametrize("cache", ["f16", "bf16"])
def test_store_rounds_as_the_type(rai, cache):
    """Ties, overflow, subnormals and non-finite values reach the cache as one rounding to nearest even gives them."""
    hd = 64
    v = np.zeros((16, hd), np.float32)
    if cache == "f16":
        v[:, :10] = [2049.0, 2051.0, 65519.0, 65520.0, 1e-8, 2.0 ** -25, 3 * 2.0 ** -25, np.inf, -np.inf, np.nan]
    else:
        v[:, :10] = [257.0, 259.0, 3.3895e38, 3.4028e38, 1e-40, 1.00390625, 1.01171875, np.inf, -np.inf, np.nan]
    pool = Pool(cache, 16, 1, hd, [16], seed=1)
    dev = Dev(rai)
    pg, batch = dev.pages(pool), dev.batch(pool, [0, 16], [16], 16, 16, 16)
    dv = dev.up(v)
    rai._check(rai.lib().rai_paged_store_dev(pg, 0, batch, None, None, 0, None, 0, 0, dv.ptr, hd, dv.ptr, hd, None))
    rai._check(rai.lib().rai_device_synchronize())
    gk, gv = dev.pool_back(pool)
    want = decode(encode(v, cache), cache)
    p = pool.tables[0, 0]
    assert np.array_equal(decode(gk[0, p, 0], cache), want, equal_nan=True)
    assert np.array_equal(decode(gv[0, p, 0], cache), want.T, equal_nan=True)


# --------------------------------------------------------- forks and moves --

def _random_pool(cache, page, kv_heads, hd, lengths, layers, spare, seed=0):
    pool = Pool(cache, page, kv_heads, hd, lengths, seed=seed, layers=layers, spare=spare)
    r = np.random.default_rng(seed)
    for a in (pool.k, pool.v):
        a[...] = r.integers(0, 30000, a.shape).astype(a.dtype)
    return pool


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("page,kv_heads,hd,layers", [(16, 1, 8, 1), (64, 2, 128, 3), (128, 3, 72, 2)])
def test_fork(rai, cache, page, kv_heads, hd, layers):
    lengths = [page * 3, page + 5, 1, 0, 2 * page - 1]
    parent = np.int32([0, 1, 1, 1, 2, 2, 3, 3, -1, 5, 4, 0, 1, 4])
    n = len(parent)
    pool = _random_pool(cache, page, kv_heads, hd, lengths, layers, n)
    fresh = np.int32(pool.spare[:n])
    fresh[5] = pool.pages  # none for the second child of sequence 2
    dev = Dev(rai)
    pg, (seqs, stride) = dev.pages(pool), pool.tables.shape
    out = [dev.up(np.full(m, 77, np.int32)) for m in (n * stride, n, n)]
    for _ in range(2):
        rai._check(rai.lib().rai_paged_fork_dev(pg, dev.up(pool.tables).ptr, stride, dev.up(np.int32(lengths)).ptr, seqs,
                                                dev.up(parent).ptr, dev.up(fresh).ptr, n, *[o.ptr for o in out], None))
    rai._check(rai.lib().rai_device_synchronize())
    tables, length, used = (o.to_host(np.int32, m) for o, m in zip(out, (n * stride, n, n)))
    k, v = pool.k.copy(), pool.v.copy()
    for i, p in enumerate(parent):
        if not 0 <= p < seqs:
            assert length[i] == 0 and used[i] == 0 and (tables.reshape(n, -1)[i] == -1).all()
            continue
        row = pool.tables[p].copy()
        take = lengths[p] % page != 0 and p in parent[:i]
        if take:
            f = fresh[i] if fresh[i] < pool.pages else -1
            if f >= 0:
                k[:, f], v[:, f] = pool.k[:, row[lengths[p] // page]], pool.v[:, row[lengths[p] // page]]
            row[lengths[p] // page] = f
        assert np.array_equal(tables.reshape(n, -1)[i], row), i
        assert length[i] == lengths[p] and used[i] == (take and fresh[i] < pool.pages)
    gk, gv = dev.pool_back(pool)
    assert np.array_equal(gk, k) and np.array_equal(gv, v)


def test_fork_bad_entries(rai):
    """Lengths past the table and pages that are not there: no copy."""
    pool = _random_pool("f32", 16, 1, 8, [40, 40], 2, 4)
    pool.tables[1, 2] = -3
    dev = Dev(rai)
    pg, parent, fresh = dev.pages(pool), np.int32([0, 0, 1, 1]), np.int32(pool.spare[:4])
    out = [dev.up(np.zeros(m, np.int32)) for m in (12, 4, 4)]
    rai._check(rai.lib().rai_paged_fork_dev(pg, dev.up(pool.tables).ptr, 3, dev.up(np.int32([10 ** 9, 40])).ptr, 2,
                                            dev.up(parent).ptr, dev.up(fresh).ptr, 4, *[o.ptr for o in out], None))
    rai._check(rai.lib().rai_device_synchronize())
    assert out[1].to_host(np.int32, 4).tolist() == [48, 48, 40, 40]
    t = out[0].to_host(np.int32, 12).reshape(4, 3)
    assert np.array_equal(t[:2], pool.tables[[0, 0]]) and np.array_equal(t[2], pool.tables[1])
    assert t[3].tolist() == pool.tables[1, :2].tolist() + [fresh[3]] and out[2].to_host(np.int32, 4).tolist() == [0, 0, 0, 1]
    gk, gv = dev.pool_back(pool)
    assert np.array_equal(gk, pool.k) and np.array_equal(gv, pool.v)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("missing", [-1, -3, "pages", 1 << 30])
def test_fork_of_a_last_page_that_is_not_there(rai, cache, missing):
    """No child sees a key there, and no fresh page is taken: it holds what another sequence left in it."""
    heads, hd, lengths, parent = 4, 64, [40, 40, 21], np.int32([1, 0, 1, 0, 1, 2, 2])
    n = len(parent)
    pool = Pool(cache, 16, 2, hd, lengths, seed=9, layers=2, spare=n)
    for layer in (0, 1):
        pool.fill(layer, lengths)
    for page in pool.spare:  # as another sequence left them
        pool.tables[2, 2] = page
        for layer in (0, 1):
            for p in range(32, 48):
                pool.put(layer, 2, p, *pool.rng.standard_normal((2, 2, hd)))
    pool.tables[1, 2], pool.tables[2, 2] = pool.pages if missing == "pages" else missing, -1
    dev = Dev(rai)
    pg, fresh = dev.pages(pool), np.int32(pool.spare)
    out = [dev.up(np.full(m, 77, np.int32)) for m in (3 * n, n, n)]
    rai._check(rai.lib().rai_paged_fork_dev(pg, dev.up(pool.tables).ptr, 3, dev.up(np.int32(lengths)).ptr, 3,
                                            dev.up(parent).ptr, dev.up(fresh).ptr, n, *[o.ptr for o in out], None))
    rai._check(rai.lib().rai_device_synchronize())
    tables, length, used = (o.to_host(np.int32, m) for o, m in zip(out, (3 * n, n, n)))
    tables = tables.reshape(n, 3)
    # Children 3 and 6 are the later ones of parents whose last page is there.
    assert used.tolist() == [0, 0, 0, 1, 0, 0, 1] and length.tolist() == [lengths[p] for p in parent]
    want = pool.tables[parent].copy()
    want[3, 2], want[6, 1] = fresh[3], fresh[6]
    assert np.array_equal(tables, want)
    k, v = pool.k.copy(), pool.v.copy()
    for child, last in ((3, 2), (6, 1)):
        src = pool.tables[parent[child], last]
        k[:, fresh[child]], v[:, fresh[child]] = pool.k[:, src], pool.v[:, src]
    gk, gv = dev.pool_back(pool)
    for got, copied in ((gk, k), (gv, v)):
        assert np.array_equal(got.view(np.uint8), copied.view(np.uint8))
    # Attention over a child is attention over its parent.
    q = np.random.default_rng(1).standard_normal((n, heads, hd)).astype(np.float32)
    opts = rai.AttentionOptions(hd ** -0.5, 0.0, 0, None)
    batch = rai.PageBatch(out[0].ptr, 3, dev.up(np.int32(np.arange(n + 1))).ptr, out[1].ptr, n, n, 1, 40)
    got = _run_attention(rai, dev, pg, batch, q, heads, hd, opts, layer=1)
    for i, p in enumerate(parent):
        ref, tol = attend(pool, 1, (i, 1, lengths[p]), p, q, heads, hd ** -0.5)
        assert (np.abs(got[i] - ref[0]) <= tol[0]).all(), i


def test_fork_lengths_past_the_table(rai):
    """A length past the table becomes the table's: whole pages, shared by every child."""
    pool = _random_pool("f32", 16, 1, 8, [40, 40], 2, 4)
    dev = Dev(rai)
    pg, parent, fresh = dev.pages(pool), np.int32([0, 0, 1, 0]), np.int32(pool.spare[:4])
    out = [dev.up(np.zeros(m, np.int32)) for m in (12, 4, 4)]
    rai._check(rai.lib().rai_paged_fork_dev(pg, dev.up(pool.tables).ptr, 3, dev.up(np.int32([10 ** 9, -5])).ptr, 2,
                                            dev.up(parent).ptr, dev.up(fresh).ptr, 4, *[o.ptr for o in out], None))
    rai._check(rai.lib().rai_device_synchronize())
    assert out[1].to_host(np.int32, 4).tolist() == [48, 48, 0, 48] and not out[2].to_host(np.int32, 4).any()
    assert np.array_equal(out[0].to_host(np.int32, 12).reshape(4, 3), pool.tables[parent])
    gk, gv = dev.pool_back(pool)
    assert np.array_equal(gk, pool.k) and np.array_equal(gv, pool.v)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("page,kv_heads,hd,layers,n,entries", [(16, 1, 8, 1, 1, 0), (64, 2, 128, 2, 9, 40),
                                                              (32, 3, 72, 3, 300, 5000)])
def test_move(rai, cache, page, kv_heads, hd, layers, n, entries):
    pool = _random_pool(cache, page, kv_heads, hd, [1], layers, 2 * n + 8)
    ids = np.random.default_rng(n).permutation(pool.pages).astype(np.int32)
    src, dst = ids[:n].copy(), ids[n:2 * n].copy()
    tables = np.random.default_rng(1).integers(-2, pool.pages + 2, entries).astype(np.int32)
    if n > 4:
        src[2], dst[4] = -1, pool.pages  # left out
    dev = Dev(rai)
    pg = dev.pages(pool)
    dt = dev.up(tables) if entries else None
    rai._check(rai.lib().rai_paged_move_dev(pg, dev.up(src).ptr, dev.up(dst).ptr, n, dt.ptr if dt else None, entries, None))
    rai._check(rai.lib().rai_device_synchronize())
    k, v, name = pool.k.copy(), pool.v.copy(), {}
    for a, b in zip(src, dst):
        if 0 <= a < pool.pages and 0 <= b < pool.pages:
            k[:, b], v[:, b], name[a] = pool.k[:, a], pool.v[:, a], b
    gk, gv = dev.pool_back(pool)
    assert np.array_equal(gk, k) and np.array_equal(gv, v)
    if entries:
        assert dt.to_host(np.int32, entries).tolist() == [name.get(t, t) for t in tables]


@pytest.mark.parametrize("n,entries", [(2100, 70001), (4096, 65536), (65535, 3)])
def test_move_many(rai, n, entries):
    """More pairs than are looked through in one go, more table entries than the launch has threads."""
    pool = _random_pool("f16", 16, 1, 8, [1], 1, 2 * n + 8)
    r = np.random.default_rng(n)
    ids = r.permutation(pool.pages).astype(np.int32)
    src, dst = ids[:n].copy(), ids[n:2 * n].copy()
    src[n // 2], dst[n - 2] = pool.pages, -1  # left out
    tables = r.integers(-2, pool.pages + 2, entries).astype(np.int32)
    tables[-3:] = src[0], src[n - 1], src[n - 2]
    dev = Dev(rai)
    pg, dt = dev.pages(pool), dev.up(tables)
    rai._check(rai.lib().rai_paged_move_dev(pg, dev.up(src).ptr, dev.up(dst).ptr, n, dt.ptr, entries, None))
    rai._check(rai.lib().rai_device_synchronize())
    ok = (src < pool.pages) & (dst >= 0)
    k, v, name = pool.k.copy(), pool.v.copy(), np.arange(-2, pool.pages + 2)
    k[:, dst[ok]], v[:, dst[ok]], name[src[ok] + 2] = pool.k[:, src[ok]], pool.v[:, src[ok]], dst[ok]
    gk, gv = dev.pool_back(pool)
    assert np.array_equal(gk.view(np.uint16), k.view(np.uint16)) and np.array_equal(gv.view(np.uint16), v.view(np.uint16))
    assert np.array_equal(dt.to_host(np.int32, entries), name[tables + 2])


def test_move_of_the_largest_launch(rai):
    """65535 pairs x 128 layers, one below the limit of pages x layers; all but the first and last left out."""
    n, pool = 65535, _random_pool("f16", 16, 1, 8, [1], 128, 7)
    src, dst = np.full(n, -1, np.int32), np.full(n, -1, np.int32)
    (src[0], src[-1]), (dst[0], dst[-1]) = pool.spare[:2], pool.spare[2:4]
    dev = Dev(rai)
    pg = dev.pages(pool)
    rai._check(rai.lib().rai_paged_move_dev(pg, dev.up(src).ptr, dev.up(dst).ptr, n, None, 0, None))
    rai._check(rai.lib().rai_device_synchronize())
    k, v = pool.k.copy(), pool.v.copy()
    k[:, pool.spare[2:4]], v[:, pool.spare[2:4]] = pool.k[:, pool.spare[:2]], pool.v[:, pool.spare[:2]]
    gk, gv = dev.pool_back(pool)
    assert np.array_equal(gk.view(np.uint16), k.view(np.uint16)) and np.array_equal(gv.view(np.uint16), v.view(np.uint16))


# -------------------------------------------------------------------- beam --

def _select(x, scores, done, end, beams, take):
    """By the definition: (parent, token, score in f64) of each group."""
    rows, vocab = x.shape
    out = []
    for g in range(rows // beams):
        cand = []
        for b in range(beams):
            r = g * beams + b
            base = float(scores[r])
            if not base > -np.inf:
                continue
            if done is not None and done[r]:
                cand += [(-base, r, 0.0, end)]
                continue
            v = np.where(np.isnan(x[r]), -np.inf, x[r].astype(np.float64))
            top = v.max()
            if not np.isfinite(top):
                continue
            t = base + (v - top - np.log(np.exp(v - top).sum()))  # a large top would swallow the logarithm
            best = np.lexsort((np.arange(vocab), -v))[:take]
            cand += [(-t[i], r, -v[i], int(i)) for i in best if v[i] > -np.inf]
        cand = sorted(cand)[:take]
        out += [(c[1], c[3], -c[0]) for c in cand] + [(-1, -1, -np.inf)] * (take - len(cand))
    return [np.array(a) for a in zip(*out)]


def _check_beam(rai, x, scores, done, end, beams, take, extra=0):
    dev, (rows, vocab) = Dev(rai), x.shape
    groups = rows // beams
    wide = np.full((rows, vocab + extra), np.nan if extra % 2 else np.inf, np.float32)
    wide[:, :vocab] = x
    n, need = groups * take, rai.beam_workspace(vocab, groups, beams, take)
    outs = [dev.up(np.full(n + 1, 99, t)) for t in (np.int32, np.int32, np.float32)]
    work = dev.up(np.full(need // 4 + 17, np.nan, np.float32))
    rai._check(rai.lib().rai_beam_select_dev(dev.up(wide).ptr, vocab + extra, vocab, dev.up(np.float32(scores)).ptr,
                                             None if done is None else dev.up(np.uint8(done)).ptr, end, groups, beams,
                                             take, *[o.ptr for o in outs], work.ptr, need, None))
    rai._check(rai.lib().rai_device_synchronize())
    assert np.isnan(work.to_host(np.float32, need // 4 + 17)[-(-need // 4):]).all()
    got = [o.to_host(t, n + 1) for o, t in zip(outs, (np.int32, np.int32, np.float32))]
    assert all(g[n] == 99 for g in got)
    parent, token, score = _select(x, scores, done, end, beams, take)
    assert np.array_equal(got[0][:n], parent) and np.array_equal(got[1][:n], token)
    ok = score > -np.inf
    # One rounding to f32; 1e-6 for the f32 exponentials in the log-sum (each within a few half steps).
    assert (np.abs(got[2][:n][ok] - score[ok]) <= EPS32 * np.abs(score[ok]) + 1e-6).all()
    assert (got[2][:n][~ok] == -np.inf).all()


def _normal(r, rows, vocab, std):
    """Random logits: two candidates of different beams within the rounding of a log-sum (1e-8) of each other
    are rarer than one in 10^5 selections."""
    return (std * r.standard_normal((rows, vocab))).astype(np.float32)


@pytest.mark.parametrize("groups,beams,vocab,take", [(1, 1, 1, 1), (1, 4, 32000, 8), (3, 2, 7, 14), (2, 5, 1000, 10),
                                                     (2, 3, 50304, 6), (5, 16, 300, 32), (1, 64, 129, 64),
                                                     (1, 1, 128256, 64), (7, 8, 4097, 16)])
@pytest.mark.parametrize("extra", [0, 3])
def test_beam(rai, groups, beams, vocab, take, extra):
    r = np.random.default_rng(vocab + take)
    x = _normal(r, groups * beams, vocab, 2.5)
    _check_beam(rai, x, -np.abs(3 * r.standard_normal(groups * beams)), None, 0, beams, take, extra)


@pytest.mark.parametrize("best", ["spread", "last beams", "one chunk"])
@pytest.mark.parametrize("take", [7, 64])
def test_beam_many_lists(rai, best, take):
    """64 beams of 38 chunks: more lists than the merge looks at in one go, so that the first places of some come
    after later places of others."""
    r = np.random.default_rng(take)
    vocab = 151936
    x = _normal(r, 64, vocab, 2.0)
    scores = -np.abs(3 * r.standard_normal(64))
    if best == "last beams":
        scores[:] = np.linspace(-40, -1, 64)
    if best == "one chunk":  # the best are the later places of the last list, behind everything else's first
        scores[:] = np.linspace(-9, -8, 64)
        x[63, vocab - 300:vocab - 300 + 2 * 80:2] = 14.0 + 0.01 * r.permutation(80)
    _check_beam(rai, x, scores, None, 0, 64, take)


@pytest.mark.parametrize("vocab,take", [(5, 8), (1000, 8), (20000, 20)])
def test_beam_finished(rai, vocab, take):
    r = np.random.default_rng(vocab)
    x = _normal(r, 24, vocab, 2.0)
    done = r.random(24) < 0.4
    done[:4] = True  # a group of finished beams: four candidates
    _check_beam(rai, x, -np.abs(r.standard_normal(24)), done, vocab - 2, 4, take)


@pytest.mark.parametrize("vocab", [3, 64, 5000, 40000])
def test_beam_ties(rai, vocab):
    """Equal logits (whole rows of one value, many repeated ones, zeros of both signs), equal rows and
    scores: by beam, then logit, then token."""
    r = np.random.default_rng(vocab)
    x = r.integers(-2, 3, (16, vocab)).astype(np.float32)
    x[4:8] = 1.5
    x[8:12] = x[8]
    x[12:16] = np.where(r.random((4, vocab)) < 0.5, 0.0, -0.0)
    x[13, vocab // 2], x[13, vocab - 1] = 1e-30, 2e-30  # differ as logits, not in the f64 score
    for take in (1, 8, 64):
        _check_beam(rai, x, np.zeros(16), None, 0, 4, take)


@pytest.mark.parametrize("vocab", [10, 3000])
def test_beam_nothing_to_choose(rai, vocab):
    """NaN, infinities, masks of the type's lowest value, empty rows, beams that are not in use."""
    r = np.random.default_rng(vocab)
    x = _normal(r, 24, vocab, 2.0)
    low = np.finfo(np.float32).min
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 3] = np.inf
    x[3, 1:] = -np.inf  # one token left
    x[4, ::2] = np.nan
    x[5, 1::2] = low
    x[6, 2:] = low
    x[7] = low
    x[8:12] = -np.inf
    scores = -np.abs(r.standard_normal(24))
    scores[13:16] = -np.inf  # the first step: one beam in use
    scores[16], scores[20:24] = np.nan, -np.inf
    _check_beam(rai, x, scores, None, 0, 4, 8)
    _check_beam(rai, x, scores, r.random(24) < 0.3, 1, 4, 8)


@pytest.mark.parametrize("every,at", [(64, 5), (2, 1), (16, 0)])
@pytest.mark.parametrize("take", [1, 16, 64])
def test_beam_masked_in_a_pattern(rai, every, at, take):
    """Masks that leave whole lanes of the selection empty, over chunks of which one is part filled."""
    r = np.random.default_rng(every)
    x = _normal(r, 4, 9001, 2.0)
    x[:, np.arange(9001) // 4 % every == at] = -np.inf
    x[1, 4096:] = -np.inf
    x[2] = np.sort(x[2])
    x[3] = -np.sort(-x[3])
    _check_beam(rai, x, np.float32([-1, -2, -1.5, -1.25]), None, 0, 2, take)


def test_beam_in_a_graph(rai):
    L, P = rai.lib(), ctypes.c_void_p
    groups, beams, vocab, take = 2, 4, 9000, 8
    dev, r, n = Dev(rai), np.random.default_rng(0), 16
    xs = [_normal(r, 8, vocab, 2.0) for _ in range(3)]
    scores = np.float32(-np.abs(r.standard_normal(8)))
    dx, ds, need = dev.up(xs[0]), dev.up(scores), rai.beam_workspace(vocab, groups, beams, take)
    outs, work = [rai.DeviceArray(4 * n) for _ in range(3)], rai.DeviceArray(need)
    stream, graph, ex = P(), P(), P()
    rai._check(L.rai_stream_create(ctypes.byref(stream)))
    gc.collect()
    gc.disable()
    try:
        assert L.hipStreamBeginCapture(stream, 1) == 0
        rc = L.rai_beam_select_dev(dx.ptr, vocab, vocab, ds.ptr, None, 0, groups, beams, take, *[o.ptr for o in outs],
                                   work.ptr, need, stream)
        assert L.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    finally:
        gc.enable()
    rai._check(rc)
    assert L.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0)) == 0
    for i in (0, 1, 2, 0):
        rai._check(L.rai_memcpy_h2d(dx.ptr, xs[i].ctypes.data, xs[i].nbytes))
        assert L.hipGraphLaunch(ex, stream) == 0
        rai._check(L.rai_stream_synchronize(stream))
        parent, token, _ = _select(xs[i], scores, None, 0, beams, take)
        assert np.array_equal(outs[0].to_host(np.int32, n), parent) and np.array_equal(outs[1].to_host(np.int32, n), token)
        _check_beam(rai, xs[(i + 1) % 3], scores, None, 0, beams, take)
    assert L.hipGraphExecDestroy(ex) == 0 and L.hipGraphDestroy(graph) == 0
    rai._check(L.rai_stream_destroy(stream))


# ---------------------------------------------------------------- together --

def test_a_step_in_a_graph(rai):
    """Selection, fork, store, attention and a move captured as one graph and replayed on other logits and
    rows, with eager runs of the same step on other buffers between the replays: equal bits."""
    L, P = rai.lib(), ctypes.c_void_p
    heads, kv_heads, hd, page, beams, vocab, n, stride = 8, 2, 64, 16, 4, 5000, 40, 4
    # No length ends a page: two children of such a sequence would share its last slot, which this step writes.
    lengths = [n, n - 3, n - 7, 5]
    rng = np.random.default_rng(3)
    inputs = [[a.astype(np.float32) for a in (2.0 * rng.standard_normal((beams, vocab)), rng.standard_normal((beams, heads * hd)),
                                              rng.standard_normal((2, beams, kv_heads * hd)))] for _ in range(3)]
    scores = np.float32([-1.0, -1.5, -0.5, -2.0])
    inv, gain = rai.rope_frequencies(rai.ROPE_NONE, 1e4, hd)
    options = rai.AttentionOptions(0.125, 0.0, 0, None)

    class Step:
        """Buffers of one step, and the calls."""

        def __init__(self):
            self.pool = Pool("f16", page, kv_heads, hd, lengths, seed=2, spare=20, stride=stride)
            self.pool.fill(0, lengths)
            self.dev = d = Dev(rai)
            self.pages = d.pages(self.pool)
            self.logits, self.q, self.kv = (d.up(a) for a in inputs[0])
            self.scores, self.inv = d.up(scores), d.up(inv)
            self.tables, self.lengths = d.up(self.pool.tables), d.up(np.int32(lengths))
            self.parent, self.token, self.score, self.next_len, self.used = (d.up(np.zeros(beams, np.int32)) for _ in range(5))
            self.fresh = d.up(np.int32(self.pool.spare[:beams]))
            self.next_tables, self.starts = d.up(np.zeros((beams, stride), np.int32)), d.up(np.int32(np.arange(beams + 1)))
            self.src, self.dst = d.up(np.int32(self.pool.spare[:1])), d.up(np.int32(self.pool.spare[beams:beams + 1]))
            self.out = d.up(np.zeros((beams, heads * hd), np.float32))
            self.batch = rai.PageBatch(self.next_tables.ptr, stride, self.starts.ptr, self.next_len.ptr, beams, beams, 1, n)
            self.need = rai.beam_workspace(vocab, 1, beams, beams)
            self.work = rai.DeviceArray(self.need)

        def give(self, values):
            for to, a in zip((self.logits, self.q, self.kv), values):
                rai._check(L.rai_memcpy_h2d(to.ptr, a.ctypes.data, a.nbytes))
            for to, a in zip((self.dev.k, self.dev.v), (self.pool.k, self.pool.v)):
                rai._check(L.rai_memcpy_h2d(to.ptr, a.ctypes.data, a.nbytes))

        def run(self, stream):
            rope, w, kw = rai.Rope(self.inv.ptr, hd, 0, gain), heads * hd, kv_heads * hd
            return [L.rai_beam_select_dev(self.logits.ptr, vocab, vocab, self.scores.ptr, None, 0, 1, beams, beams,
                                          self.parent.ptr, self.token.ptr, self.score.ptr, self.work.ptr, self.need, stream),
                    L.rai_paged_fork_dev(self.pages, self.tables.ptr, stride, self.lengths.ptr, beams, self.parent.ptr,
                                         self.fresh.ptr, beams, self.next_tables.ptr, self.next_len.ptr, self.used.ptr, stream),
                    L.rai_paged_store_dev(self.pages, 0, self.batch, rope, self.q.ptr, w, self.q.ptr, w, heads, self.kv.ptr,
                                          kw, self.kv.ptr + 4 * beams * kw, kw, stream),
                    L.rai_paged_move_dev(self.pages, self.src.ptr, self.dst.ptr, 1, self.next_tables.ptr, beams * stride, stream),
                    L.rai_paged_attention_dev(self.out.ptr, w, self.q.ptr, w, heads, self.pages, 0, self.batch, options, None,
                                              0, stream)]

        def results(self):
            rai._check(L.rai_device_synchronize())
            ints = [a.to_host(np.int32, beams) for a in (self.parent, self.token, self.next_len, self.used)]
            return ints + [self.next_tables.to_host(np.int32, beams * stride), self.out.to_host(np.uint32, beams * heads * hd),
                           *(a.view(np.uint16) for a in self.dev.pool_back(self.pool))]

    captured, eager = Step(), Step()
    stream, graph, ex = P(), P(), P()
    rai._check(L.rai_stream_create(ctypes.byref(stream)))
    gc.collect()
    gc.disable()
    try:
        assert L.hipStreamBeginCapture(stream, 1) == 0
        rcs = captured.run(stream)
        assert L.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    finally:
        gc.enable()
    assert rcs == [0] * 5, L.rai_last_error()
    assert L.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, ctypes.c_size_t(0)) == 0
    seen = []
    for i in (0, 1, 2, 0, 1):
        captured.give(inputs[i])
        eager.give(inputs[i])
        assert L.hipGraphLaunch(ex, stream) == 0
        rai._check(L.rai_stream_synchronize(stream))
        got = captured.results()
        assert eager.run(None) == [0] * 5
        for a, b in zip(got, eager.results()):
            assert np.array_equal(a, b)
        assert np.isfinite(got[5].view(np.float32)).all()
        seen.append(tuple(got[0]) + tuple(got[1]))
    assert len(set(seen)) == 3 and seen[0] == seen[3]
    assert L.hipGraphExecDestroy(ex) == 0 and L.hipGraphDestroy(graph) == 0
    rai._check(L.rai_stream_destroy(stream))


@pytest.mark.parametrize("cache", CACHES)
def test_an_attention_block_of_the_framework_s_calls(rai, ora, cache):
    """Norm, fused W4A8 projection, store (queries turned in place, in the projection's rows), attention and
    output projection on one stream, over two layers of pages: each stage from what the one before left."""
    from rai_amd.workload import gemv_operands
    L, heads, kv_heads, hd, gs, wide = rai.lib(), 4, 2, 64, 64, 256
    news, lengths, rows = [1, 9, 2], [40, 29, 2], (4 + 2 * 2) * 64
    tokens, starts = sum(news), _starts(news)
    pool = Pool(cache, 16, kv_heads, hd, lengths, seed=13, layers=2)
    for layer in (0, 1):
        pool.fill(layer, [n - m for m, n in zip(news, lengths)])
    dev, r = Dev(rai), np.random.default_rng(7)
    pg, batch = dev.pages(pool), dev.batch(pool, starts, lengths, tokens, max(news), max(lengths))
    inv, gain = rai.rope_frequencies(rai.ROPE_LLAMA3, 1e4, hd, 8.0, 32.0)
    rope, opts = rai.Rope(dev.up(inv).ptr, hd, 0, gain), rai.AttentionOptions(hd ** -0.5, 0.0, 0, None)
    x, weight = r.standard_normal((tokens, wide)).astype(np.float32), r.standard_normal(wide).astype(np.float32)
    need = rai.attention_workspace(heads, pg, batch, opts)
    dw, dx, dg = rai.DeviceArray(max(need, 16)), dev.up(x), dev.up(weight)
    for layer in (0, 1):
        qkv, proj = (gemv_operands(a, wide, 1, gs, seed=layer + a)[:2] for a in (rows, wide))
        dy, dq, da, do = (rai.DeviceArray(4 * tokens * n) for n in (wide, rows, wide, wide))
        base = dq.ptr
        weights = [dev.up(a).ptr for a in (*qkv, *proj)]
        rcs = [L.rai_rms_norm_dev(dy.ptr, dx.ptr, dg.ptr, tokens, wide, 1e-5, None),
               L.rai_w4a8_matmul_dev(dq.ptr, weights[0], weights[1], dy.ptr, rows, wide, tokens, gs, None)]
        rai._check(L.rai_device_synchronize())
        before = dq.to_host(np.float32, tokens * rows).reshape(tokens, rows)
        rcs += [L.rai_paged_store_dev(pg, layer, batch, rope, base, rows, base, rows, heads, base + 4 * heads * hd, rows,
                                      base + 4 * (heads + kv_heads) * hd, rows, None),
                L.rai_paged_attention_dev(da.ptr, wide, base, rows, heads, pg, layer, batch, opts, dw.ptr, need, None),
                L.rai_w4a8_matmul_dev(do.ptr, weights[2], weights[3], da.ptr, wide, wide, tokens, gs, None)]
        assert rcs == [0] * 5, L.rai_last_error()
        rai._check(L.rai_device_synchronize())
        y, after, att, out = (a.to_host(np.float32, tokens * n).reshape(tokens, n)
                              for a, n in ((dy, wide), (dq, rows), (da, wide), (do, wide)))
        assert np.array_equal(before.reshape(-1), ora.w4a8_matmul(*qkv, y, rows, wide, tokens, gs).reshape(-1))
        assert np.array_equal(out.reshape(-1), ora.w4a8_matmul(*proj, att, wide, wide, tokens, gs).reshape(-1))
        assert np.array_equal(after[:, heads * hd:], before[:, heads * hd:])
        pool.k[:], pool.v[:] = dev.pool_back(pool)
        for s, (a, m, n) in enumerate(zip(starts, news, lengths)):
            for j in range(m):
                q = before[a + j, :heads * hd].reshape(heads, hd)
                # Two products, a sum and the angle's cosine and sine, each within three half steps.
                size = 8 * EPS32 * gain * np.sqrt(2) * np.abs(before[a + j]).max()
                want = rotate(q, n - m + j, inv, hd, 0, gain)
                assert (np.abs(after[a + j, :heads * hd].reshape(heads, hd) - want) <= size).all()
            q = after[:, :heads * hd].reshape(tokens, heads, hd)
            want, tol = attend(pool, layer, (int(a), m, n), s, q, heads, hd ** -0.5)
            assert (np.abs(att[a:a + m].reshape(m, heads, hd) - want) <= tol).all()
        dx = do


@pytest.mark.parametrize("cache", CACHES)
def test_beam_search_over_the_pages(rai, cache):
    """A beam search as a program runs it: the prompt stored and attended as a chunk, then steps of
    selection, fork, store and attention; every step's attention equals attention over each beam's own
    history, kept apart on the host."""
    heads, kv_heads, hd, page, beams, steps, prompt, vocab = 4, 2, 64, 16, 4, 6, 21, 40
    stride, pool_pages = 4, 64
    rng = np.random.default_rng(5)
    table_k, table_v, table_q = (rng.standard_normal((vocab, n * hd)).astype(np.float32) for n in (kv_heads, kv_heads, heads))
    out_w = rng.standard_normal((heads * hd, vocab)).astype(np.float32)
    inv, gain = rai.rope_frequencies(rai.ROPE_LINEAR, 1e4, hd, 2.0)
    pool = Pool(cache, page, kv_heads, hd, [0] * beams, layers=1, spare=pool_pages, stride=stride)
    free = [int(p) for p in pool.spare]
    dev = Dev(rai)
    pg, L = dev.pages(pool), rai.lib()
    rope = rai.Rope(dev.up(inv).ptr, hd, 0, gain)
    opts = rai.AttentionOptions(hd ** -0.5, 0.0, 0, None)
    tables, lengths = np.full((beams, stride), -1, np.int32), np.zeros(beams, np.int32)

    def forward(news):
        """Stores and attends news[i] at the end of sequence i; logits of each last token."""
        tokens = [t for new in news for t in new]
        for i, new in enumerate(news):
            for p in range(lengths[i], lengths[i] + len(new)):
                if tables[i, p // page] < 0:
                    tables[i, p // page] = free.pop()
            lengths[i] += len(new)
        n, q = len(tokens), table_q[tokens]
        starts = _starts([len(new) for new in news])
        batch = rai.PageBatch(dev.up(tables).ptr, stride, dev.up(np.int32(starts)).ptr, dev.up(lengths).ptr, len(news), n,
                              max(map(len, news)), int(lengths.max()))
        dq, do = dev.up(q), rai.DeviceArray(q.nbytes)
        rai._check(L.rai_paged_store_dev(pg, 0, batch, rope, dq.ptr, heads * hd, dq.ptr, heads * hd, heads,
                                         dev.up(table_k[tokens]).ptr, kv_heads * hd, dev.up(table_v[tokens]).ptr,
                                         kv_heads * hd, None))
        work = rai.attention_workspace(heads, pg, batch, opts)
        dw = rai.DeviceArray(max(work, 16))
        rai._check(L.rai_paged_attention_dev(do.ptr, heads * hd, dq.ptr, heads * hd, heads, pg, 0, batch, opts, dw.ptr,
                                             work, None))
        rai._check(L.rai_device_synchronize())
        return do.to_host(np.float32, n * heads * hd).reshape(n, heads * hd)[starts[1:] - 1]

    def alone(history):
        """The last token's attention over a beam's own history, in f64."""
        own = Pool(cache, page, kv_heads, hd, [len(history)])
        for p, t in enumerate(history):
            k = rotate(table_k[t].reshape(kv_heads, hd), p, inv, hd, 0, gain)
            own.put(0, 0, p, k, table_v[t].reshape(kv_heads, hd))
        q = rotate(table_q[history[-1]].reshape(heads, hd), len(history) - 1, inv, hd, 0, gain)
        return attend(own, 0, (0, 1, len(history)), 0, q[None], heads, hd ** -0.5)[0].reshape(-1)

    first = rng.integers(0, vocab, prompt).tolist()
    histories, scores = [list(first) for _ in range(beams)], np.float32([0.0] + [-np.inf] * (beams - 1))
    hidden = forward([first] + [[]] * (beams - 1))
    hidden = np.repeat(hidden[:1], beams, 0)
    tables[1:], lengths[1:] = tables[0], lengths[0]
    # A rounding of a stored key to the cache's type may fall on either side: its share of the output.
    slack = {"f32": 1e-5, "f16": 1e-2, "bf16": 8e-2}[cache]
    for _ in range(steps):
        logits = 0.05 * hidden @ out_w
        dl, ds, need = dev.up(logits), dev.up(scores), rai.beam_workspace(vocab, 1, beams, beams)
        parent, token, score = (rai.DeviceArray(4 * beams) for _ in range(3))
        work = rai.DeviceArray(need)
        rai._check(L.rai_beam_select_dev(dl.ptr, vocab, vocab, ds.ptr, None, 0, 1, beams, beams, parent.ptr, token.ptr,
                                         score.ptr, work.ptr, need, None))
        fresh = np.int32([free.pop() for _ in range(beams)])
        to, lo, uo = rai.DeviceArray(4 * beams * stride), rai.DeviceArray(4 * beams), rai.DeviceArray(4 * beams)
        rai._check(L.rai_paged_fork_dev(pg, dev.up(tables).ptr, stride, dev.up(lengths).ptr, beams, parent.ptr,
                                        dev.up(fresh).ptr, beams, to.ptr, lo.ptr, uo.ptr, None))
        rai._check(L.rai_device_synchronize())
        pick, tok = parent.to_host(np.int32, beams), token.to_host(np.int32, beams)
        want = _select(logits, scores, None, 0, beams, beams)
        assert np.array_equal(pick, want[0]) and np.array_equal(tok, want[1])
        scores = score.to_host(np.float32, beams)
        tables, lengths = to.to_host(np.int32, beams * stride).reshape(beams, stride), lo.to_host(np.int32, beams)
        free += [int(f) for f, u in zip(fresh, uo.to_host(np.int32, beams)) if not u]
        histories = [histories[p] + [int(t)] for p, t in zip(pick, tok)]
        hidden = forward([[int(t)] for t in tok])
        for h, got in zip(histories, hidden):
            assert np.abs(got - alone(h)).max() <= slack, len(h)
    # Compaction: the pages in use move to the lowest free places; attention reads the same.
    live = sorted({int(p) for p in tables.reshape(-1) if p >= 0})
    holes = [p for p in range(len(live)) if p not in live]
    high = [p for p in live if p >= len(live)]
    dt = dev.up(tables)
    rai._check(L.rai_paged_move_dev(pg, dev.up(np.int32(high)).ptr, dev.up(np.int32(holes)).ptr, len(high), dt.ptr,
                                    tables.size, None))
    rai._check(L.rai_device_synchronize())
    tables = dt.to_host(np.int32, tables.size).reshape(tables.shape)
    assert tables.max() < len(live)
    free = [p for p in range(pool.pages) if p >= len(live)]
    hidden = forward([[int(h[0])] for h in histories])
    for h, got in zip(histories, hidden):
        assert np.abs(got - alone(h + [h[0]])).max() <= slack
