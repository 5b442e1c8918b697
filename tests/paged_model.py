"""A paged KV cache on the host and the operators over it in 64 bits, from their
definitions (numpy only)."""
import numpy as np

EPS32 = 2.0 ** -24  # half a step of f32, relative


def bf16_bits(x):
    """f32 -> bf16 bits, to nearest, ties to even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def encode(x, cache):
    x = np.asarray(x, np.float32)
    if cache == "f32":
        return x
    if cache == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    return bf16_bits(x)


def decode(a, cache):
    if cache == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32)
    return a.astype(np.float32)


def store_dtype(cache):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[cache]


class Pool:
    """k [layers][pages][kv_heads][slot][hd], v [layers][pages][kv_heads][hd][slot], every slot NaN at first;
    tables over scattered pages, -1 behind a sequence's last."""

    def __init__(self, cache, page, kv_heads, hd, lengths, seed=0, layers=1, spare=2, stride=None):
        self.cache, self.page, self.kv_heads, self.hd, self.layers = cache, page, kv_heads, hd, layers
        self.rng = np.random.default_rng(seed)
        counts = [-(-n // page) for n in lengths]
        self.pages = sum(counts) + spare
        ids = self.rng.permutation(self.pages).astype(np.int32)
        self.tables = np.full((len(lengths), stride or max(counts + [1])), -1, np.int32)
        at = 0
        for i, n in enumerate(counts):
            self.tables[i, :n] = ids[at:at + n]
            at += n
        self.spare = ids[at:]
        nan = encode(np.full(1, np.nan, np.float32), cache)[0]
        self.k = np.full((layers, self.pages, kv_heads, page, hd), nan, store_dtype(cache))
        self.v = np.full((layers, self.pages, kv_heads, hd, page), nan, store_dtype(cache))

    def place(self, seq, pos):
        """(page, slot) of a position, None where there is none."""
        if pos < 0 or pos // self.page >= self.tables.shape[1]:
            return None
        p = int(self.tables[seq, pos // self.page])
        return (p, pos % self.page) if 0 <= p < self.pages else None

    def put(self, layer, seq, pos, k, v):
        """Row k, v [kv_heads][hd] (f32) at a position."""
        where = self.place(seq, pos)
        if where is not None:
            self.k[layer, where[0], :, where[1]] = encode(k, self.cache)
            self.v[layer, where[0], :, :, where[1]] = encode(v, self.cache)

    def fill(self, layer, lengths, std=1.0):
        for s, n in enumerate(lengths):
            for p in range(n):
                self.put(layer, s, p, *(std * self.rng.standard_normal((2, self.kv_heads, self.hd))))

    def rows(self, layer, seq, positions):
        """k, v [len(positions)][kv_heads][hd] in f64, and which are there."""
        there = np.array([self.place(seq, int(p)) is not None for p in positions], bool)
        k = np.zeros((len(positions), self.kv_heads, self.hd))
        v = np.zeros_like(k)
        for i in np.flatnonzero(there):
            pg, slot = self.place(seq, int(positions[i]))
            k[i] = decode(self.k[layer, pg, :, slot], self.cache)
            v[i] = decode(self.v[layer, pg, :, :, slot], self.cache)
        return k, v, there


def spans(q_start, kv_len, tokens, max_q, max_kv):
    """(first row, rows, length) of each sequence, cut to the bounds."""
    out = []
    for s in range(len(kv_len)):
        a = min(max(int(q_start[s]), 0), tokens)
        b = min(max(int(q_start[s + 1]), a), tokens)
        out.append((a, min(b - a, max_q), min(max(int(kv_len[s]), 0), max_kv)))
    return out


def rotate(x, pos, inv, rot, interleaved, gain):
    """x [heads][hd] in f64."""
    y = np.array(x, np.float64)
    c, s = np.cos(pos * inv) * gain, np.sin(pos * inv) * gain
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    x0, x1 = y[:, a].copy(), y[:, b].copy()
    y[:, a], y[:, b] = x0 * c - x1 * s, x1 * c + x0 * s
    return y


def attend(pool, layer, span, seq, q, heads, scale, softcap=0.0, window=0, slopes=None):
    """Rows [nq][heads][hd] of one sequence in f64, and a bound of what f32 arithmetic may be off by.

    The bound: a score is a sum of hd products, in f32 off by at most (hd + 8) half steps of the sum of
    their magnitudes (8: the cast operands, the scale, the cap and the bias, each once or twice); the
    exponential turns that, and the half steps of its own argument, into a relative error of the weight;
    the sums over the n keys add n + 16 half steps of the sum of the weighted magnitudes."""
    q0, nq, n = span
    hd, per = pool.hd, heads // pool.kv_heads
    out, tol = np.zeros((nq, heads, hd)), np.zeros((nq, heads, hd))
    k, v, there = pool.rows(layer, seq, np.arange(n))
    for j in range(nq):
        pos = n - nq + j
        lo = max(0, pos - window + 1) if window else 0
        if pos < 0:
            continue
        seen = np.flatnonzero(there[lo:pos + 1]) + lo
        if not len(seen):
            continue
        for h in range(heads):
            kk, vv, x = k[seen, h // per], v[seen, h // per], q[q0 + j, h].astype(np.float64)
            s = kk @ x * scale
            mag = np.abs(kk) @ np.abs(x) * abs(scale)
            if softcap:
                s = softcap * np.tanh(s / softcap)
            if slopes is not None:
                s = s - float(slopes[h]) * (pos - seen)
                mag = mag + abs(float(slopes[h])) * (pos - seen)
            d = s - s.max()
            w = np.exp(d)
            p = w / w.sum()
            out[j, h] = p @ vv
            off = EPS32 * ((hd + 8) * mag + 4 * np.abs(s) + 4 * np.abs(d))
            worst = (p * np.expm1(np.minimum(2 * (off + off.max()), 50.0))) @ np.abs(vv)
            tol[j, h] = worst + EPS32 * (len(seen) + 16) * (p @ np.abs(vv)) + EPS32 * (p @ np.abs(vv))
    return out, tol


# How far normal inputs' attention may be off in f32, in half steps of the 2-norm.  A score's sum of hd products
# passes through at most 96 f32 sums (hd 256 in sixteenths, six products each), the output's through 57 per 300 keys
# of a block's share and part; a rounding is off by at most two half steps (one when to nearest) of a partial sum
# that is 0.7 of the result in the mean square.  Independent ones add up as squares: 0.7 * 2 * sqrt(96) = 14 for the
# score, 0.7 * 2 * sqrt(3 * 57) / sqrt(3) = 11 for the output, 5 for the exponential and its argument: 18, and
# dividing, joining and the operands' last bits (2) are within 25.  A row by itself, few of whose weights may carry
# it: twice that.
ACCURATE = 25


def off_by(got, want):
    """Half steps of the 2-norm: all rows [..][hd] together, and the worst row."""
    d = np.linalg.norm(got.astype(np.float64) - want, axis=-1)
    n = np.linalg.norm(want, axis=-1)
    return np.linalg.norm(d) / np.linalg.norm(n) / EPS32, (d / n).max() / EPS32


def cut(x, cache, parts):
    """f32 values as the parts that a 16-bit matrix operand holds, largest first: bf16 parts cut off, f16 parts
    rounded."""
    out, rest = [], np.array(x, np.float32)
    for _ in range(parts):
        if cache == "f16":
            h = rest.astype(np.float16).astype(np.float32)
        else:
            h = (rest.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        out.append(h.astype(np.float64))
        rest = rest - h
    return out


def attend_cut(q, k, v, cache, query_parts, weight_parts, key_parts=1, value_parts=1, products=None):
    """softmax(q k^T / sqrt(hd)) v in f64 whose operands are cut into parts, of whose pairs i + j < products count."""
    def dot(a, b, m):
        return sum(x @ y for i, x in enumerate(a) for j, y in enumerate(b) if i + j < (products or len(a) + m))

    s = dot(cut(q, cache, query_parts), [x.T for x in cut(k, cache, key_parts)], key_parts) / np.sqrt(q.shape[1])
    p = np.exp(s - s.max(1, keepdims=True))
    return dot(cut(p * 2.0 ** 14, cache, weight_parts), cut(v, cache, value_parts), value_parts) / 2.0 ** 14 / p.sum(1, keepdims=True)
