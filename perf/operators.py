"""Operators of serving over a paged KV cache: what they compute, and the calls that a program makes of them.

Four operators, each case a dict of plain values:

  store      rotary positions of a batch's queries and keys (half or interleaved pairs, part of the
             head, scaled frequencies), keys and values put into the pages of their sequences
             (rai_paged_store_dev)
  attention  a batch's new tokens over the pages of their sequences: from one token a sequence to
             chunks of a prompt, ragged, with a score cap, a window or a distance bias
             (rai_paged_attention_dev)
  pages      rai_paged_fork_dev (sequences that go on from others, as beams do: shared full pages, a
             copy of a part-filled one) and rai_paged_move_dev (pages moved and renamed, as a
             compaction does)
  beam       beam search's selection over beams and vocabulary (rai_beam_select_dev)

Activations are f32, as everywhere in the framework; the cache is f32, f16 or bf16.  Pages lie as
[layer][page][kv_head][slot][head_dim] for keys and [layer][page][kv_head][head_dim][slot] for values.
"""
import ctypes
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": (0, torch.float32, 4), "f16": (1, torch.float16, 2), "bf16": (2, torch.bfloat16, 2)}

# Head layouts of the benchmarked model families.
TINYLLAMA = dict(heads=32, kv_heads=4, head_dim=64)
MISTRAL = dict(heads=32, kv_heads=8, head_dim=128)
OLMOE = dict(heads=16, kv_heads=16, head_dim=128)


def _attention(shape, cache, page, seqs, q, kv, mix, layers=1, softcap=0.0, window=0, bias=False, fused=False):
    """`seqs` sequences of q[0]..q[1] new tokens behind kv[0]..kv[1] cached ones, spread by `mix`; `fused`: the
    queries are columns of a wider row (a fused projection's output)."""
    return {"kind": "attention", **shape, "cache": cache, "page": page, "seqs": seqs, "q_lo": q[0], "q_hi": q[1],
            "kv_lo": kv[0], "kv_hi": kv[1], "mix": mix, "layers": layers, "softcap": softcap, "window": window,
            "bias": bias, "fused": fused}


def _store(shape, cache, page, seqs, q, kv, mix, rot, interleaved, scaling, factor, fused=False):
    return {"kind": "store", **shape, "cache": cache, "page": page, "seqs": seqs, "q_lo": q[0], "q_hi": q[1],
            "kv_lo": kv[0], "kv_hi": kv[1], "mix": mix, "layers": 2, "rot": rot, "interleaved": interleaved,
            "scaling": scaling, "factor": factor, "fused": fused}


def _fork(shape, cache, page, layers, groups, beams, kv, mix):
    return {"kind": "fork", **shape, "cache": cache, "page": page, "layers": layers, "groups": groups,
            "beams": beams, "kv_lo": kv[0], "kv_hi": kv[1], "mix": mix}


def _move(shape, cache, page, layers, pages, moved, seqs):
    return {"kind": "move", **shape, "cache": cache, "page": page, "layers": layers, "pages": pages, "moved": moved,
            "seqs": seqs}


def _beam(groups, beams, vocab, take, finished):
    return {"kind": "beam", "groups": groups, "beams": beams, "vocab": vocab, "take": take, "finished": finished}


def listed():
    cases = {
        # The smallest call: one decoded token of a short chat, TinyLlama's heads, the framework's own f32 rows.
        "decode1_tinyllama_200_f32": _attention(TINYLLAMA, "f32", 16, 1, (1, 1), (200, 200), 1),
        # A decode step of a serving batch: 32 sequences of very different lengths.
        "decode32_mistral_4096_bf16": _attention(MISTRAL, "bf16", 16, 32, (1, 1), (64, 4096), 2),
        # One sequence far into a long document: few rows, a long axis.
        "decode1_mistral_32768_f16": _attention(MISTRAL, "f16", 64, 1, (1, 1), (32768, 32768), 3),
        # Verify batches (8 drafts + 1) of eight sequences, every head with keys of its own.
        "verify9x8_olmoe_4000_f32": _attention(OLMOE, "f32", 32, 8, (9, 9), (500, 4000), 4, fused=True),
        # A chunk of a long prompt.
        "prefill1024_mistral_4096_bf16": _attention(MISTRAL, "bf16", 64, 1, (1024, 1024), (4096, 4096), 5),
        # A mixed step: chunks of prompts and decoded tokens together, capped scores, a sliding window.
        "mixed6_mistral_capped_window_f32": _attention(MISTRAL, "f32", 16, 6, (1, 700), (0, 5000), 6, softcap=30.0,
                                                       window=1500),
        # One token's keys and values into their page.
        "store1_tinyllama_f32": _store(TINYLLAMA, "f32", 16, 1, (1, 1), (200, 200), 8, 64, False, "none", 1.0),
        # Chunks of four prompts, part of the head rotated in interleaved pairs, scaled for a long context.
        "store2000_mistral_yarn_bf16": _store(MISTRAL, "bf16", 64, 4, (300, 701), (0, 20000), 9, 96, True, "yarn",
                                              4.0, fused=True),
        # After a beam step: 4 x 8 sequences go on from their parents.
        "fork32_mistral_bf16": _fork(MISTRAL, "bf16", 64, 16, 4, 8, (100, 2000), 10),
        # A compaction: a quarter of a pool's pages move to free places.
        "move300_tinyllama_f16": _move(TINYLLAMA, "f16", 32, 22, 1201, 300, 48),
        # Beam selection of one request: latency.
        "beam1x4_32000": _beam(1, 4, 32000, 8, False),
        # Beam selection of a serving batch, some beams finished.
        "beam32x8_50304": _beam(32, 8, 50304, 16, True),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention"] * 10 + ["store"] * 4 + ["fork"] * 2 + ["move"] * 2 + ["beam"] * 4)
    if kind == "beam":
        while True:
            c = _beam(_log(rng, 1, 64), rng.randint(1, 16), _log(rng, 1000, 130000), 0, rng.random() < 0.5)
            if c["groups"] * c["beams"] * c["vocab"] <= 32 * 8 * 50304:
                return dict(c, take=rng.choice([c["beams"], 2 * c["beams"]]))
    per, kv_heads = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8, 16])
    while per * kv_heads < 4 or per * kv_heads > 32:
        per, kv_heads = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8, 16])
    shape = dict(heads=per * kv_heads, kv_heads=kv_heads, head_dim=rng.choice([64, 64, 80, 96, 128, 128, 128]))
    cache, page, mix = rng.choice(["f32", "f16", "bf16"]), rng.choice([16, 16, 32, 64, 128]), rng.randint(1, 1 << 20)
    row = kv_heads * shape["head_dim"] * TYPES[cache][2]  # bytes of one position's keys
    if kind == "move":
        layers, pages = rng.randint(1, 24), _log(rng, 64, 2000)
        moved = _log(rng, 4, pages // 3)
        if layers * moved * page * row > 22 * 300 * 32 * 512:
            moved = max(1, 22 * 300 * 32 * 512 // (layers * page * row))
        layers = max(1, min(layers, (1 << 30) // (pages * page * row)))
        return _move(shape, cache, page, layers, pages, moved, rng.randint(1, 64))
    if kind == "fork":
        groups, beams = rng.randint(1, 4), rng.randint(2, 8)
        c = _fork(shape, cache, page, rng.randint(1, 16), groups, beams, (rng.randint(1, 100), _log(rng, 101, 2000)), mix)
        while c["layers"] * page * row > 16 * 64 * 2048:
            c["layers"] -= 1
        return c
    new = rng.choice([(1, 1), (1, 1), (2, 17), (1, 300), (100, 1024)])
    q_hi = _log(rng, *new)
    q_lo = max(1, q_hi // rng.choice([1, 2, 8]))
    fused = rng.random() < 0.3
    if kind == "store":
        rot = rng.choice([shape["head_dim"], shape["head_dim"], shape["head_dim"] // 2, 32])
        most = max(1, 2000 * 8 * 128 // (q_hi * kv_heads * shape["head_dim"]))
        scaling, factor = rng.choice([("none", 1.0), ("linear", 4.0), ("llama3", 8.0), ("yarn", 4.0), ("yarn", 16.0)])
        return _store(shape, cache, page, rng.randint(1, min(32, most)), (q_lo, q_hi), (0, _log(rng, 1, 20000)), mix,
                      rot, rng.random() < 0.5, scaling, factor, fused)
    seqs = rng.randint(1, max(1, min(32, 1500 // q_hi)))
    kv_hi = _log(rng, 16, max(17, min(32768, 131072 // seqs, (1 << 22) // (q_hi * seqs))))
    return _attention(shape, cache, page, seqs, (q_lo, q_hi), (rng.choice([0, kv_hi // 4, kv_hi]), kv_hi), mix,
                      layers=rng.choice([1, 2]), softcap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                      window=rng.choice([0, 0, _log(rng, 64, 4096)]), bias=rng.random() < 0.25, fused=fused)


# ----------------------------------------------------------------- inputs --

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 6271 + 29)


def _normal(g, *shape):
    return torch.empty(*shape, device="cuda").normal_(0.0, 1.0, generator=g)


def _lengths(c):
    """New tokens and cached positions of each sequence: the case's own, the same for every seed."""
    r = random.Random(c["mix"])
    new = [r.randint(c["q_lo"], c["q_hi"]) for _ in range(c["seqs"])]
    old = [r.randint(c["kv_lo"], c["kv_hi"]) for _ in range(c["seqs"])]
    new[0], old[-1] = c["q_hi"], c["kv_hi"]
    return new, old


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pool(g, c, pages):
    """The pages of a cache that has been in use: no slot is empty."""
    t = TYPES[c["cache"]][1]
    shape = (c["layers"], pages, c["kv_heads"])
    return (_normal(g, *shape, c["page"], c["head_dim"]).to(t), _normal(g, *shape, c["head_dim"], c["page"]).to(t))


def _tables(seed, lengths, page, spare):
    """Page tables [sequence][most pages] over scattered pages, -1 past a sequence's last, and the pool's size."""
    counts = [-(-n // page) for n in lengths]
    ids = np.random.default_rng(seed).permutation(sum(counts) + spare).astype(np.int32)
    tables, at = np.full((len(counts), max(counts)), -1, np.int32), 0
    for i, n in enumerate(counts):
        tables[i, :n] = ids[at:at + n]
        at += n
    return tables, ids[at:], sum(counts) + spare


def _frequencies(c):
    """Inverse frequencies of the rotated pairs in 64 bits, and the factor on the rotated values; the published
    rules of position interpolation, Llama 3.1 and YaRN, for a model trained on 8192 positions at base 10000."""
    rot, base, factor, trained = c["rot"], 10000.0, c["factor"], 8192.0
    inv = base ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    if c["scaling"] == "linear":
        return inv / factor, 1.0
    if c["scaling"] == "llama3":  # low frequencies divided, high ones kept, those between blended
        turns = trained * inv / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return inv * (keep + (1 - keep) / factor), 1.0
    if c["scaling"] == "yarn":  # blended by the pair's index between those that turn 32 times and once
        edge = [rot * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32.0, 1.0)]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
        ramp = np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return inv * ((1 - ramp) + ramp / factor), 0.1 * math.log(factor) + 1.0
    return inv, 1.0


def _batch(c, g, seed):
    """A batch's page tables, row starts and lengths on the GPU, the pages, and the batch's rows of activations."""
    new, old = _lengths(c)
    lengths = [a + b for a, b in zip(new, old)]
    tables, _, pages = _tables(seed, lengths, c["page"], 3)
    k, v = _pool(g, c, pages)
    starts = np.concatenate([[0], np.cumsum(new)])
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    tokens, wide = sum(new), (nh + 2 * nkv) * hd
    if c["fused"]:
        rows = _normal(g, tokens, wide)
        parts = rows[:, :nh * hd], rows[:, nh * hd:(nh + nkv) * hd], rows[:, (nh + nkv) * hd:]
    else:
        parts = _normal(g, tokens, nh * hd), _normal(g, tokens, nkv * hd), _normal(g, tokens, nkv * hd)
    return {"case": c, "k_pages": k, "v_pages": v, "tables": _ints(tables), "starts": _ints(starts),
            "lengths": _ints(lengths), "tokens": tokens, "max_q": max(new), "max_kv": max(lengths),
            "q": parts[0], "k": parts[1], "v": parts[2]}


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] == "beam":
        rows = c["groups"] * c["beams"]
        logits = _normal(g, rows, c["vocab"]).mul_(2.5)
        scores = _normal(g, rows).abs_().mul_(-3.0)
        done = (torch.rand(rows, device="cuda", generator=g) < 0.15).to(torch.uint8) if c["finished"] else None
        n = c["groups"] * c["take"]
        out = [torch.zeros(n, dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.float32)]
        return {"case": c, "logits": logits, "scores": scores, "done": done, "out": out,
                "work": torch.empty(1 << 25, dtype=torch.uint8, device="cuda")}
    if c["kind"] == "move":
        k, v = _pool(g, c, c["pages"])
        r = np.random.default_rng(seed)
        ids = r.permutation(c["pages"]).astype(np.int32)
        src, dst, live = ids[:c["moved"]], ids[c["moved"]:2 * c["moved"]], np.delete(ids, slice(c["moved"], 2 * c["moved"]))
        return {"case": c, "k_pages": k, "v_pages": v, "src": _ints(src), "dst": _ints(dst),
                "tables": _ints(r.choice(live, (c["seqs"], 32)))}
    if c["kind"] == "fork":
        r = random.Random(c["mix"])
        lengths = [n for n in (r.randint(c["kv_lo"], c["kv_hi"]) for _ in range(c["groups"])) for _ in range(c["beams"])]
        n = len(lengths)
        tables, spare, pages = _tables(seed, lengths, c["page"], n)
        k, v = _pool(g, c, pages)
        group = np.arange(n) // c["beams"] * c["beams"]
        parent = group + np.random.default_rng(seed + 1).integers(0, c["beams"], n)
        return {"case": c, "k_pages": k, "v_pages": v, "tables": _ints(tables), "lengths": _ints(lengths),
                "parent": _ints(parent), "fresh": _ints(spare), "tables_out": torch.zeros_like(_ints(tables)),
                "lengths_out": _ints(lengths).zero_(), "used": _ints(lengths).zero_()}
    s = _batch(c, g, seed)
    nh, hd = c["heads"], c["head_dim"]
    s["out"] = torch.zeros(s["tokens"], nh * hd, device="cuda")
    if c["kind"] == "store":
        inv, s["gain"] = _frequencies(c)
        s["inv"] = torch.from_numpy(inv).to("cuda")
        return s
    s["slopes"] = torch.exp2(-8.0 * torch.arange(1, nh + 1, device="cuda") / nh) if c["bias"] else None
    s["work"] = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")  # a program's own, kept between calls
    return s


# -------------------------------------------------------------------- run --

def run(state):
    c = state["case"]
    if own:
        import rai_amd
        return _own(state, c, rai_amd)
    if c["kind"] == "beam":
        return _plain_beam(state, c)
    if c["kind"] == "move":
        return _plain_move(state)
    if c["kind"] == "fork":
        return _plain_fork(state, c)
    return _plain_store(state, c) if c["kind"] == "store" else _plain_attention(state, c)


def _address(t):
    return None if t is None else t.data_ptr()


def _own(s, c, rai):
    def check(rc):
        if rc:
            raise RuntimeError(lib.rai_last_error().decode())

    lib, stream = rai.lib(), torch.cuda.current_stream().cuda_stream
    if c["kind"] == "beam":
        parent, token, score = s["out"]
        check(lib.rai_beam_select_dev(s["logits"].data_ptr(), c["vocab"], c["vocab"], s["scores"].data_ptr(),
                                          _address(s["done"]), 0, c["groups"], c["beams"], c["take"],
                                          parent.data_ptr(), token.data_ptr(), score.data_ptr(),
                                          s["work"].data_ptr(), s["work"].numel(), stream))
        return {"parent": parent, "token": token, "score": score}
    kp, vp = s["k_pages"], s["v_pages"]
    pages = rai.Pages(kp.data_ptr(), vp.data_ptr(), c["layers"], kp.shape[1], c["page"], c["kv_heads"], c["head_dim"],
                      TYPES[c["cache"]][0])
    t = s["tables"]
    if c["kind"] == "move":
        check(lib.rai_paged_move_dev(ctypes.byref(pages), s["src"].data_ptr(), s["dst"].data_ptr(), c["moved"],
                                         t.data_ptr(), t.numel(), stream))
        return {"k": kp, "v": vp, "tables": t}
    if c["kind"] == "fork":
        out = s["tables_out"]
        check(lib.rai_paged_fork_dev(ctypes.byref(pages), t.data_ptr(), t.shape[1], s["lengths"].data_ptr(),
                                         t.shape[0], s["parent"].data_ptr(), s["fresh"].data_ptr(), out.shape[0],
                                         out.data_ptr(), s["lengths_out"].data_ptr(), s["used"].data_ptr(), stream))
        return {"k": kp, "v": vp, "tables": out, "lengths": s["lengths_out"], "used": s["used"]}
    batch = rai.PageBatch(t.data_ptr(), t.shape[1], s["starts"].data_ptr(), s["lengths"].data_ptr(), t.shape[0],
                          s["tokens"], s["max_q"], s["max_kv"])
    q, layer, wide = s["q"], c["layers"] - 1, c["heads"] * c["head_dim"]
    if c["kind"] == "store":
        rope = rai.Rope(s["inv"].data_ptr(), c["rot"], c["interleaved"], s["gain"])
        check(lib.rai_paged_store_dev(ctypes.byref(pages), layer, ctypes.byref(batch), ctypes.byref(rope),
                                          s["out"].data_ptr(), wide, q.data_ptr(), q.stride(0), c["heads"],
                                          s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0),
                                          stream))
        return {"q": s["out"], "k": kp, "v": vp}
    how = rai.AttentionOptions(1.0 / math.sqrt(c["head_dim"]), c["softcap"], c["window"], _address(s["slopes"]))
    check(lib.rai_paged_attention_dev(s["out"].data_ptr(), wide, q.data_ptr(), q.stride(0), c["heads"],
                                          ctypes.byref(pages), layer, ctypes.byref(batch), ctypes.byref(how),
                                          s["work"].data_ptr(), s["work"].numel(), stream))
    return s["out"]


def _plain_beam(s, c):
    groups, beams, vocab = c["groups"], c["beams"], c["vocab"]
    # In 64 bits: near the border of the best, the order decides.
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    total = s["scores"].double()[:, None] + (x - top - (x - top).exp().sum(1, keepdim=True).log())
    if s["done"] is not None:  # a finished beam goes on with token 0 alone, at the score it has
        done = s["done"].bool()[:, None]
        kept = torch.full_like(total, -math.inf)
        kept[:, 0] = s["scores"].double()
        total = torch.where(done, kept, total)
    score, at = total.view(groups, beams * vocab).sort(dim=1, descending=True, stable=True)
    score, at = score[:, :c["take"]], at[:, :c["take"]]
    parent = at // vocab + torch.arange(groups, device=at.device)[:, None] * beams
    none = score == -math.inf  # fewer candidates than asked for
    parent, token = parent.masked_fill(none, -1), (at % vocab).masked_fill(none, -1)
    return {"parent": parent.int().view(-1), "token": token.int().view(-1), "score": score.float().reshape(-1)}


def _plain_move(s):
    src, dst, names = s["src"].long(), s["dst"].long(), torch.arange(s["k_pages"].shape[1], device="cuda")
    s["k_pages"][:, dst] = s["k_pages"][:, src]
    s["v_pages"][:, dst] = s["v_pages"][:, src]
    names[src] = dst
    s["tables"].copy_(names[s["tables"].long()])
    return {"k": s["k_pages"], "v": s["v_pages"], "tables": s["tables"]}


def _plain_fork(s, c):
    parent, fresh, n = s["parent"].long(), s["fresh"].long(), s["parent"].numel()
    length = s["lengths"].long()[parent]
    order = torch.arange(n, device="cuda")
    again = ((parent[:, None] == parent[None]) & (order[None] < order[:, None])).any(1)
    need = again & (length % c["page"] != 0)  # a later child of a part-filled page takes a copy of it
    tables, last = s["tables"][parent], (length - 1) // c["page"]
    src = torch.where(need, tables[order, last].long(), fresh)
    s["k_pages"][:, fresh] = s["k_pages"][:, src]
    s["v_pages"][:, fresh] = s["v_pages"][:, src]
    tables[order, last] = torch.where(need, fresh.int(), tables[order, last])
    return {"k": s["k_pages"], "v": s["v_pages"], "tables": tables, "lengths": length.int(), "used": need.int()}


def _positions(s):
    """Each row's sequence and its position."""
    row = torch.arange(s["tokens"], device="cuda")
    starts = s["starts"].long()
    seq = torch.searchsorted(starts, row, right=True) - 1
    return seq, s["lengths"].long()[seq] - starts[seq + 1] + row


def _rotate(x, heads, c, inv, gain, pos):
    hd, rot = c["head_dim"], c["rot"]
    angle = pos.double()[:, None] * inv  # far positions: 64 bits
    co, si = (angle.cos() * gain).float()[:, None], (angle.sin() * gain).float()[:, None]
    x = x.reshape(-1, heads, hd)
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * co - b * si, b * co + a * si], 3).flatten(2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * co - b * si, b * co + a * si], 2)
    return torch.cat([turned, x[..., rot:]], 2)


def _plain_store(s, c):
    nh, nkv, hd, layer = c["heads"], c["kv_heads"], c["head_dim"], c["layers"] - 1
    seq, pos = _positions(s)
    q = _rotate(s["q"], nh, c, s["inv"], s["gain"], pos).reshape(-1, nh * hd)
    k = _rotate(s["k"], nkv, c, s["inv"], s["gain"], pos)
    page, slot = s["tables"][seq, pos // c["page"]].long(), pos % c["page"]
    s["k_pages"][layer][page, :, slot] = k.to(s["k_pages"].dtype)
    s["v_pages"][layer][page, :, :, slot] = s["v"].reshape(-1, nkv, hd).to(s["v_pages"].dtype)
    return {"q": q, "k": s["k_pages"], "v": s["v_pages"]}


def _plain_attention(s, c):
    nh, nkv, hd, layer, n = c["heads"], c["kv_heads"], c["head_dim"], c["layers"] - 1, s["max_kv"]
    starts, lengths, seqs, per = s["starts"].long(), s["lengths"].long(), c["seqs"], c["heads"] // c["kv_heads"]
    new, most = starts[1:] - starts[:-1], s["max_q"]
    at = torch.arange(n, device="cuda")
    page, slot = s["tables"][:, at // c["page"]].clamp_min(0).long(), (at % c["page"]).expand(seqs, n)
    k = s["k_pages"][layer][page, :, slot].float().permute(0, 2, 3, 1).reshape(seqs * nkv, hd, n)
    v = s["v_pages"][layer][page, :, :, slot].float().transpose(1, 2).reshape(seqs * nkv, n, hd)
    row = torch.arange(most, device="cuda")
    q = s["q"][(starts[:-1, None] + row).clamp_max(s["tokens"] - 1)].view(seqs, most, nkv, per, hd)
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs * nkv, most * per, hd)
    score = torch.bmm(q, k).mul_(1.0 / math.sqrt(hd)).view(seqs, nkv, most, per, n)
    if c["softcap"]:
        score = torch.tanh(score / c["softcap"]) * c["softcap"]
    pos = (lengths - new)[:, None] + row  # [sequence][row]
    away = pos[:, :, None] - at  # how far back a key lies
    if c["bias"]:
        score = score - s["slopes"].view(1, nkv, 1, per, 1) * away[:, None, :, None].float()
    seen = (away >= 0) & (away < c["window"]) if c["window"] else away >= 0
    score = score.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = (score - score.amax(4, keepdim=True)).exp_()
    p = p / p.sum(4, keepdim=True)
    o = torch.bmm(p.view(seqs * nkv, most * per, n), v).view(seqs, nkv, most, per, hd)
    seq = torch.searchsorted(starts, torch.arange(s["tokens"], device="cuda"), right=True) - 1
    o = o.permute(0, 2, 1, 3, 4).reshape(seqs, most, nh * hd)
    return o[seq, torch.arange(s["tokens"], device="cuda") - starts[seq]]


# ------------------------------------------------------------------- work --

def work(case):
    c = case
    if c["kind"] == "beam":
        rows, n = c["groups"] * c["beams"], c["groups"] * c["take"]
        return {"bytes": 4 * rows * c["vocab"] + 5 * rows + 12 * n, "flops": 4 * rows * c["vocab"]}
    size = TYPES[c["cache"]][2]
    page = 2 * c["layers"] * c["kv_heads"] * c["page"] * c["head_dim"] * size
    if c["kind"] == "move":
        return {"bytes": 2 * c["moved"] * page + 8 * c["moved"] + 8 * c["seqs"] * 32, "flops": 0}
    if c["kind"] == "fork":
        # Of n children of n random parents about n / e are later ones, which take a copy.
        n = c["groups"] * c["beams"]
        again = round(n * (1 - 1 / c["beams"]) ** c["beams"])
        return {"bytes": 2 * again * page + 4 * n * (c["kv_lo"] + c["kv_hi"]) // c["page"] + 24 * n, "flops": 0}
    new, old = _lengths(c)
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    if c["kind"] == "store":
        return {"bytes": sum(new) * hd * (8 * nh + (4 + size) * 2 * nkv), "flops": 3 * sum(new) * (nh + nkv) * c["rot"]}
    seen, pairs = 0, 0
    for m, p in zip(new, old):
        first = 0 if not c["window"] else max(0, p + 1 - c["window"])
        seen += p + m - first
        pairs += sum(min(p + j + 1, c["window"] or p + j + 1) for j in range(m))
    return {"bytes": 8 * sum(new) * nh * hd + 2 * seen * nkv * hd * size, "flops": 4 * pairs * nh * hd}


# ------------------------------------------------------------------ exact --

def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "beam":
        x = s["logits"].cpu().numpy().astype(np.float64).reshape(c["groups"], c["beams"], -1)
        base = s["scores"].cpu().numpy().astype(np.float64).reshape(c["groups"], c["beams"], 1)
        done = None if s["done"] is None else s["done"].cpu().numpy().reshape(c["groups"], c["beams"])
        best = []
        for i in range(c["groups"]):
            t = base[i] + x[i] - (np.log(np.exp(x[i] - x[i].max(1, keepdims=True)).sum(1, keepdims=True)) +
                                  x[i].max(1, keepdims=True))
            if done is not None:
                t[done[i] != 0] = -np.inf
                t[done[i] != 0, 0] = base[i][done[i] != 0, 0]
            best.append(np.sort(t.reshape(-1))[::-1][:c["take"]])
        return {"parent": None, "token": None, "score": np.concatenate(best)}
    k, v = s["k_pages"], s["v_pages"]
    if c["kind"] == "move":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            k[:, b], v[:, b] = k[:, a], v[:, a]
        return {"k": k, "v": v, "tables": None}
    if c["kind"] == "fork":
        taken = set()
        for p, f in zip(s["parent"].tolist(), s["fresh"].tolist()):
            n = int(s["lengths"][p])
            if p in taken and n % c["page"]:
                a = int(s["tables"][p, n // c["page"]])
                k[:, f], v[:, f] = k[:, a], v[:, a]
            taken.add(p)
        return {"k": k, "v": v, "tables": None, "lengths": None, "used": None}
    nh, nkv, hd, per, layer = c["heads"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"], c["layers"] - 1
    new, old = _lengths(c)
    if c["kind"] == "store":
        inv, gain = _frequencies(c)
        pos = torch.cat([torch.arange(p, p + m) for m, p in zip(new, old)]).cuda()
        z = torch.polar(torch.full((1, 1), gain, dtype=torch.float64), pos.cpu().double()[:, None] * torch.from_numpy(inv)).cuda()

        def turn(x, heads):
            x = x.reshape(-1, heads, hd).double()
            pair = x[..., :c["rot"]].reshape(-1, heads, c["rot"] // 2, 2) if c["interleaved"] else \
                x[..., :c["rot"]].reshape(-1, heads, 2, c["rot"] // 2).transpose(2, 3)
            pair = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z[:, None])
            pair = pair if c["interleaved"] else pair.transpose(2, 3)
            return torch.cat([pair.reshape(-1, heads, c["rot"]), x[..., c["rot"]:]], 2)

        kk, vv = turn(s["k"], nkv), s["v"].reshape(-1, nkv, hd).double()
        k, v = k.double(), v.double()
        at = 0
        for i, (m, p) in enumerate(zip(new, old)):
            where = torch.arange(p, p + m, device="cuda")
            page, slot = s["tables"][i][where // c["page"]].long(), where % c["page"]
            for h in range(nkv):
                k[layer, page, h, slot] = kk[at:at + m, h]
                v[layer].transpose(2, 3)[page, h, slot] = vv[at:at + m, h]
            at += m
        return {"q": turn(s["q"], nh).reshape(-1, nh * hd), "k": k, "v": v}
    out, at = torch.empty(s["tokens"], nh, hd, dtype=torch.float64, device="cuda"), 0
    for i, (m, p) in enumerate(zip(new, old)):
        ids = s["tables"][i, :-(-(p + m) // c["page"])].long()
        kk = k[layer, ids].double().transpose(0, 1).reshape(nkv, -1, hd)[:, :p + m]
        vv = v[layer, ids].double().permute(1, 0, 3, 2).reshape(nkv, -1, hd)[:, :p + m]
        far = torch.arange(p, p + m, device="cuda")[:, None] - torch.arange(p + m, device="cuda")[None]
        for h in range(nh):
            t = s["q"][at:at + m, h * hd:(h + 1) * hd].double() @ kk[h // per].t() * hd ** -0.5
            if c["softcap"]:
                t = c["softcap"] * (t / c["softcap"]).tanh()
            if c["bias"]:
                t = t - far * float(s["slopes"][h])
            t[(far < 0) | (far >= (c["window"] or 1 << 40))] = -math.inf
            out[at:at + m, h] = t.softmax(1) @ vv[h // per]
        at += m
    return out.reshape(-1, nh * hd)
