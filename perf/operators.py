"""The paged KV cache's operators, as cases that can be timed and compared.

A decoder's layer appends the keys and values of its new tokens to the pages of
its sequences and attends over what they hold; between steps a scheduler forks,
admits and frees sequences and compacts the pool. One case is one such call:

    append    rope of q and k, and k and v written into their pages
    attn      attention of the new tokens over their sequences' pages
    assign    a scheduling step: sequences forked, admitted and freed
    compact   the live pages moved to the front of the pool, the page tables with them

`run` computes each in plain torch operations in 32 bits (rope's angles in 64),
or, where `own` is set, through the package's kv module. A page of P tokens
holds, for each k/v head of D values, K as [D/8][P][8] (8 values of a token
together) and V as [P/16][2][D][8] (of each 16 tokens, for both halves h, the
tokens 4h..4h+3 and 8+4h..8+4h+3 of a column together).

Sizes: the small shape (hidden 1024: 16 heads of 64), the Qwen3-4B shape (32
query and 8 k/v heads of 128, 36 layers, 8192 tokens in 2048-token chunks), the
27B-class shape (48 query and 8 k/v heads of 128, chunks of 4096), and heads
and groups between them; one sequence to 128, one token to tens of thousands.
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# query heads, k/v heads, head width: the three model shapes
SMALL = dict(q_heads=16, kv_heads=16, head=64)
B4 = dict(q_heads=32, kv_heads=8, head=128)
B27 = dict(q_heads=48, kv_heads=8, head=128)


def _package():
    import importlib.util
    if "ggml_xdna_amd" not in sys.modules:
        pkg = Path(__file__).resolve().parents[1] / "ggml-xdna_amd"
        spec = importlib.util.spec_from_file_location("ggml_xdna_amd", pkg / "__init__.py",
                                                      submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["ggml_xdna_amd"] = mod
        spec.loader.exec_module(mod)
        mod.init(0)
    from ggml_xdna_amd import kv
    return kv


# ---- the cases ----------------------------------------------------------------

def _attn(name, shape, type, page, seqs, new, length, causal=True, window=0, softcap=0.0, ragged=1):
    c = dict(kind="attn", **shape, type=type, page=page, seqs=seqs, new_min=new[0], new_max=new[1], len_min=length[0],
             len_max=length[1], causal=causal, window=window, softcap=softcap, ragged=ragged)
    return dict(c, name=name) if name else c


def _append(name, shape, type, source, page, seqs, new, length, rot, neox, yarn, ragged=1):
    c = dict(kind="append", **shape, type=type, source=source, page=page, seqs=seqs, new_min=new[0], new_max=new[1],
             len_min=length[0], len_max=length[1], rot=rot, neox=neox, yarn=yarn, ragged=ragged)
    return dict(c, name=name) if name else c


def _pages(name, kind, shape, layers, page, seqs, length, ragged=1, **more):
    c = dict(kind=kind, kv_heads=shape["kv_heads"], head=shape["head"], type="bf16", layers=layers, page=page, seqs=seqs,
             len_min=length[0], len_max=length[1], ragged=ragged, **more)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's next token, a short context: the smallest call, all latency
        _attn("attn_decode_1", B4, "bf16", 64, 1, (1, 1), (1000, 1000)),
        # a serving batch's next tokens, contexts from short to the whole prompt
        _attn("attn_decode_64", B4, "bf16", 64, 64, (1, 1), (256, 8192)),
        # the ordinary prefill: the last of four 2048-token chunks of a prompt
        _attn("attn_chunk_2048", B4, "bf16", 64, 1, (2048, 2048), (8192, 8192)),
        # the small model serving prompts and next tokens together, fp16, short pages, a softcap
        _attn("attn_mixed_small", SMALL, "f16", 16, 9, (1, 300), (1, 2500), softcap=30.0, ragged=3),
        # the 27B-class model's first chunk, six query heads a k/v head
        _attn("attn_chunk_27b_4096", B27, "bf16", 128, 1, (4096, 4096), (4096, 4096)),
        # a few drafted tokens checked against long contexts, a sliding window that most of them pass
        _attn("attn_verify_long", B27, "bf16", 64, 4, (5, 5), (20000, 40000), window=32768, ragged=5),
        # a serving batch's next tokens into the cache, NeoX rope
        _append("append_decode_64", B4, "bf16", "f32", 64, 64, (1, 1), (256, 8192), 128, True, False),
        # a prefill chunk's q, k and v as the matmuls give them (fp32), YaRN positions far out
        _append("append_chunk_2048", B4, "bf16", "f32", 64, 1, (2048, 2048), (60000, 60000), 128, True, True),
        # the small model's scheduler: a few sequences forked, admitted, freed
        _pages("assign_small", "assign", SMALL, 16, 16, 12, (20, 200), forks=3, admits=2, frees=2),
        # a step of parallel sampling over the Qwen3-4B shape: every fork copies its open page in all layers
        _pages("assign_4b", "assign", B4, 36, 64, 96, (200, 1500), ragged=2, forks=40, admits=20, frees=20),
        # the small model's pool, a few pages out of place
        _pages("compact_small", "compact", SMALL, 16, 16, 10, (20, 300), ragged=4, spare=0.1),
        # the Qwen3-4B shape's pool after most sequences have ended
        _pages("compact_4b", "compact", B4, 36, 64, 24, (200, 1500), ragged=2, spare=0.6),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _draw_shape(rng):
    if rng.random() < 0.5:
        return dict(rng.choice([SMALL, B4, B4, B27]))
    kv = rng.randint(1, 12)
    return dict(q_heads=kv * rng.randint(1, 8), kv_heads=kv, head=rng.choice([64, 96, 128, 192, 256]))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "append", "assign", "compact"])
    shape, page, ragged = _draw_shape(rng), rng.choice([16, 32, 64, 64, 128, 256]), rng.randrange(1 << 20)
    if kind in ("attn", "append"):
        how = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
        width = shape["kv_heads"] * shape["head"]
        if how in ("decode", "verify"):
            seqs = _log_uniform(rng, 1, 128)
            new = (1, 1) if how == "decode" else (2, rng.randint(3, 8))
            hi = min(_log_uniform(rng, 64, 65536), int(4e8 / (seqs * width)))
        elif how == "chunk":
            seqs, n = 1, _log_uniform(rng, 33, 4096)
            new, hi = (n, n), n + (0 if rng.random() < 0.3 else _log_uniform(rng, 1, 30000))
            hi = max(n, min(hi, int(4e8 / (n * shape["q_heads"]))))
        else:
            seqs, n = rng.randint(2, 12), _log_uniform(rng, 16, 700)
            new, hi = (1, n), n + _log_uniform(rng, 16, 4000)
            hi = max(n, min(hi, int(4e8 / (seqs * n * shape["q_heads"]))))
        lo = hi if seqs == 1 else rng.choice([1, max(1, hi // 8), hi])
        if kind == "attn":
            return _attn(None, shape, rng.choice(["bf16", "f16"]), page, seqs, new, (lo, hi), causal=rng.random() < 0.85,
                         window=_log_uniform(rng, 16, 8192) if rng.random() < 0.25 else 0,
                         softcap=rng.choice([0.0, 0.0, 0.0, 30.0]), ragged=ragged)
        rot = shape["head"] if rng.random() < 0.6 else shape["head"] // 32 * rng.choice([8, 16])
        return _append(None, shape, rng.choice(["bf16", "f16"]), rng.choice(["f32", "f32", "bf16", "f16"]), page, seqs,
                       new, (lo, min(4 * hi, 200000) if seqs == 1 else hi), rot, rng.random() < 0.5,
                       rng.random() < 0.3, ragged=ragged)
    layers = rng.randint(1, 36)
    seqs = _log_uniform(rng, 8, 96)
    lo = rng.randint(1, 200)
    # the pool stays within the largest listed one's: 4e9 bytes
    hi = lo + min(_log_uniform(rng, 16, 4000), int(4e9 / (4 * layers * shape["kv_heads"] * shape["head"] * 2 * seqs)))
    if kind == "assign":
        forks, admits, frees = (rng.randint(0 if i else 1, seqs // 4) for i in range(3))
        return _pages(None, kind, shape, layers, page, seqs, (lo, hi), ragged=ragged, forks=forks, admits=admits, frees=frees)
    return _pages(None, kind, shape, layers, page, seqs, (lo, hi), ragged=ragged, spare=round(rng.uniform(0.05, 0.8), 2))


# ---- inputs -------------------------------------------------------------------

def _lengths(c):
    """The new tokens and the length of each sequence of an attn or append case."""
    rng = random.Random(c["ragged"])
    new, length = [], []
    for _ in range(c["seqs"]):
        n = _log_uniform(rng, c["new_min"], c["new_max"])
        new.append(n)
        length.append(max(n, _log_uniform(rng, c["len_min"], c["len_max"])))
    return new, length


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rope(c):
    """The frequency of each rotated pair, and the magnitude: plain, or YaRN from a 32768-token context by 4."""
    n, base = c["rot"], 1e6 if c["neox"] else 1e4
    f = [base ** (-2.0 * p / n) for p in range(n // 2)]
    if not c["yarn"]:
        return f, 1.0
    first, last = (n * math.log(32768 / (beta * 2 * math.pi)) / (2 * math.log(base)) for beta in (32.0, 1.0))
    first, last = max(0, math.floor(first)), min(n - 1, math.ceil(last))
    for p in range(n // 2):
        ramp = 1.0 - min(1.0, max(0.0, (p - first) / max(0.001, last - first)))
        f[p] *= 0.25 * (1.0 - ramp) + ramp
    return f, 1.0 + 0.1 * math.log(4.0)


def _sequences(c, seed):
    """A batch over one layer's pool: the pages of all sequences dealt out in no order."""
    g = _generator(seed)
    new, length = _lengths(c)
    page, rng = c["page"], random.Random(c["ragged"] + 1)
    count = [-(-n // page) for n in length]
    pages = sum(count) + 3
    ids = list(range(pages))
    rng.shuffle(ids)
    table, at = [], 0
    for n in count:
        table.append(ids[at:at + n] + [-1] * (max(count) - n))
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    refs = [0] * pages
    for i in ids[:at]:
        refs[i] = 1
    s = {"case": c, "starts": _i32(starts), "tables": _i32(table), "lens": _i32(length), "refs": _i32(refs), "rows": starts[-1],
         "max_new": max(new), "max_len": max(length),
         "pool": torch.randn((1, pages, c["kv_heads"], 2 * page * c["head"]), generator=g, device="cuda").to(DTYPES[c["type"]])}
    return s, g


def _scheduled(c):
    """The pages of an assign or compact case's sequences, and the step's entries: all of it by the case alone."""
    rng, page = random.Random(c["ragged"]), c["page"]
    length = [rng.randint(c["len_min"], c["len_max"]) for _ in range(c["seqs"])]
    dst, src, grow = [], [], []
    if c["kind"] == "assign":
        slots = list(range(c["seqs"]))
        rng.shuffle(slots)
        changed = c["forks"] + c["admits"] + c["frees"]
        parents = slots[changed:]
        for i, s in enumerate(slots[:changed]):
            if i < c["forks"] + c["admits"]:
                length[s] = rng.randint(0, 2 * page)  # what an earlier step left in the row
            dst.append(s)
            src.append(rng.choice(parents) if i < c["forks"] else -1)
            grow.append(1 if i < c["forks"] else rng.randint(c["len_min"], c["len_max"]) if i < c["forks"] + c["admits"] else 0)
    count = [-(-n // page) for n in length]
    after = [-(-(g + (length[s] if s >= 0 else 0)) // page) for g, s in zip(grow, src)]
    if c["kind"] == "assign":
        pages = sum(count) + sum(after) + 1
    else:
        pages = int(sum(count) / (1.0 - c["spare"])) + 1
    ids = list(range(pages))
    rng.shuffle(ids)
    cols = max(count + after + [1]) + 1
    table, at = [], 0
    refs = [0] * pages
    for n in count:
        row = ids[at:at + n]
        at += n
        if table and n and rng.random() < 0.2 and table[-1][0] >= 0:  # a prompt's first page shared with the row before
            row[0] = table[-1][0]
        for i in row:
            refs[i] += 1
        table.append(row + [-1] * (cols - n))
    return dict(length=length, table=table, refs=refs, pages=pages, dst=dst, src=src, grow=grow)


def prepare(case, seed):
    c, kind = case, case["kind"]
    if kind in ("attn", "append"):
        s, g = _sequences(c, seed)
        q, kv = (s["rows"], c["q_heads"], c["head"]), (s["rows"], c["kv_heads"], c["head"])
        if kind == "attn":
            s["q"] = (1.5 * torch.randn(q, generator=g, device="cuda")).to(DTYPES[c["type"]])
            return s
        for name, size in (("q", q), ("k", kv), ("v", kv)):
            s[name] = torch.randn(size, generator=g, device="cuda").to(DTYPES[c["source"]])
        f, s["magnitude"] = _rope(c)
        s["freqs"] = torch.tensor(f, dtype=torch.float64, device="cuda")
        return s
    p, g = _scheduled(c), _generator(seed)
    s = {"case": c, "tables": _i32(p["table"]), "lens": _i32(p["length"]), "refs": _i32(p["refs"]),
         "pool": torch.empty((c["layers"], p["pages"], c["kv_heads"], 2 * c["page"] * c["head"]), dtype=DTYPES[c["type"]],
                             device="cuda").normal_(generator=g)}
    if kind == "assign":
        s.update(dst=_i32(p["dst"]), src=_i32(p["src"]), grow=_i32(p["grow"]))
    else:
        s.update(new_tables=torch.empty_like(s["tables"]), new_refs=torch.empty_like(s["refs"]))
    return s


# ---- one pass, in plain operations ----------------------------------------------

def _rows_of(s):
    """The sequence and the place in it of every row of a batch."""
    t = torch.arange(s["rows"], device="cuda")
    seq = (t[:, None] >= s["starts"][1:][None, :]).sum(dim=1)
    return seq, t - s["starts"][seq]


def _plain_attn(c, s):
    heads, d, page, b = c["kv_heads"], c["head"], c["page"], c["seqs"]
    group, n = c["q_heads"] // heads, s["max_new"]
    held = s["pool"][0][s["tables"].clamp(min=0).long()]  # [seqs][columns][heads][2 * page * d]
    cols = held.shape[1]
    k = held[..., :page * d].reshape(b, cols, heads, d // 8, page, 8).permute(0, 2, 1, 4, 3, 5)
    v = held[..., page * d:].reshape(b, cols, heads, page // 16, 2, d, 2, 4).permute(0, 2, 1, 3, 6, 4, 7, 5)
    k, v = (x.reshape(b, heads, cols * page, d).float() for x in (k, v))
    starts, lens = s["starts"].long(), s["lens"].long()
    new = starts[1:] - starts[:-1]
    i = torch.arange(n, device="cuda")
    q = s["q"][(starts[:-1, None] + i).clamp(max=s["rows"] - 1)].float()  # [seqs][n][query heads][d]
    q = q.reshape(b, n, heads, group, d).permute(0, 2, 1, 3, 4).reshape(b, heads, n * group, d)
    x = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    t = torch.arange(cols * page, device="cuda")
    pos = (lens - new)[:, None] + i  # [seqs][n]
    ok = (t < lens[:, None])[:, None, :].expand(b, n, cols * page)
    if c["causal"]:
        ok = ok & (t <= pos[:, :, None])
    if c["window"]:
        ok = ok & (t > pos[:, :, None] - c["window"])
    ok = ok[:, None, :, None, :]
    x = x.reshape(b, heads, n, group, cols * page).masked_fill_(~ok, -math.inf)
    top = x.amax(dim=4, keepdim=True)
    x = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = x.sum(dim=4, keepdim=True)
    x = torch.matmul(x.reshape(b, heads, n * group, cols * page), v).reshape(b, heads, n, group, d)
    x = torch.where(total > 0, x / total, torch.zeros_like(x))
    seq, at = _rows_of(s)
    return x.permute(0, 2, 1, 3, 4)[seq, at].reshape(s["rows"], c["q_heads"], d).to(DTYPES[c["type"]])


def _turned(x, a, c, magnitude):
    """The first `rot` values of every head turned by the angles a[row][pair]."""
    x, cos, sin = x.float(), (torch.cos(a) * magnitude).float()[:, None], (torch.sin(a) * magnitude).float()[:, None]
    r, half = c["rot"], c["rot"] // 2
    x0, x1 = (x[..., :half], x[..., half:r]) if c["neox"] else (x[..., 0:r:2], x[..., 1:r:2])
    y0, y1 = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    y = torch.cat([y0, y1], dim=2) if c["neox"] else torch.stack([y0, y1], dim=3).reshape(x.shape[0], x.shape[1], r)
    return torch.cat([y, x[..., r:]], dim=2)


def _plain_append(c, s):
    d, page, dtype = c["head"], c["page"], DTYPES[c["type"]]
    seq, at = _rows_of(s)
    lens, starts = s["lens"].long(), s["starts"].long()
    place = (lens - (starts[1:] - starts[:-1]))[seq] + at
    a = place.double()[:, None] * s["freqs"]
    q, k = (_turned(s[n], a, c, s["magnitude"]).to(dtype) for n in ("q", "k"))
    t, e = place % page, torch.arange(d, device="cuda")
    base = s["tables"].long()[seq, place // page][:, None] * c["kv_heads"] + torch.arange(c["kv_heads"], device="cuda")
    base = (base * (2 * page * d))[:, :, None]
    k_at = (e // 8) * (page * 8) + t[:, None] * 8 + e % 8
    v_at = page * d + ((t // 16 * 2 + t // 4 % 2)[:, None] * d + e) * 8 + (t % 4 + t // 8 % 2 * 4)[:, None]
    flat = s["pool"].view(-1)
    flat[base + k_at[:, None]] = k
    flat[base + v_at[:, None]] = s["v"].to(dtype)
    return q, s["pool"]


def _plain_assign(c, s):
    page, (seqs, cols) = c["page"], s["tables"].shape
    tables, lens, refs = s["tables"].long(), s["lens"].long(), s["refs"].long()
    dst, src, grow = s["dst"].long(), s["src"].long(), s["grow"].long()
    col = torch.arange(cols, device="cuda")
    forked = src >= 0
    # the rows' former pages are released
    had = col < ((lens[dst] + page - 1) // page)[:, None]
    refs = refs.scatter_add(0, tables[dst].clamp(min=0).reshape(-1), -had.long().reshape(-1))
    # the pages a fork shares, and how many the step takes
    base = torch.where(forked, lens[src.clamp(min=0)], torch.zeros_like(src))
    shared, total = base // page, (base + grow + page - 1) // page
    need = total - shared
    first = torch.cumsum(need, dim=0) - need
    free = torch.argsort((refs > 0).long(), stable=True)  # the free pages, lowest first, then the others
    parent = tables[src.clamp(min=0)]
    fresh = free[(first[:, None] + col - shared[:, None]).clamp(0, free.numel() - 1)]
    row = torch.where(col < shared[:, None], parent, torch.where(col < total[:, None], fresh, torch.full_like(fresh, -1)))
    refs = refs.scatter_add(0, row.clamp(min=0).reshape(-1), (row >= 0).long().reshape(-1))
    # the open page of a fork's parent is copied
    opened = forked & (base % page > 0)
    pick = opened.nonzero()[:, 0]
    at = shared[pick]
    s["pool"][:, row[pick, at]] = s["pool"][:, parent[pick, at]]
    s["tables"][dst] = row.int()
    s["lens"][dst] = (base + grow).int()
    s["refs"].copy_(refs)
    return s["pool"], s["refs"], s["tables"], s["lens"]


def _plain_compact(c, s):
    refs, tables = s["refs"], s["tables"].long()
    live = refs > 0
    n = live.sum()
    ids = torch.arange(refs.numel(), device="cuda")
    to, moved = (~live & (ids < n)).nonzero()[:, 0], (live & (ids >= n)).nonzero()[:, 0]
    s["pool"][:, to] = s["pool"][:, moved]
    place = ids.clone()
    place[moved] = to
    s["new_refs"].copy_(refs)
    s["new_refs"][to] = refs[moved]
    s["new_refs"][moved] = 0
    s["new_tables"].copy_(torch.where(tables >= 0, place[tables.clamp(min=0)], tables))
    return s["pool"], s["new_refs"], s["new_tables"], n.int().reshape(1)


# ---- one pass, through the package ------------------------------------------------

def _handles(c, s):
    """What a program keeps beside its tensors: the cache and the batch, made once."""
    kv = _package()
    s["kv"] = kv
    s["cache"] = kv.Cache(s["pool"], s["tables"], s["lens"], s["refs"], c["page"], c["head"])
    if "starts" in s:
        s["batch"] = kv.Batch(s["starts"], s["rows"], s["max_new"], s["max_len"])
    if "freqs" in s:
        s["rope"] = kv.Rope(s["freqs"], kv.ROPE_NEOX if c["neox"] else kv.ROPE_NORMAL, s["magnitude"])


def _own(c, s):
    if "kv" not in s:
        _handles(c, s)
    kv, cache = s["kv"], s["cache"]
    if c["kind"] == "attn":
        return kv.attention(cache, 0, s["batch"], s["q"], 1.0 / math.sqrt(c["head"]), causal=c["causal"], window=c["window"],
                            softcap=c["softcap"])
    if c["kind"] == "append":
        return kv.append(cache, 0, s["batch"], s["k"], s["v"], q=s["q"], rope=s["rope"]), s["pool"]
    if c["kind"] == "assign":
        kv.assign(cache, s["dst"], s["src"], s["grow"])
        return s["pool"], s["refs"], s["tables"], s["lens"]
    live = kv.compact(cache, refs=s["new_refs"], tables=s["new_tables"])
    return s["pool"], s["new_refs"], s["new_tables"], live


def run(state):
    c = state["case"]
    if own:
        return _own(c, state)
    return {"attn": _plain_attn, "append": _plain_append, "assign": _plain_assign, "compact": _plain_compact}[c["kind"]](c, state)


# ---- what a pass cannot do without ----------------------------------------------

def _span(c, n, length):
    """The pairs of a sequence's new tokens with the tokens they see, and the tokens that any of them sees."""
    pairs, first = 0, length
    for i in range(n):
        pos = length - n + i
        hi = min(length, pos + 1) if c["causal"] else length
        lo = max(0, pos - c["window"] + 1) if c["window"] else 0
        if hi > lo:
            pairs, first = pairs + hi - lo, min(first, lo)
    return pairs, length - first


def work(case):
    c, kind, d = case, case["kind"], case["head"]
    if kind in ("attn", "append"):
        new, length = _lengths(c)
        rows = sum(new)
        if kind == "append":
            values = rows * (c["q_heads"] + 2 * c["kv_heads"]) * d
            return {"bytes": values * (DTYPES[c["source"]].itemsize + 2), "flops": 3.0 * rows * (c["q_heads"] + c["kv_heads"]) * c["rot"]}
        spans = [_span(c, n, m) for n, m in zip(new, length)]
        return {"bytes": 4.0 * rows * c["q_heads"] * d + 4.0 * c["kv_heads"] * d * sum(t for _, t in spans),
                "flops": 4.0 * d * c["q_heads"] * sum(p for p, _ in spans)}
    p = _scheduled(c)
    size = 4.0 * c["layers"] * c["kv_heads"] * c["page"] * d  # one page, all layers
    if kind == "assign":
        copies = sum(1 for s in p["src"] if s >= 0 and p["length"][s] % c["page"])
        entries = sum(-(-p["length"][s] // c["page"]) for s in p["dst"]) + sum(-(-p["length"][s] // c["page"]) for s in p["src"] if s >= 0)
        return {"bytes": 2 * copies * size + 4.0 * (2 * p["pages"] + 2 * entries + 4 * len(p["dst"])), "flops": 0.0}
    n = sum(1 for r in p["refs"] if r > 0)
    moves = sum(1 for r in p["refs"][n:] if r > 0)
    return {"bytes": 2 * moves * size + 8.0 * (p["pages"] + len(p["table"]) * len(p["table"][0])), "flops": 0.0}


# ---- the same in 64 bits, from the definitions --------------------------------------

def _exact_attn(c, s):
    """One sequence and one k/v head at a time; each token's keys and values picked out by their offsets."""
    d, page, group = c["head"], c["page"], c["q_heads"] // c["kv_heads"]
    new, length = _lengths(c)
    out = torch.zeros((s["rows"], c["q_heads"], d), dtype=torch.float64, device="cuda")
    e, row = torch.arange(d, device="cuda"), 0
    for b, (n, m) in enumerate(zip(new, length)):
        t = torch.arange(m, device="cuda")
        held, u = s["tables"][b].long()[t // page], t % page
        k_at = (torch.div(e, 8, rounding_mode="floor") * page)[None, :] * 8 + u[:, None] * 8 + (e % 8)[None, :]
        half, inner = (u >> 2) & 1, (u & 3) | (((u >> 3) & 1) << 2)
        v_at = page * d + (((u >> 4) * 2 + half)[:, None] * d + e[None, :]) * 8 + inner[:, None]
        for h in range(c["kv_heads"]):
            flat = s["pool"][0, :, h]
            k, v = flat[held[:, None], k_at].double(), flat[held[:, None], v_at].double()
            for r in range(0, n, 1024):
                i = torch.arange(r, min(n, r + 1024), device="cuda")
                q = s["q"][row + i, h * group:(h + 1) * group].double()
                x = (q.reshape(-1, d) @ k.T).reshape(len(i), group, m) / math.sqrt(d)
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                at = m - n + i
                hidden = torch.zeros((len(i), m), dtype=torch.bool, device="cuda")
                if c["causal"]:
                    hidden |= t[None, :] > at[:, None]
                if c["window"]:
                    hidden |= t[None, :] <= at[:, None] - c["window"]
                x[hidden[:, None, :].expand_as(x)] = -math.inf
                p = torch.nan_to_num(torch.softmax(x, dim=2))
                out[row + i, h * group:(h + 1) * group] = (p.reshape(-1, m) @ v).reshape(len(i), group, d)
        row += n
    return out


def _exact_append(c, s):
    """Every value's own place, a token at a time in its sequence's pages."""
    d, page, r = c["head"], c["page"], c["rot"]
    new, length = _lengths(c)
    place = np.concatenate([np.arange(m - n, m) for n, m in zip(new, length)])
    seq = np.concatenate([np.full(n, b) for b, n in enumerate(new)])
    f, magnitude = _rope(c)
    a = place[:, None].astype(np.float64) * np.array(f)
    turn = torch.from_numpy(magnitude * np.exp(1j * a)).cuda()[:, None, :]
    got = {}
    for n in ("q", "k"):
        x = s[n].double()
        pairs = torch.stack([x[..., :r // 2], x[..., r // 2:r]], dim=3) if c["neox"] else x[..., :r].unflatten(2, (r // 2, 2))
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y = torch.cat([y[..., 0], y[..., 1]], dim=2) if c["neox"] else y.flatten(2)
        got[n] = torch.cat([y, x[..., r:]], dim=2)
    pool = s["pool"].double()
    held = torch.from_numpy(s["tables"].cpu().numpy()[seq, place // page].astype(np.int64)).cuda()
    u = torch.from_numpy(place % page).cuda()
    k = pool[0, :, :, :page * d].unflatten(2, (d // 8, page, 8))
    k[held, :, :, u] = got["k"].unflatten(2, (d // 8, 8))
    v = pool[0, :, :, page * d:].unflatten(2, (page // 16, 2, d, 2, 4))
    v[held, :, u // 16, u // 4 % 2, :, u // 8 % 2, u % 4] = s["v"].double()
    return got["q"], pool


def _exact_assign(c, s):
    """One entry after the other: a host's bookkeeping."""
    page = c["page"]
    tables, lens, refs = (s[n].cpu().numpy().copy() for n in ("tables", "lens", "refs"))
    entries = list(zip(*(s[n].cpu().tolist() for n in ("dst", "src", "grow"))))
    pool = s["pool"].double()
    for dst, _, _ in entries:
        for j in range(-(-int(lens[dst]) // page)):
            refs[tables[dst, j]] -= 1
        tables[dst], lens[dst] = -1, 0
    free = [i for i in range(len(refs)) if refs[i] == 0]
    for dst, src, grow in entries:
        m = int(lens[src]) if src >= 0 else 0
        for j in range(-(-(m + grow) // page)):
            if j < m // page:
                tables[dst, j] = tables[src, j]
            else:
                tables[dst, j] = free.pop(0)
                if j * page < m:
                    pool[:, int(tables[dst, j])] = pool[:, int(tables[src, j])]
            refs[tables[dst, j]] += 1
        lens[dst] = m + grow
    return pool, refs, tables, lens


def _exact_compact(c, s):
    """The live pages past the last place, each into the first free one."""
    tables, refs = s["tables"].cpu().numpy().copy(), s["refs"].cpu().numpy().copy()
    n = int((refs > 0).sum())
    pool, hole = s["pool"].double(), 0
    before = tables.copy()
    for i in range(n, len(refs)):
        if refs[i] > 0:
            while refs[hole] > 0:
                hole += 1
            pool[:, hole] = pool[:, i]
            refs[hole], refs[i] = refs[i], 0
            tables[before == i] = hole
    return pool, refs, tables, n


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "append": _exact_append, "assign": _exact_assign, "compact": _exact_compact}[case["kind"]](case, s)
