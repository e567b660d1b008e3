"""The operators of a decoding step, as cases that can be timed and compared.

After a prompt a decoder makes one token a sequence and step (or checks a few
drafted ones): products of few rows with the quantised weights, attention over
contexts that parallel samples of one prompt share, and the choice of the next
token from the logits. One case is one such call:

    matvec   y = x W^T (+ a residual) for one or more GGUF weights on one x, or the
             GLU of two, x of a few rows
    shared   attention over a paged KV cache whose sequences name the same leading
             pages in groups
    sample   temperature, top-k, top-p, min-p and the draw from a given random
             number, a token a row

`run` computes each in plain torch operations in 32 bits (the sampler in 64: a
draw lies next to a border of the sums), or, where `own` is set, through the
package. The weights are GGUF rows as a model file holds them; a page of P
tokens holds, for each k/v head of D values, K as [D/8][P][8] (8 values of a
token together) and V as [P/16][2][D][8] (of each 16 tokens, for both halves h,
the tokens 4h..4h+3 and 8+4h..8+4h+3 of a column together).

Sizes: the small shape (hidden 1024, 16 heads of 64), the Qwen3-4B shape (hidden
2560, FFN 9728, 32 query and 8 k/v heads of 128, a vocabulary of 151936) and the
27B-class shape (hidden 5120, FFN 17408, 48 query heads), and sizes between.
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

# GGUF type number, values and bytes of a block
BLOCKS = {"q4_0": (2, 32, 18), "q4_1": (3, 32, 20), "q8_0": (8, 32, 34), "q4_k": (12, 256, 144), "iq4_nl": (20, 32, 18),
          "iq4_xs": (23, 256, 136)}
# the published levels of IQ4_NL and IQ4_XS
LEVELS = [-127, -104, -83, -65, -49, -35, -22, -10, 1, 13, 25, 38, 53, 69, 89, 113]


def _package(name=None):
    import importlib
    import importlib.util
    if "ggml_xdna_amd" not in sys.modules:
        pkg = Path(__file__).resolve().parents[1] / "ggml-xdna_amd"
        spec = importlib.util.spec_from_file_location("ggml_xdna_amd", pkg / "__init__.py",
                                                      submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["ggml_xdna_amd"] = mod
        spec.loader.exec_module(mod)
        mod.init(0)
    return importlib.import_module("ggml_xdna_amd" + ("." + name if name else ""))


# ---- the cases ----------------------------------------------------------------

def _matvec(name, type, rows, k, ns, residual=False, glu=False, outliers=0.0):
    c = dict(kind="matvec", type=type, rows=rows, k=k, weights=len(ns), residual=residual, glu=glu, outliers=outliers)
    c.update({"n%d" % i: n for i, n in enumerate(ns)})
    return dict(c, name=name) if name else c


def _shared(name, shape, type, page, groups, members, alone, shared, more, new=(1, 1), window=0, softcap=0.0, ragged=1):
    """groups prompts with `members` samples each, and `alone` sequences of their own. A prompt has shared[0..1] tokens, a
    sample more[0..1] tokens beyond it, of which new[0..1] are this call's."""
    c = dict(kind="shared", **shape, type=type, page=page, groups=groups, members=members, alone=alone, shared_min=shared[0],
             shared_max=shared[1], more_min=more[0], more_max=more[1], new_min=new[0], new_max=new[1], window=window,
             softcap=softcap, ragged=ragged)
    return dict(c, name=name) if name else c


def _sample(name, type, rows, vocab, temperature=(1.0, 1.0), top_k=(0, 0), top_p=(1.0, 1.0), min_p=(0.0, 0.0), spread=2.5,
            gone=0.0, greedy=0.0):
    """Parameters between the two values, a row each; greedy: the share of rows at temperature 0; gone: of logits at -inf."""
    c = dict(kind="sample", type=type, rows=rows, vocab=vocab, t_min=temperature[0], t_max=temperature[1], k_min=top_k[0],
             k_max=top_k[1], p_min=top_p[0], p_max=top_p[1], m_min=min_p[0], m_max=min_p[1], spread=spread, gone=gone,
             greedy=greedy)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the small model's O projection for three sequences, its residual added: the smallest call
        _matvec("matvec_small_3", "q4_0", 3, 1024, [1024], residual=True),
        # one user's next token: q, k and v of the Qwen3-4B shape on one normed row
        _matvec("matvec_qkv_1", "q4_k", 1, 2560, [4096, 1024, 1024]),
        # the same layer's down projection, eight bits, its residual added
        _matvec("matvec_down_1", "q8_0", 1, 9728, [2560], residual=True),
        # the 27B-class model's gate and up for four drafted tokens, outlier channels
        _matvec("matvec_glu_27b_4", "q4_k", 4, 5120, [17408, 17408], glu=True, outliers=0.005),
        # the output projection over the vocabulary for a batch of 16
        _matvec("matvec_logits_16", "iq4_xs", 16, 2560, [151936]),
        # 64 samples of one long prompt, each some way into its answer
        _shared("shared_4b_64", B4, "bf16", 64, 1, 64, 0, (8192, 8192), (1, 512)),
        # the small model serving three prompts, four samples each, and three sequences of their own
        _shared("shared_small", SMALL, "f16", 16, 3, 4, 3, (100, 2000), (1, 300), softcap=30.0, ragged=3),
        # five drafted tokens of 16 samples of a very long prompt
        _shared("shared_27b_verify", B27, "bf16", 128, 1, 16, 0, (32000, 32000), (5, 1000), new=(5, 5), ragged=5),
        # a small vocabulary, every parameter in use, some rows greedy: latency
        _sample("sample_small", "f16", 3, 1003, (0.5, 1.5), (5, 100), (0.5, 0.95), (0.0, 0.1), gone=0.1, greedy=0.4),
        # one user's next token with the parameters a chat program sets
        _sample("sample_1", "f32", 1, 151936, (0.7, 0.7), (20, 20), (0.8, 0.8)),
        # a serving batch with nucleus sampling alone
        _sample("sample_64", "f32", 64, 151936, (0.6, 1.2), (0, 0), (0.9, 0.98)),
        # a large batch of bf16 logits, min-p alone
        _sample("sample_256_bf16", "bf16", 256, 151936, (0.8, 1.5), (0, 0), (1.0, 1.0), (0.01, 0.1)),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _draw_matvec(rng):
    type = rng.choice(list(BLOCKS))
    block = BLOCKS[type][1]
    k = block * _log_uniform(rng, max(1, 256 // block), 17408 // block)
    glu = rng.random() < 0.25
    ns, most = [], 3.8e8 / k
    for _ in range(1 if glu else rng.choice([1, 1, 2, 3, 4])):
        ns.append(_log_uniform(rng, 16, int(max(16, min(152000, most / (8 if glu else 4))))))
    return _matvec(None, type, rng.choice([1, 1, 2, 3, 4, 5, 8, rng.randint(1, 16)]), k, ns * 2 if glu else ns,
                   residual=not glu and rng.random() < 0.4, glu=glu, outliers=rng.choice([0.0, 0.005]))


def _draw_shared(rng):
    shape = dict(rng.choice([SMALL, B4, B27]))
    if rng.random() < 0.4:
        kv = rng.randint(1, 12)
        shape = dict(q_heads=kv * rng.randint(1, 8), kv_heads=kv, head=rng.choice([64, 96, 128, 192, 256]))
    groups, members = rng.randint(1, 4), _log_uniform(rng, 2, 64)
    alone = rng.choice([0, 0, rng.randint(1, 6)])
    seqs = groups * members + alone
    new = rng.choice([(1, 1), (1, 1), (2, 5), (1, _log_uniform(rng, 2, 40))])
    # no more keys and values, all sequences' and the distinct ones, and no more rows than the largest listed cases have
    width = shape["kv_heads"] * shape["head"]
    most = min(5e8 / (2 * seqs * width), 2.5e7 / ((groups + alone) * width), 1.5e9 / (seqs * new[1] * shape["q_heads"]))
    shared = max(4, min(_log_uniform(rng, 64, 33000), int(most)))
    more = new[1] + min(_log_uniform(rng, 1, 1500), shared, int(2.5e7 / (seqs * width)))
    return _shared(None, shape, rng.choice(["bf16", "f16"]), rng.choice([16, 32, 64, 64, 128, 256]), groups, members, alone,
                   (rng.choice([shared, max(1, shared // 4)]), shared), (new[1], more), new,
                   window=_log_uniform(rng, 64, 8192) if rng.random() < 0.15 else 0, softcap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                   ragged=rng.randrange(1 << 20))


def _draw_sample(rng):
    vocab = _log_uniform(rng, 100, 262144)
    rows = min(_log_uniform(rng, 1, 256), int(3.8e7 / vocab))
    t, k, p, m = rng.uniform(0.3, 1.5), _log_uniform(rng, 1, 300), rng.uniform(0.3, 0.99), rng.uniform(0.001, 0.2)
    return _sample(None, rng.choice(["f32", "f32", "bf16", "f16"]), max(1, rows), vocab, (t, t * rng.choice([1.0, 1.5])),
                   rng.choice([(0, 0), (k, 2 * k)]), rng.choice([(1.0, 1.0), (p, min(1.0, p + 0.05))]),
                   rng.choice([(0.0, 0.0), (m, 2 * m)]), spread=round(rng.uniform(0.5, 4.0), 3), gone=rng.choice([0.0, 0.0, 0.3]),
                   greedy=rng.choice([0.0, 0.0, 0.2]))


def draw(rng):
    return rng.choice([_draw_matvec, _draw_shared, _draw_sample])(rng)


# ---- inputs -------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rand(g, *size):
    return torch.rand(size, generator=g, device="cuda")


def _bytes(g, *size, high=256):
    return torch.randint(0, high, size, generator=g, device="cuda", dtype=torch.uint8)


def _halves(v):
    """Values as the bytes of their fp16."""
    return v.half()[..., None].view(torch.uint8)


def _ns(c):
    return [c["n%d" % i] for i in range(c["weights"])]


def _weight(type, n, k, g):
    """GGUF rows [n][bytes]: codes of all values, scales within a factor of four, so that a weight is about 0.02."""
    _, values, size = BLOCKS[type]
    b = k // values
    d = 0.5 + 1.5 * _rand(g, n, b)
    if type in ("q4_0", "iq4_nl"):
        return torch.cat([_halves(d * (0.004 if type == "q4_0" else 0.0003)), _bytes(g, n, b, 16)], dim=2).reshape(n, -1)
    if type == "q4_1":
        return torch.cat([_halves(0.004 * d), _halves(-0.03 * d), _bytes(g, n, b, 16)], dim=2).reshape(n, -1)
    if type == "q8_0":
        return torch.cat([_halves(0.0003 * d), _bytes(g, n, b, 32)], dim=2).reshape(n, -1)
    if type == "iq4_xs":  # a scale of 2 bits above and 4 below for each 32 values
        return torch.cat([_halves(0.00002 * d), _bytes(g, n, b, 6), _bytes(g, n, b, 128)], dim=2).reshape(n, -1)
    # q4_k: 6-bit scales and minima about as large as the scales, packed in 12 bytes
    sc = _bytes(g, n, b, 8, high=64)
    m = (sc.int() + torch.randint(-4, 5, (n, b, 8), generator=g, device="cuda")).clamp(0, 63).to(torch.uint8)
    packed = torch.cat([sc[..., :4] | (sc[..., 4:] >> 4) << 6, m[..., :4] | (m[..., 4:] >> 4) << 6, sc[..., 4:] & 15 | (m[..., 4:] & 15) << 4],
                       dim=2)
    return torch.cat([_halves(0.0001 * d), _halves(0.00075 * d), packed, _bytes(g, n, b, 128)], dim=2).reshape(n, -1)


def _prepare_matvec(c, g):
    x = torch.randn((c["rows"], c["k"]), generator=g, device="cuda")
    if c["outliers"]:
        channels = torch.randperm(c["k"], generator=g, device="cuda")[:max(1, int(c["outliers"] * c["k"]))]
        x[:, channels] *= 30.0
    s = {"case": c, "x": x, "w": [_weight(c["type"], n, c["k"], g) for n in _ns(c)]}
    if c["residual"]:
        s["res"] = [torch.randn((c["rows"], n), generator=g, device="cuda") for n in _ns(c)]
    return s


def _lengths(c):
    """Of each sequence: the pages it shares with its group, its length and its new tokens; by the case alone."""
    rng, page = random.Random(c["ragged"]), c["page"]
    shared, length, new = [], [], []
    for i in range(c["groups"] + c["alone"]):
        prompt = _log_uniform(rng, c["shared_min"], c["shared_max"])
        for _ in range(c["members"] if i < c["groups"] else 1):
            more = _log_uniform(rng, c["more_min"], c["more_max"])
            shared.append(prompt // page if i < c["groups"] else 0)
            length.append(prompt + more)
            new.append(min(more, _log_uniform(rng, c["new_min"], c["new_max"])))
    return shared, length, new


def _prepare_shared(c, g):
    """One layer's pool, the pages dealt out in no order; the members of a group name its first member's leading pages."""
    shared, length, new = _lengths(c)
    page, rng = c["page"], random.Random(c["ragged"] + 1)
    count = [-(-n // page) for n in length]
    lead = [b < c["groups"] * c["members"] and b % c["members"] > 0 for b in range(len(length))]
    pages = sum(n - (s if f else 0) for n, s, f in zip(count, shared, lead)) + 3
    ids = list(range(pages))
    rng.shuffle(ids)
    table, refs, at = [], [0] * pages, 0
    for n, s, f in zip(count, shared, lead):
        row = table[-1][:s] if f else []
        row = row + ids[at:at + n - len(row)]
        at += n - (s if f else 0)
        for i in row:
            refs[i] += 1
        table.append(row)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    pool = torch.randn((1, pages, c["kv_heads"], 2 * page * c["head"]), generator=g, device="cuda").to(DTYPES[c["type"]])
    q = 1.5 * torch.randn((starts[-1], c["q_heads"], c["head"]), generator=g, device="cuda")
    return {"case": c, "pool": pool, "q": q.to(DTYPES[c["type"]]), "tables": _i32([r + [-1] * (max(count) - len(r)) for r in table]),
            "lens": _i32(length), "refs": _i32(refs), "starts": _i32(starts), "rows": starts[-1], "max_new": max(new),
            "max_len": max(length), "groups": _i32([i * c["members"] for i in range(c["groups"] + 1)]),
            "max_shared": max(shared) * page}


def _prepare_sample(c, g):
    rows, vocab = c["rows"], c["vocab"]
    x = c["spread"] * torch.randn((rows, vocab), generator=g, device="cuda")
    # a few tokens stand out, as a model's do
    peaks = torch.randint(0, vocab, (rows, 6), generator=g, device="cuda")
    x.scatter_(1, peaks, 2.0 * c["spread"] + c["spread"] * 2.0 * _rand(g, rows, 6))
    if c["gone"]:
        x[_rand(g, rows, vocab) < c["gone"]] = -math.inf
        x.scatter_(1, peaks[:, :1], 1.0)
    between = lambda lo, hi: lo + (hi - lo) * _rand(g, rows)  # noqa: E731
    s = {"case": c, "logits": x.to(DTYPES[c["type"]]), "u": _rand(g, rows), "temperature": between(c["t_min"], c["t_max"])}
    if c["greedy"]:
        s["temperature"][_rand(g, rows) < c["greedy"]] = 0.0
    if c["k_max"]:
        s["top_k"] = between(c["k_min"], c["k_max"] + 0.99).int()
    if c["p_min"] < 1.0:
        s["top_p"] = between(c["p_min"], c["p_max"])
    if c["m_max"] > 0.0:
        s["min_p"] = between(c["m_min"], c["m_max"])
    return s


def prepare(case, seed):
    return {"matvec": _prepare_matvec, "shared": _prepare_shared, "sample": _prepare_sample}[case["kind"]](case, _generator(seed))


# ---- one pass, in plain operations ----------------------------------------------

def _half_at(b, at):
    return b[..., at:at + 2].contiguous().view(torch.float16).float()


def _nibbles(q):
    """The low, then the high halves of each run of bytes."""
    return torch.cat([q & 15, q >> 4], dim=-1)


def _dequantised(type, raw, k):
    """GGUF rows as fp32 values [n][k]."""
    n, (_, values, size) = raw.shape[0], BLOCKS[type]
    b = raw.reshape(n, k // values, size)
    d = _half_at(b, 0)
    if type == "q8_0":
        w = d * b[..., 2:].contiguous().view(torch.int8).float()
    elif type == "q4_0":
        w = d * (_nibbles(b[..., 2:]).float() - 8.0)
    elif type == "q4_1":
        w = d * _nibbles(b[..., 4:]).float() + _half_at(b, 2)
    elif type == "iq4_nl":
        w = d * torch.tensor(LEVELS, dtype=torch.float32, device=raw.device)[_nibbles(b[..., 2:]).int()]
    elif type == "iq4_xs":
        high = b[..., 2:3].int() | b[..., 3:4].int() << 8
        j = torch.arange(8, device=raw.device)
        low = torch.stack([b[..., 4:8] & 15, b[..., 4:8] >> 4], dim=-1).flatten(-2).int()
        scale = d * ((low | (high >> 2 * j & 3) << 4) - 32).float()
        q = _nibbles(b[..., 8:].unflatten(-1, (8, 16))).int()
        w = scale[..., None] * torch.tensor(LEVELS, dtype=torch.float32, device=raw.device)[q]
    else:
        s = b[..., 4:16]
        sc = torch.cat([s[..., :4] & 63, s[..., 8:] & 15 | s[..., :4] >> 6 << 4], dim=-1).float()
        m = torch.cat([s[..., 4:8] & 63, s[..., 8:] >> 4 | s[..., 4:8] >> 6 << 4], dim=-1).float()
        q = _nibbles(b[..., 16:].unflatten(-1, (4, 32))).reshape(n, k // 256, 8, 32).float()
        w = (d * sc)[..., None] * q - (_half_at(b, 2) * m)[..., None]
    return w.reshape(n, k)


def _plain_matvec(c, s):
    y = [s["x"] @ _dequantised(c["type"], w, c["k"]).T for w in s["w"]]
    if c["glu"]:
        return [y[0] * torch.sigmoid(y[0]) * y[1]]
    return [a + r for a, r in zip(y, s["res"])] if c["residual"] else y


def _plain_shared(c, s):
    heads, d, page = c["kv_heads"], c["head"], c["page"]
    group, n, b = c["q_heads"] // heads, s["max_new"], s["lens"].numel()
    held = s["pool"][0][s["tables"].clamp(min=0).long()]  # [seqs][columns][heads][2 * page * d]
    cols = held.shape[1]
    k = held[..., :page * d].reshape(b, cols, heads, d // 8, page, 8).permute(0, 2, 1, 4, 3, 5)
    v = held[..., page * d:].reshape(b, cols, heads, page // 16, 2, d, 2, 4).permute(0, 2, 1, 3, 6, 4, 7, 5)
    k, v = (x.reshape(b, heads, cols * page, d).float() for x in (k, v))
    starts, lens = s["starts"].long(), s["lens"].long()
    i, t = torch.arange(n, device="cuda"), torch.arange(cols * page, device="cuda")
    q = s["q"][(starts[:-1, None] + i).clamp(max=s["rows"] - 1)].float()  # [seqs][n][query heads][d]
    q = q.reshape(b, n, heads, group, d).permute(0, 2, 1, 3, 4).reshape(b, heads, n * group, d)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    at = (lens - starts[1:] + starts[:-1])[:, None] + i  # [seqs][n]
    ok = (t < lens[:, None])[:, None] & (t <= at[:, :, None])
    if c["window"]:
        ok = ok & (t > at[:, :, None] - c["window"])
    x = x.reshape(b, heads, n, group, cols * page).masked_fill_(~ok[:, None, :, None, :], -math.inf)
    x = torch.exp(x - x.amax(dim=4, keepdim=True).clamp(min=-3e38))
    total = x.sum(dim=4, keepdim=True)
    x = torch.matmul(x.reshape(b, heads, n * group, cols * page), v).reshape(b, heads, n, group, d)
    x = torch.where(total > 0, x / total, torch.zeros_like(x))
    row = torch.arange(s["rows"], device="cuda")
    seq = (row[:, None] >= s["starts"][1:][None, :]).sum(dim=1)
    return x.permute(0, 2, 1, 3, 4)[seq, row - starts[seq]].reshape(s["rows"], c["q_heads"], d).to(DTYPES[c["type"]])


def _plain_sample(c, s):
    x = s["logits"].double()
    rows, vocab = x.shape
    every = torch.ones((rows, 1), dtype=torch.float64, device="cuda")
    param = lambda name, off: s[name].double()[:, None] if name in s else off * every  # noqa: E731
    t, p, m = param("temperature", 1.0), param("top_p", 1.0), param("min_p", 0.0)
    k = torch.where(t > 0, param("top_k", vocab), every)  # at temperature 0 the largest alone
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.where(x == x[:, :1], every, torch.exp((x - x[:, :1]) / torch.where(t > 0, t, every)))
    w = w * (torch.arange(vocab, device="cuda") < k)
    upto = torch.cumsum(w, dim=1)
    w = w * ((p >= 1) | (upto - w < p * upto[:, -1:])) * (w >= m)
    w = torch.zeros_like(w).scatter_(1, order, w)
    upto = torch.cumsum(w, dim=1)
    token = ((upto <= s["u"].double()[:, None] * upto[:, -1:]) | (w == 0)).int()
    token = token.argmin(dim=1)  # the first that passes u
    w = w.gather(1, token[:, None])[:, 0]
    return token.int(), (w / upto[:, -1]).float()


# ---- one pass, through the package ------------------------------------------------

def _own_matvec(c, s):
    z = _package()
    type = BLOCKS[c["type"]][0]
    if c["glu"]:
        return [z.matvec_glu(z.GLU_SWIGLU, type, s["x"], s["w"][0], s["w"][1], c["n0"])]
    return z.matvec(type, s["x"], s["w"], _ns(c), residuals=s.get("res"))


def _own_shared(c, s):
    kv = _package("kv")
    if "batch" not in s:  # what a program keeps beside its tensors, made once
        s["cache"] = kv.Cache(s["pool"], s["tables"], s["lens"], s["refs"], c["page"], c["head"])
        s["batch"] = kv.Batch(s["starts"], s["rows"], s["max_new"], s["max_len"])
        s["kv_groups"] = kv.Groups(s["groups"], s["max_shared"])
    return kv.attention(s["cache"], 0, s["batch"], s["q"], 1.0 / math.sqrt(c["head"]), window=c["window"], softcap=c["softcap"],
                        groups=s["kv_groups"])


def _own_sample(c, s):
    return _package("sampling").sample(s["logits"], s["u"], s["temperature"], s.get("top_k"), s.get("top_p"), s.get("min_p"),
                                       probs=True)


def run(state):
    c = state["case"]
    if own:
        return {"matvec": _own_matvec, "shared": _own_shared, "sample": _own_sample}[c["kind"]](c, state)
    return {"matvec": _plain_matvec, "shared": _plain_shared, "sample": _plain_sample}[c["kind"]](c, state)


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    c = case
    if c["kind"] == "matvec":
        n, (_, values, size) = sum(_ns(c)), BLOCKS[c["type"]]
        y = c["n0"] if c["glu"] else 2 * n if c["residual"] else n
        return {"bytes": n * (c["k"] // values) * size + 4.0 * c["rows"] * (c["k"] + y), "flops": 2.0 * c["rows"] * n * c["k"]}
    if c["kind"] == "sample":
        return {"bytes": c["rows"] * (c["vocab"] * DTYPES[c["type"]].itemsize + 28.0), "flops": 0.0}
    shared, length, new = _lengths(c)
    pairs = tokens = 0
    for b, (s, m, n) in enumerate(zip(shared, length, new)):
        first = m
        for at in range(m - n, m):
            lo = max(0, at - c["window"] + 1) if c["window"] else 0
            pairs, first = pairs + at + 1 - lo, min(first, lo)
        one = b < c["groups"] * c["members"] and b % c["members"] > 0  # its shared tokens are read with the first member's
        tokens += m - max(first, s * c["page"] if one else 0)
    return {"bytes": 4.0 * sum(new) * c["q_heads"] * c["head"] + 4.0 * c["kv_heads"] * c["head"] * tokens,
            "flops": 4.0 * c["head"] * c["q_heads"] * pairs}


# ---- the same in 64 bits, from the definitions --------------------------------------

def _exact_weight(type, raw, k):
    """Every value's own byte, shift and scale, by its index in the row."""
    _, values, size = BLOCKS[type]
    i = torch.arange(k, device=raw.device)
    block, e = i // values * size, i % values
    at = lambda o: raw[:, o].long()  # noqa: E731
    scale = lambda o: torch.stack([raw[:, o], raw[:, o + 1]], dim=2).view(torch.float16)[:, :, 0].double()  # noqa: E731
    level = torch.tensor(LEVELS, dtype=torch.float64, device=raw.device)
    if type == "q8_0":
        q = at(block + 2 + e)
        return scale(block) * (q - 256 * (q > 127)).double()
    if type in ("q4_0", "q4_1", "iq4_nl"):
        q = at(block + size - 16 + e % 16) >> 4 * (e // 16) & 15
        if type == "q4_1":
            return scale(block) * q.double() + scale(block + 2)
        return scale(block) * (level[q] if type == "iq4_nl" else (q - 8).double())
    j, r = e // 32, e % 32  # the sub-block of 32, and the place in it
    if type == "iq4_xs":
        low, high = at(block + 4 + j // 2) >> 4 * (j % 2) & 15, at(block + 2 + j // 4) >> 2 * (j % 4) & 3
        return scale(block) * (16 * high + low - 32).double() * level[at(block + 8 + 16 * j + r % 16) >> 4 * (r // 16) & 15]
    q = at(block + 16 + 32 * (j // 2) + r) >> 4 * (j % 2) & 15
    a, b, both = at(block + 4 + j % 4), at(block + 8 + j % 4), at(block + 12 + j % 4)
    near = (j < 4)[None, :]
    sc = torch.where(near, a % 64, both % 16 + a // 64 * 16)
    m = torch.where(near, b % 64, both // 16 + b // 64 * 16)
    return scale(block) * sc.double() * q.double() - scale(block + 2) * m.double()


def _exact_matvec(c, s):
    y = []
    for w in s["w"]:
        step = max(1, int(2e7 / c["k"]))
        y.append(torch.cat([s["x"].double() @ _exact_weight(c["type"], w[r:r + step], c["k"]).T.contiguous()
                            for r in range(0, w.shape[0], step)], dim=1))
    if c["glu"]:
        return [y[0] / (1.0 + torch.exp(-y[0])) * y[1]]
    return [a + r.double() for a, r in zip(y, s["res"])] if c["residual"] else y


def _exact_shared(c, s):
    """One sequence and one k/v head at a time; each token's keys and values picked out by their offsets."""
    d, page, group = c["head"], c["page"], c["q_heads"] // c["kv_heads"]
    _, length, new = _lengths(c)
    out = torch.zeros((s["rows"], c["q_heads"], d), dtype=torch.float64, device="cuda")
    e, row = torch.arange(d, device="cuda"), 0
    for b, (n, m) in enumerate(zip(new, length)):
        t, i = torch.arange(m, device="cuda"), torch.arange(n, device="cuda")
        held, u = s["tables"][b].long()[t // page], t % page
        k_at = (e // 8 * page)[None, :] * 8 + u[:, None] * 8 + (e % 8)[None, :]
        half, inner = u // 4 % 2, u % 4 + u // 8 % 2 * 4
        v_at = page * d + ((u // 16 * 2 + half)[:, None] * d + e[None, :]) * 8 + inner[:, None]
        hidden = t[None, :] > m - n + i[:, None]
        if c["window"]:
            hidden |= t[None, :] <= m - n + i[:, None] - c["window"]
        for h in range(c["kv_heads"]):
            flat = s["pool"][0, :, h]
            k, v = flat[held[:, None], k_at].double(), flat[held[:, None], v_at].double()
            q = s["q"][row:row + n, h * group:(h + 1) * group].double()
            x = (q.reshape(-1, d) @ k.T).reshape(n, group, m) / math.sqrt(d)
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            x[hidden[:, None, :].expand_as(x)] = -math.inf
            p = torch.nan_to_num(torch.softmax(x, dim=2))
            out[row:row + n, h * group:(h + 1) * group] = (p.reshape(-1, m) @ v).reshape(n, group, d)
        row += n
    return out


def _exact_sample(c, s):
    """A row at a time on the host; the chosen token's probability."""
    get = lambda name, off: s[name].cpu().numpy() if name in s else np.full(c["rows"], off)  # noqa: E731
    t, k, p, m = get("temperature", 1.0), get("top_k", c["vocab"]), get("top_p", 1.0), get("min_p", 0.0)
    logits, u, probs = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy(), []
    for r in range(c["rows"]):
        if t[r] <= 0:
            probs.append(1.0)
            continue
        best = np.argsort(-logits[r], kind="stable")[:max(1, int(k[r]))]
        w = np.exp((logits[r][best] - logits[r][best[0]]) / np.float64(t[r]))
        if p[r] < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            best, w = best[before < np.float64(p[r]) * w.sum()], w[before < np.float64(p[r]) * w.sum()]
        best, w = best[w >= np.float64(m[r])], w[w >= np.float64(m[r])]
        w = w[np.argsort(best)]
        at = min(len(w) - 1, int(np.searchsorted(np.cumsum(w), u[r] * w.sum(), side="right")))
        probs.append(w[at] / w.sum())
    return None, np.array(probs)


def exact(case, seed):
    s = prepare(case, seed)
    return {"matvec": _exact_matvec, "shared": _exact_shared, "sample": _exact_sample}[case["kind"]](case, s)
