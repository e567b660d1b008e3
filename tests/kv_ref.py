"""Plain 64-bit forms of the paged KV cache's operators, on the CPU, and the
cache's layout one value at a time."""
from __future__ import annotations

import math

import numpy as np
import torch


def k_offset(t: int, e: int, page: int, d: int) -> int:
    """Where value e of token t (of a page) lies in a head's part of the page."""
    return (e // 8) * page * 8 + t * 8 + e % 8


def v_offset(t: int, e: int, page: int, d: int) -> int:
    g, u = divmod(t, 16)
    half, inner = (u // 4) % 2, u % 4 + 4 * (u // 8)
    return page * d + ((g * 2 + half) * d + e) * 8 + inner


def page_index(page: int, d: int) -> tuple[torch.Tensor, torch.Tensor]:
    """[page][d] offsets of K and of V."""
    k = [[k_offset(t, e, page, d) for e in range(d)] for t in range(page)]
    v = [[v_offset(t, e, page, d) for e in range(d)] for t in range(page)]
    return torch.tensor(k), torch.tensor(v)


class Book:
    """Sequences' keys and values as plain arrays, and the pool that holds them. Every place that holds no token is
    NaN, in pages that are used too."""

    def __init__(self, lens, page, kv_heads, d, dtype, seed=0, spare=3, cols=None):
        g = torch.Generator().manual_seed(seed)
        self.page, self.kv_heads, self.d, self.dtype, self.lens = page, kv_heads, d, dtype, list(lens)
        self.k = [torch.randn((n, kv_heads, d), generator=g).to(dtype) for n in lens]
        self.v = [torch.randn((n, kv_heads, d), generator=g).to(dtype) for n in lens]
        count = [-(-n // page) for n in lens]
        self.pages = sum(count) + spare
        ids = torch.randperm(self.pages, generator=g).tolist()
        cols = cols or max(count + [1])
        self.table = torch.full((len(lens), cols), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(count):
            self.table[b, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
            at += n
        self.refs = torch.zeros(self.pages, dtype=torch.int32)
        for i in ids[:at]:
            self.refs[i] = 1
        self.pool = torch.full((1, self.pages, kv_heads, 2 * page * d), math.nan, dtype=dtype)
        self.fill()

    def fill(self):
        ki, vi = page_index(self.page, self.d)
        for b, n in enumerate(self.lens):
            for j in range(-(-n // self.page)):
                m = min(self.page, n - j * self.page)
                held = self.pool[0, int(self.table[b, j])]
                for h in range(self.kv_heads):
                    held[h][ki[:m].reshape(-1)] = self.k[b][j * self.page:j * self.page + m, h].reshape(-1)
                    held[h][vi[:m].reshape(-1)] = self.v[b][j * self.page:j * self.page + m, h].reshape(-1)

    def cache(self, kv):
        return kv.Cache(self.pool.cuda(), self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32, device="cuda"),
                        self.refs.cuda(), self.page, self.d)


def read_cache(pool, table_row, n, page, d, layer=0):
    """The n tokens of a sequence, [n][kv_heads][d] each of K and V, read from a pool on the CPU."""
    ki, vi = page_index(page, d)
    k, v = [], []
    for j in range(-(-n // page)):
        held = pool[layer, int(table_row[j])]
        k.append(held[:, ki].permute(1, 0, 2))
        v.append(held[:, vi].permute(1, 0, 2))
    return torch.cat(k)[:n], torch.cat(v)[:n]


def attention(q, k, v, scale, causal=True, window=0, softcap=0.0, place0=None, unseen=None):
    """q [n][q_heads][d], k and v [len][kv_heads][d] -> (out, a): the output in 64 bits and, for the error bound, the
    weighted mean of |v|; the largest |score| sum for it is `reach`. unseen: tokens that no row sees."""
    n, heads, d = q.shape
    m, kvh = k.shape[0], k.shape[1]
    place0 = m - n if place0 is None else place0
    qd, kd, vd = q.double(), k.double(), v.double()
    out, spread = torch.zeros((n, heads, d), dtype=torch.float64), torch.zeros((n, heads, d), dtype=torch.float64)
    reach = 0.0
    t, pos = torch.arange(m), place0 + torch.arange(n)
    seen = torch.ones((n, m), dtype=torch.bool)
    if causal:
        seen &= t[None] <= pos[:, None]
    if window:
        seen &= t[None] > pos[:, None] - window
    if unseen is not None:
        seen &= ~unseen[None]
    for j in range(heads):
        h = j // (heads // kvh)
        for i in range(n):
            at = seen[i]
            if not at.any():
                continue
            ks, vs = kd[at, h], vd[at, h]
            x = (ks @ qd[i, j]) * scale
            reach = max(reach, float((ks.abs() @ qd[i, j].abs()).max()) * abs(scale))
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            p = torch.softmax(x, dim=0)
            out[i, j], spread[i, j] = p @ vs, p @ vs.abs()
    return out, spread, reach


def attention_bound(out, spread, reach, d, cache_dtype, out_dtype):
    """How far a kernel may be off, value by value: each weight rounded once to the cache's type (half a step), a
    score's sum of d products in fp32 (d + 4 roundings of at most `reach`, which move a weight by that much, above and
    below the line), the exponential and its argument (2^-20), the output rounded once."""
    u = torch.finfo(cache_dtype).eps / 2
    s = (d + 4) * 2.0 ** -24 * reach
    return (u + 2 * s + 2.0 ** -19) * spread + torch.finfo(out_dtype).eps / 2 * out.abs() + 1e-30


def rope(x, pos, freqs, mode, magnitude):
    """x [rows][heads][d], the first 2 len(freqs) dims turned by pos * freqs, in 64 bits."""
    n = 2 * len(freqs)
    a = torch.as_tensor(pos, dtype=torch.float64)[:, None] * torch.tensor(freqs, dtype=torch.float64)
    cos, sin = (torch.cos(a) * magnitude)[:, None], (torch.sin(a) * magnitude)[:, None]
    y = x.double().clone()
    i0 = torch.arange(n // 2) if mode == 2 else torch.arange(0, n, 2)
    i1 = i0 + (n // 2 if mode == 2 else 1)
    x0, x1 = y[..., i0].clone(), y[..., i1].clone()
    y[..., i0], y[..., i1] = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    return y


def assign(tables, lens, refs, page, dst, src, grow):
    """A scheduling step, one entry after the other: (copies [(from, to)], whether an entry was left undone or a count
    was wrong). Changes the numpy arrays it is given."""
    slots, cols = tables.shape
    pages = len(refs)
    old_tables, old_lens = tables.copy(), lens.copy()
    replaced = {d for d, s in zip(dst, src) if 0 <= d < slots and s != d}
    bad, fine, copies = False, [], []
    for i, (d, s, g) in enumerate(zip(dst, src, grow)):
        ok = 0 <= d < slots and -1 <= s < slots and g >= 0 and list(dst).count(d) == 1
        ok = ok and (s < 0 or s == d or s not in replaced)
        ok = ok and (int(old_lens[s]) if s >= 0 else 0) + int(g) <= cols * page
        bad |= not ok
        if ok:
            fine.append(i)
    for i in fine:
        if src[i] != dst[i]:
            for j in range(-(-int(old_lens[dst[i]]) // page)):
                refs[old_tables[dst[i], j]] -= 1
    free = [p for p in range(pages) if refs[p] <= 0]
    taken = 0
    for i in fine:
        d, s, g = dst[i], src[i], int(grow[i])
        base = int(old_lens[s]) if s >= 0 else 0
        held = -(-base // page) if s == d else base // page
        total = -(-(base + g) // page)
        need = total - held
        mine = free[taken:taken + need]
        taken += need
        if len(mine) < need:
            bad = True
            if s != d:
                tables[d], lens[d] = -1, 0
            continue
        row = [int(p) for p in (old_tables[s, :held] if s >= 0 else [])] + mine
        if s != d:
            for p in row[:held]:
                refs[p] += 1
            if base % page:
                copies.append((int(old_tables[s, held]), mine[0]))
        for p in mine:
            refs[p] = 1
        tables[d, :] = -1
        tables[d, :len(row)] = row
        lens[d] = base + g
    return copies, bad


def compact(tables, refs):
    """(new tables, new refs, moves [(from, to)], live, whether an entry named nothing)."""
    live = int((refs > 0).sum())
    to = [p for p in range(live) if refs[p] <= 0]
    movers = [p for p in range(live, len(refs)) if refs[p] > 0]
    place = {p: p for p in range(live) if refs[p] > 0} | dict(zip(movers, to))
    new_refs = np.zeros_like(refs)
    for p, q in place.items():
        new_refs[q] = refs[p]
    new_tables = np.array([[place.get(int(p), -1) for p in row] for row in tables], dtype=np.int32)
    return new_tables, new_refs, list(zip(movers, to)), live, bool(((new_tables < 0) & (tables != -1)).any())
