"""The paged KV cache's kernels against their plain 64-bit forms (kv_ref), at the
sizes, masks and contents where they can go wrong. The pool's unused places,
behind a sequence's end included, hold NaN throughout."""
from __future__ import annotations

import ctypes
import math

import kv_ref
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def kv(zest_gpu):
    from ggml_xdna_amd import kv as m
    return m


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


def _flag():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


class Case:
    """A batch over a Book: q on the CPU, the cache and the batch on the GPU."""

    def __init__(self, kv, seqs, page=16, kv_heads=2, group=2, d=64, dtype=BF16, q_dtype=None, seed=0, q_scale=2.0, **more):
        self.new, lens = [n for n, _ in seqs], [m for _, m in seqs]
        self.book = kv_ref.Book(lens, page, kv_heads, d, dtype, seed, **more)
        self.starts, self.rows, self.heads = _starts(self.new), sum(self.new), kv_heads * group
        g = torch.Generator().manual_seed(seed + 1)
        self.q = (q_scale * torch.randn((self.rows, self.heads, d), generator=g)).to(q_dtype or dtype)
        self.cache = self.book.cache(kv)
        self.batch = kv.Batch(_i32(self.starts), self.rows, max(self.new + [1]), max(lens + [1]))

    def check(self, got, causal=True, window=0, softcap=0.0, scale=None, unseen=None):
        b = self.book
        scale = 1.0 / math.sqrt(b.d) if scale is None else scale
        got = got.cpu().reshape(self.rows, self.heads, b.d)
        for i, n in enumerate(self.new):
            r = slice(self.starts[i], self.starts[i] + n)
            q = self.q[r].to(b.dtype)
            out, spread, reach = kv_ref.attention(q, b.k[i], b.v[i], scale, causal, window, softcap,
                                                  unseen=None if unseen is None else unseen[i])
            bound = kv_ref.attention_bound(out, spread, reach, b.d, b.dtype, got.dtype)
            off = (got[r].double() - out).abs()
            assert bool((off <= bound).all()), (i, n, b.lens[i], float((off / bound).max()))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,group,page", [(64, 1, 16), (64, 2, 32), (96, 3, 64), (128, 4, 64), (128, 6, 128), (192, 5, 16),
                                          (256, 8, 32), (128, 32, 256), (64, 33, 16)])
def test_attention(kv, dtype, d, group, page):
    """Every head width, page size and group shape (more columns than a tile among them) over one token to a few
    hundred: lengths around the pages, the 16-, 32- and 128-token units and a tile's columns."""
    seqs = [(1, 1), (1, 15), (1, 16), (1, 17), (2, 31), (1, 32), (3, 33), (1, 127), (5, 129), (1, 300), (40, 40), (33, 161)]
    c = Case(kv, seqs, page, 2 if group < 8 else 1, group, d, dtype, seed=d + group)
    bad = _flag()
    got = kv.attention(c.cache, 0, c.batch, c.q.cuda(), bad=bad)
    assert got.dtype == dtype and got.shape == c.q.shape
    c.check(got)
    assert int(bad) == 0


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window,softcap,scale", [(0, 0.0, 0.3), (1, 0.0, None), (7, 0.0, None), (40, 5.0, None), (500, 0.0, None),
                                                 (0, 2.0, None), (0, 0.0, 0.0), (0, 0.0, -0.2)])
def test_attention_masks(kv, causal, window, softcap, scale):
    c = Case(kv, [(1, 50), (20, 20), (9, 200), (70, 130), (1, 1)], 32, 2, 3, 64, BF16, seed=window)
    c.check(kv.attention(c.cache, 0, c.batch, c.q.cuda(), scale, causal, window, softcap), causal, window, softcap, scale)


@pytest.mark.parametrize("softcap", [1e-30, 0.05, 3.0, 64.0, 65.0, 1e3, 1e4, 1e6, 1e9, 3e38])
@pytest.mark.parametrize("d,new", [(64, 1), (64, 70), (128, 3), (128, 90)])
def test_softcap_of_any_size(kv, d, new, softcap):
    """Caps that flatten every score to those that change none. Up to 64 a capped score is off by 2^-22 of the cap,
    beyond by 2^-20 of the score (at most `reach`): twice that of a weight, above and below the line."""
    c = Case(kv, [(new, 150), (1, 40), (new, 700)], 32, 2, 4, d, F16, seed=int(d + new))
    scale = 1.0 / math.sqrt(d)
    got = kv.attention(c.cache, 0, c.batch, c.q.cuda(), softcap=softcap, out_dtype=F32).cpu()
    for i, n in enumerate(c.new):
        r = slice(c.starts[i], c.starts[i] + n)
        out, spread, reach = kv_ref.attention(c.q[r], c.book.k[i], c.book.v[i], scale, softcap=softcap)
        bound = kv_ref.attention_bound(out, spread, reach, d, F16, F32)
        bound += 2 * (2.0 ** -22 * softcap if softcap <= 64 else 2.0 ** -20 * reach) * spread
        off = (got[r].double() - out).abs()
        assert bool((off <= bound).all()), (i, float((off / bound).max()))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("q_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("out_dtype", [F32, F16, BF16])
def test_attention_types_and_strides(kv, dtype, q_dtype, out_dtype):
    """q and the output of any type, as column slices of wider buffers; the rest of the output's buffer stays as it was."""
    c = Case(kv, [(3, 20), (1, 64), (17, 100)], 16, 2, 2, 64, dtype, q_dtype, seed=3)
    wide = torch.full((c.rows, 3 * 256), math.nan, dtype=q_dtype, device="cuda")
    wide[:, 256:512] = c.q.reshape(c.rows, 256)
    out = torch.full((c.rows, 2 * 256 + 16), 7.0, dtype=out_dtype, device="cuda")
    got = kv.attention(c.cache, 0, c.batch, wide[:, 256:512], out=out[:, 16:272])
    c.check(got)
    assert bool((out[:, :16] == 7).all()) and bool((out[:, 272:] == 7).all())


def test_attention_split_over_workgroups(kv):
    """Contexts long enough that a column tile's keys are split among workgroups and joined, beside short ones; the
    same bits from run to run."""
    c = Case(kv, [(1, 5000), (2, 700), (1, 1), (3, 9001)], 64, 2, 4, 128, BF16, seed=9)
    q = c.q.cuda()
    got = kv.attention(c.cache, 0, c.batch, q, out_dtype=F32)
    c.check(got)
    for _ in range(3):
        assert torch.equal(kv.attention(c.cache, 0, c.batch, q, out_dtype=F32), got)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("new,group", [(1, 1), (2, 5), (1, 11), (3, 5), (4, 4), (1, 17), (8, 4)])
def test_decoding_of_every_width(kv, dtype, d, new, group):
    """Batches without a chunk, of one column a k/v head to two whole tiles (1, 10, 11, 15, 16, 17, 32), over contexts
    that end inside a workgroup's share and that many workgroups share: every value of the output is written, and no
    row behind the last sequence."""
    seqs = [(new, 90), (new, 130), (1, 700), (new, 5000)]
    c = Case(kv, seqs, 64, 2, group, d, dtype, seed=d + 10 * new + group)
    bad = _flag()
    out = torch.full((c.rows, c.heads, d), math.nan, dtype=dtype, device="cuda")
    c.check(kv.attention(c.cache, 0, c.batch, c.q.cuda(), out=out, bad=bad))
    more = torch.full((c.rows + 2, c.heads, d), math.nan, dtype=dtype, device="cuda")
    batch = kv.Batch(c.batch.starts, c.rows + 2, new, 5000)
    kv.attention(c.cache, 0, batch, torch.cat([c.q, c.q[:2]]).cuda(), out=more, bad=bad)
    assert int(bad) == 0 and bool(more[c.rows:].isnan().all())
    c.check(more[:c.rows])


def test_attention_long_chunk(kv):
    """A chunk of many column tiles, on top of what its sequence holds."""
    c = Case(kv, [(150, 400), (1, 70), (260, 260)], 32, 1, 2, 128, BF16, seed=11)
    c.check(kv.attention(c.cache, 0, c.batch, c.q.cuda()))


@pytest.mark.parametrize("d,page,dtype", [(64, 16, F16), (96, 32, BF16), (128, 16, BF16), (128, 64, F16), (192, 16, F16),
                                          (256, 64, BF16)])
@pytest.mark.parametrize("seqs", [[(40, 3000)], [(33, 2100), (1, 2500), (50, 1300)]])
def test_chunks_split_over_their_keys(kv, d, page, dtype, seqs):
    """Few tiles over long contexts, whose keys are split and joined: tables of more than 64 columns, a page that is not
    there, NaN and infinities that only some rows see."""
    c = Case(kv, seqs, page, 2, 4, d, dtype, seed=d)
    q = c.q.cuda()
    got = kv.attention(c.cache, 0, c.batch, q)
    c.check(got)
    c.check(kv.attention(c.cache, 0, c.batch, q, causal=False), causal=False)
    c.check(kv.attention(c.cache, 0, c.batch, q, window=700, softcap=20.0), window=700, softcap=20.0)
    bad = _flag()
    c.cache.tables[0, 1100 // page] = -1
    unseen = torch.zeros(seqs[0][1], dtype=torch.bool)
    unseen[1100 // page * page:1100 // page * page + page] = True
    c.check(kv.attention(c.cache, 0, c.batch, q, bad=bad), unseen=[unseen] + [None] * (len(seqs) - 1))
    assert int(bad) == 1
    # the last tokens of sequence 0 are NaN and infinite: row i sees those up to its own
    n, m = seqs[0]
    for t, v in ((m - 5, math.nan), (m - 3, math.inf), (m - 1, -math.inf)):
        c.book.v[0][t, :, 7] = v
    c.book.fill()
    c.cache = c.book.cache(kv)
    odd = kv.attention(c.cache, 0, c.batch, q).float().cpu()
    assert torch.equal(odd[:n - 5], got[:n - 5].float().cpu()) and bool(odd[n - 5:n, :, 7].isnan().all())
    rest = [e for e in range(d) if e != 7]
    assert torch.equal(odd[..., rest], got.float().cpu()[..., rest])


@pytest.mark.parametrize("count", [64, 65, 300, 1100])
def test_many_sequences(kv, count):
    """More sequences than a wave's lanes, than a workgroup's threads, than that many each: append and attention of one
    or a few tokens each (and of a chunk among them), none of a sequence here and there."""
    rng = np.random.default_rng(count)
    new = [int(n) for n in rng.choice([0, 1, 1, 1, 2, 3], count)]
    new[count // 2] = 70
    lens = [n + int(rng.integers(0, 60)) for n in new]
    c = Case(kv, list(zip(new, lens)), 16, 1, 2, 64, BF16, seed=count)
    bad = _flag()
    c.check(kv.attention(c.cache, 0, c.batch, c.q.cuda(), bad=bad))
    k, v = (torch.randn((c.rows, 1, 64), generator=torch.Generator().manual_seed(i)) for i in (1, 2))
    kv.append(c.cache, 0, c.batch, k.cuda(), v.cuda(), bad=bad)
    assert int(bad) == 0
    pool, want = c.cache.pool.cpu(), c.book.pool.clone()
    ki, vi = kv_ref.page_index(16, 64)
    for b, (n, m, r) in enumerate(zip(new, lens, c.starts)):
        for i in range(n):
            held, t = want[0, int(c.book.table[b, (m - n + i) // 16]), 0], (m - n + i) % 16
            held[ki[t]], held[vi[t]] = k[r + i, 0].to(BF16), v[r + i, 0].to(BF16)
    assert torch.equal(pool.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("d,count,new", [(192, 100, 70), (256, 70, 40), (96, 4096, 1), (256, 4096, 1)])
def test_many_sequences_of_wide_heads(kv, d, count, new):
    """Prefix sums in shared memory beside the widest rings, with and without a chunk in the batch."""
    rng = np.random.default_rng(d + count)
    news = [int(n) for n in rng.choice([0, 1, 1], count)]
    news[count // 3] = new
    c = Case(kv, [(n, n + int(rng.integers(0, 40))) for n in news], 16, 1, 1 if count > 1000 else 2, d, F16, seed=d)
    bad = _flag()
    c.check(kv.attention(c.cache, 0, c.batch, c.q.cuda(), bad=bad))
    assert int(bad) == 0


@pytest.mark.parametrize("new", [1, 5, 90])
def test_a_place_near_the_largest(kv, new):
    """A window over the end of a sequence of 2^30 tokens, whose other pages are gone, and the append of its last ones."""
    d, page, length, window = 64, 256, 1 << 30, 150
    book = kv_ref.Book([512], page, 1, d, BF16, seed=new)  # the last two pages' tokens
    table = torch.full((1, length // page), -1, dtype=torch.int32)
    table[0, -2:] = book.table[0, :2]
    cache = kv.Cache(book.pool.cuda(), table.cuda(), _i32([length]), book.refs.cuda(), page, d)
    batch, bad = kv.Batch(_i32([0, new]), new, new, length), _flag()
    q = torch.randn((new, 4, d), generator=torch.Generator().manual_seed(new)).to(BF16)
    got = kv.attention(cache, 0, batch, q.cuda(), window=window, bad=bad).cpu()
    want, spread, reach = kv_ref.attention(q, book.k[0], book.v[0], 0.125, window=window)
    assert bool(((got.double() - want).abs() <= kv_ref.attention_bound(want, spread, reach, d, BF16, BF16)).all()) and int(bad) == 0
    k, v = (torch.randn((new, 1, d), generator=torch.Generator().manual_seed(i)) for i in (1, 2))
    freqs = [1e4 ** (-2 * p / d) for p in range(d // 2)]
    kv.append(cache, 0, batch, k.cuda(), v.cuda(), rope=kv.Rope(torch.tensor(freqs, dtype=torch.float64, device="cuda")), bad=bad)
    k1, v1 = kv_ref.read_cache(cache.pool.cpu(), book.table[0], 512, page, d)
    turned = kv_ref.rope(k, np.arange(length - new, length), freqs, 2, 1.0)
    # the angle's own error: 2^28 turns in 64 bits, a product's and a constant's rounding of 2^-25 of a turn each
    assert bool(((k1[-new:].double() - turned).abs() <= 2.0 ** -8 * turned.abs() + 8 * (2.0 ** -22 + 2 * math.pi * 2.0 ** -23)).all())
    assert torch.equal(v1[-new:], v.to(BF16)) and torch.equal(k1[:-new], book.k[0][:-new]) and int(bad) == 0


def test_offsets_past_32_bits(kv):
    """The same calls over pages at the front of a pool of 10 GB, and at its end; rows 2^27 values apart."""
    d, page, kvh, group = 128, 64, 8, 2
    bytes_each = 4 * page * d * kvh
    pages = 5 * (1 << 30) // bytes_each
    seqs = [(70, 700), (1, 900), (3, 64)]
    need = [-(-m // page) for _, m in seqs]
    cache = kv.empty_cache(2, pages, kvh, d, page, slots=5, columns=max(need) + 1)
    starts = _starts([n for n, _ in seqs])
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((sum(m for _, m in seqs), kvh, d), generator=g, device="cuda") for _ in range(2))
    q = torch.randn((starts[-1], kvh * group, d), generator=g, device="cuda")
    wide = torch.empty((starts[-1], 1 << 27), dtype=BF16, device="cuda")  # 74 rows of 256 MB: 20 GB
    fill = kv.Batch(_i32(_starts([m for _, m in seqs])), k.shape[0], 700 + 200, 1000)
    batch = kv.Batch(_i32(starts), starts[-1], 70, 1000)
    results = []
    for first in (0, pages - sum(need)):
        cache.tables.fill_(-1)
        cache.refs.zero_()
        at = first
        for b, n in enumerate(need):
            cache.tables[b, :n] = torch.arange(at, at + n, dtype=torch.int32, device="cuda")
            at += n
        cache.refs[first:at] = 1
        cache.lens.copy_(_i32([m for _, m in seqs] + [0, 0]))
        kv.append(cache, 1, fill, k, v)
        out = wide[:, 4096:4096 + kvh * group * d]
        wide[:, :kvh * group * d] = q.reshape(starts[-1], -1)
        kv.attention(cache, 1, batch, wide[:, :kvh * group * d], out=out)
        again = kv.append(cache, 1, batch, k[:starts[-1]], v[:starts[-1]], q)
        results.append((out.clone(), again))
    assert bool(results[0][0].isfinite().all()) and bool(results[0][0].any())
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    held = cache.pool[1, first:].clone()
    kv.assign(cache, _i32([3]), _i32([0]), _i32([0]))  # the open page, to the front of both layers
    assert cache.tables[3, need[0] - 1] == 0 and torch.equal(cache.pool[1, 0], held[need[0] - 1])
    kv.assign(cache, _i32([3]), _i32([-1]), _i32([0]))
    live = int(kv.compact(cache))
    cache.check()
    assert live == sum(need) and torch.equal(cache.pool[1, :live], held)
    assert cache.tables[:3].max() == live - 1


def test_batches_of_nothing(kv):
    """No sequence has new tokens; every length is 0; two sequences name the same slot."""
    c = Case(kv, [(2, 20), (40, 90)], 16, 1, 2, 64, BF16, seed=4)
    q, x, bad = c.q.cuda(), torch.zeros((42, 1, 64), device="cuda"), _flag()
    pool = c.cache.pool.clone()
    for max_new in (1, 42):
        batch = kv.Batch(_i32([0, 0, 0]), 42, max_new, 90)
        out = torch.full_like(q, 3.0)
        kv.attention(c.cache, 0, batch, q, out=out, bad=bad)
        kv.append(c.cache, 0, batch, x, x, q=q.float(), q_out=(q_out := torch.full_like(q, 3.0)), bad=bad)
        assert bool((out == 3).all()) and bool((q_out == 3).all()) and int(bad) == 0
    assert torch.equal(c.cache.pool.view(torch.int16), pool.view(torch.int16))
    want = kv.attention(c.cache, 0, c.batch, q)
    twice = kv.attention(c.cache, 0, kv.Batch(_i32([0, 40, 80]), 80, 40, 90, _i32([1, 1])), q[2:].repeat(2, 1, 1), bad=bad)
    assert torch.equal(twice[:40], twice[40:]) and int(bad) == 0
    b = c.book
    ref, spread, reach = kv_ref.attention(c.q[2:], b.k[1], b.v[1], 0.125)
    assert bool(((twice[:40].cpu().double() - ref).abs() <= kv_ref.attention_bound(ref, spread, reach, 64, BF16, BF16)).all())
    c.cache.lens.zero_()
    for new in ([0, 2, 42], [0, 1, 2]):
        got = kv.attention(c.cache, 0, kv.Batch(_i32(new), 42, new[2] - new[1], 0), q, out=torch.full_like(q, 3.0), bad=bad)
        assert bool((got[:new[2]] == 0).all()) and bool((got[new[2]:] == 3).all()) and int(bad) == 0
    assert bool(want.isfinite().all())


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_values_a_row_does_not_see_do_not_reach_it(kv, value, dtype):
    """K or V of a token that holds NaN or an infinity: only the rows that see it change."""
    c = Case(kv, [(40, 90), (1, 33)], 16, 1, 2, 64, dtype, seed=5)
    clean = kv.attention(c.cache, 0, c.batch, c.q.cuda()).cpu()
    late = 70  # token 70 of 90 is seen by the new tokens from place 70 on: rows 20 to 39
    c.book.v[0][late, 0, 5] = value
    c.book.fill()
    c.cache = c.book.cache(kv)
    got = kv.attention(c.cache, 0, c.batch, c.q.cuda()).cpu()
    assert torch.equal(got[:20], clean[:20]) and torch.equal(got[40:], clean[40:])
    assert torch.equal(got[20:40, :, :5], clean[20:40, :, :5]) and torch.equal(got[20:40, :, 6:], clean[20:40, :, 6:])
    hit = got[20:40, :, 5].float()
    assert bool(hit.isnan().all()) if math.isnan(value) else bool((hit == value).all())
    # a window that leaves the token behind
    win = kv.attention(c.cache, 0, c.batch, c.q.cuda(), window=10).cpu()
    assert bool(win[30:40].isfinite().all()) and not bool(win[20:30, :, 5].isfinite().any())
    # and the same in K
    c.book.v[0][late, 0, 5] = 1.0
    c.book.k[0][late, 0, 5] = value
    c.book.fill()
    c.cache = c.book.cache(kv)
    got = kv.attention(c.cache, 0, c.batch, c.q.cuda()).cpu()
    assert torch.equal(got[:20], clean[:20])


def test_rows_that_see_nothing_are_zero(kv):
    """Rows before a sequence's start (lens below the new tokens), a sequence of length 0, scores of -infinity alone;
    rows behind the last sequence and of one without new tokens stay as they were."""
    c = Case(kv, [(6, 6), (2, 20), (3, 3)], 16, 1, 2, 64, BF16, seed=6)
    c.cache.lens.copy_(_i32([4, 20, 0]))
    out = torch.full((c.rows + 2, 2, 64), 9.0, dtype=BF16, device="cuda")
    q = torch.cat([c.q, torch.zeros(2, 2, 64, dtype=BF16)]).cuda()
    batch = kv.Batch(_i32(c.starts), c.rows + 2, 6, 20)
    bad = _flag()
    kv.attention(c.cache, 0, batch, q, out=out, bad=bad)
    assert bool((out[:2] == 0).all()) and bool((out[8:11] == 0).all()) and bool((out[11:] == 9).all())
    want, spread, reach = kv_ref.attention(c.q[2:6], c.book.k[0][:4], c.book.v[0][:4], 0.125)
    assert bool(((out[2:6].cpu().double() - want).abs() <= kv_ref.attention_bound(want, spread, reach, 64, BF16, BF16)).all())
    # without causal the rows before the start see the whole sequence
    kv.attention(c.cache, 0, batch, q, causal=False, out=out)
    want, spread, reach = kv_ref.attention(c.q[:6], c.book.k[0][:4], c.book.v[0][:4], 0.125, causal=False)
    assert bool(((out[:6].cpu().double() - want).abs() <= kv_ref.attention_bound(want, spread, reach, 64, BF16, BF16)).all())
    assert int(bad) == 0
    # scores of -infinity alone
    c.book.k[1][:] = -math.inf
    c.book.fill()
    c.cache = c.book.cache(kv)
    q[6:8] = 1.0
    kv.attention(c.cache, 0, batch, q, out=out)
    assert bool((out[6:8] == 0).all())


def test_large_scores(kv):
    """Scores in the thousands: the running maximum keeps the weights in range."""
    c = Case(kv, [(5, 300), (1, 40)], 32, 2, 2, 64, F16, seed=8, q_scale=300.0)
    c.check(kv.attention(c.cache, 0, c.batch, c.q.cuda(), 1.0), scale=1.0)


def test_bad_device_values_are_left_out_and_reported(kv):
    """Pages outside the pool, slots outside the tables, starts outside the rows, lengths past the bounds."""
    seqs = [(2, 60), (2, 60), (2, 60)]
    for page_id in (-1, -7, 1 << 30, None):
        c = Case(kv, seqs, 16, 1, 2, 64, BF16, seed=4)
        wrong = c.book.pages if page_id is None else page_id
        c.cache.tables[1, 2] = wrong
        bad = _flag()
        got = kv.attention(c.cache, 0, c.batch, c.q.cuda(), bad=bad)
        unseen = torch.zeros(60, dtype=torch.bool)
        unseen[32:48] = True
        c.check(got, unseen=[torch.zeros(60, dtype=torch.bool), unseen, torch.zeros(60, dtype=torch.bool)])
        assert int(bad) == 1
        # the entry behind the length is not looked at
        bad.zero_()
        c.cache.tables[1, 2] = c.book.table[1, 2].cuda()
        c.cache.lens[1] = 48
        c.cache.tables[1, 3] = wrong
        kv.attention(c.cache, 0, c.batch, c.q.cuda(), bad=bad)
        assert int(bad) == 0
    c = Case(kv, seqs, 16, 1, 2, 64, BF16, seed=4)
    good = kv.attention(c.cache, 0, c.batch, c.q.cuda())
    for starts, slots, lens in [([0, 2, 7, 6], None, None), ([0, 2, -3, 6], None, None), ([0, 2, 1, 6], None, None),
                                ([0, 2, 4, 6], [0, 3, 2], None), ([0, 2, 4, 6], [0, -1, 2], None),
                                ([0, 2, 4, 6], None, [60, 61, 60]), ([0, 2, 4, 6], None, [60, -1, 60])]:
        cache = c.book.cache(kv)
        if lens:
            cache.lens.copy_(_i32(lens))
        out, bad = torch.full_like(good, 3.0), _flag()
        batch = kv.Batch(_i32(starts), 6, 2, 60, None if slots is None else _i32(slots))
        kv.attention(cache, 0, batch, c.q.cuda(), out=out, bad=bad)
        assert int(bad) == 1 and torch.equal(out[:2], good[:2]) and bool((out[2:4] == 3).all()), (starts, slots, lens)


def test_a_cache_tells_what_its_calls_left_out(kv):
    """Calls without a flag of their own report to the cache's, captured ones too; check raises once and clears it."""
    import ggml_xdna_amd as z
    c = Case(kv, [(2, 60), (2, 60)], 16, 1, 2, 64, BF16, seed=4)
    cache, q, x = c.cache, c.q.cuda(), torch.zeros((4, 1, 64), device="cuda")

    def left_out(call):
        call()
        with pytest.raises(z.ZestError, match="left out"):
            cache.check()
        cache.check()

    kv.attention(cache, 0, c.batch, q)
    kv.append(cache, 0, c.batch, x, x)
    kv.assign(cache, _i32([0]), _i32([0]), _i32([2]))
    cache.check()
    kv.assign(cache, _i32([0]), _i32([0]), _i32([-1]), bad=(own := _flag()))
    assert int(own) == 1
    cache.check()
    left_out(lambda: kv.attention(cache, 0, kv.Batch(c.batch.starts, 4, 2, 59), q))
    left_out(lambda: kv.append(cache, 0, kv.Batch(c.batch.starts, 4, 2, 62, _i32([0, 2])), x, x))
    left_out(lambda: kv.assign(cache, _i32([0]), _i32([0]), _i32([16 * 4 + 3])))
    cache.tables[1, 0] = cache.pages
    left_out(lambda: kv.compact(cache))
    cache.tables[0, 1] = cache.pages  # past this call's capture
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        kv.attention(cache, 0, kv.Batch(c.batch.starts, 4, 2, 64), q)
    torch.cuda.synchronize()
    cache.check()
    left_out(graph.replay)
    left_out(graph.replay)


def test_a_cache_dropped_while_another_stream_uses_it(kv):
    """The working memory and the flag of a cache that another stream's queued work uses go to no new tensor before that
    work is done."""
    cache = kv.empty_cache(1, 40000, 1, 64, 16, slots=4, columns=100)
    kept = cache.pool, cache.tables, cache.lens, cache.refs
    assert int(cache.refs.sum()) == 0
    used = [(t.data_ptr(), t.numel() * t.element_size()) for t in (cache._scratch, cache.bad)]
    entries = _i32([0]), _i32([-1]), _i32([1000])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        kv.assign(cache, *entries)
        done = torch.cuda.Event()
        done.record()
    del cache
    new = [torch.empty(n, dtype=torch.uint8, device="cuda") for _, n in used for _ in range(4)]
    assert not done.query()  # else this shows nothing
    for t in new:
        assert all(t.data_ptr() + t.numel() <= at or at + n <= t.data_ptr() for at, n in used)
    torch.cuda.synchronize()
    assert kept[2].tolist() == [1000, 0, 0, 0] and int(kept[3].sum()) == 63


def test_a_stack_that_outgrows_its_cache_is_told(kv):
    import ggml_xdna_amd as z
    from ggml_xdna_amd import stack
    s = stack.Stack(stack.StackConfig("tiny", 1, 256, 256, 128, 512, 8, 8, 8, 8, 100, 64, head_dim=64), seed=1, attention=True)
    s.run_prompt()
    s.run_prompt()
    s.cache.check()
    s.run_chunk(s.x[:64])
    with pytest.raises(z.ZestError, match="left out"):
        s.cache.check()


def test_outputs_that_contradict_the_call(kv):
    """An output for queries that are not given, or of another type than the one asked for, is refused before the launch."""
    import ggml_xdna_amd as z
    c = Case(kv, [(2, 20)], 16, 1, 2, 64, BF16, seed=4)
    q, x, out = c.q.cuda(), torch.zeros((2, 1, 64), dtype=BF16, device="cuda"), torch.empty((2, 2, 64), dtype=BF16, device="cuda")
    pool = c.cache.pool.clone()
    for call, said in [(lambda: kv.append(c.cache, 0, c.batch, x, x, q_out=out), "q_out"),
                       (lambda: kv.append(c.cache, 0, c.batch, x, x, q, q_out=out, q_dtype=F32), "q_dtype"),
                       (lambda: kv.attention(c.cache, 0, c.batch, q, out=out, out_dtype=F16), "out_dtype")]:
        with pytest.raises(z.ZestError, match=said):
            call()
    assert torch.equal(c.cache.pool.view(torch.int16), pool.view(torch.int16))
    assert kv.append(c.cache, 0, c.batch, x, x, q, q_out=out, q_dtype=BF16) is out
    assert kv.attention(c.cache, 0, c.batch, q, out=out, out_dtype=BF16) is out


def test_windows_that_32_bits_would_cut(kv):
    import ggml_xdna_amd as z
    c = Case(kv, [(2, 20)], 16, 1, 2, 64, BF16, seed=4)
    q = c.q.cuda()
    for window in ((1 << 32) + 5, 1 << 31, -1):
        with pytest.raises(z.ZestError, match="window"):
            kv.attention(c.cache, 0, c.batch, q, window=window)
    assert torch.equal(kv.attention(c.cache, 0, c.batch, q, window=(1 << 31) - 1), kv.attention(c.cache, 0, c.batch, q))


def _overlapping(kv, new, length, starts, group, page=16, d=64):
    """A batch of sequences of `new` rows each whose starts go back to the first row time and again."""
    c = Case(kv, [(new, length)] * (len(starts) // 2), page, 1, group, d, BF16, seed=len(starts))
    slots = _i32([i // 2 for i in range(len(starts) - 1)])
    return c, kv.Batch(_i32(starts), new, new, length, slots=slots)


@pytest.mark.parametrize("new,group,seqs", [(1, 4, 9), (600, 4, 9), (600, 2, 91), (200, 4, 1001)])
def test_starts_that_go_back(kv, new, group, seqs):
    """More rows among the sequences than the call has, as each begins at the first again: reported, and nothing is
    written beyond the output, the workspace's bytes and the new tokens' pages."""
    import ggml_xdna_amd as z
    starts = [0 if i % 2 == 0 else new for i in range(seqs + 1)]
    c, b = _overlapping(kv, new, max(new, 40) + 700 * (seqs < 100), starts, group)
    q, bad = c.q[:new].cuda(), _flag()
    need = kv.attention_workspace(c.cache, b, group)
    room = torch.full((need + (1 << 22),), 7, dtype=torch.uint8, device="cuda")
    out = torch.full((new + 64, group, 64), 7.0, dtype=BF16, device="cuda")
    ref = ctypes.byref
    z.check(z.lib().zest_kv_attn(ref(c.cache._layer[0]), ref(c.cache._batch(b)), q.data_ptr(), kv.TYPE_BF16, group * 64, group, 0.125, 1, 0,
                                 0.0, out.data_ptr(), kv.TYPE_BF16, group * 64, room.data_ptr(), need, bad.data_ptr(), z._stream()), "attn")
    assert int(bad) == 1 and bool((room[need:] == 7).all()) and bool((out[new:] == 7).all())
    bad.zero_()
    pool = c.cache.pool.clone()
    x = torch.zeros((new, 1, 64), dtype=BF16, device="cuda")
    kv.append(c.cache, 0, b, x, x, bad=bad)
    assert int(bad) == 1
    new_pages = torch.zeros(c.cache.pages, dtype=torch.bool)
    first = int(c.cache.lens[0]) - new
    for row in c.cache.tables.cpu().tolist():
        new_pages[[p for p in row[first // 16:] if p >= 0]] = True
    assert torch.equal(pool[:, ~new_pages].view(torch.int16), c.cache.pool[:, ~new_pages].view(torch.int16))


def test_two_calls_at_once(kv):
    """Attention of the same queries on two streams: each call has its workspace."""
    c = Case(kv, [(1, 3000), (40, 1500), (2, 64), (300, 300)], 64, 2, 4, 128, BF16, seed=4)
    q = c.q.cuda()
    want = kv.attention(c.cache, 0, c.batch, q)
    c.check(want)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kv.attention(c.cache, 0, c.batch, q))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for one in got for x in one)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new", [1, 5, 90])
def test_pages_that_a_window_has_left_may_be_gone(kv, page, new):
    """The table's entries of pages before every row's window are -1: nothing is reported, nothing changes."""
    c = Case(kv, [(new, 400), (1, 3)], page, 1, 2, 64, BF16, seed=new)
    want = kv.attention(c.cache, 0, c.batch, c.q.cuda(), window=50)
    first = 400 - new - 50 + 1  # the first token that the first row sees
    c.cache.tables[0, :first // page] = -1
    bad = _flag()
    got = kv.attention(c.cache, 0, c.batch, c.q.cuda(), window=50, bad=bad)
    assert int(bad) == 0 and torch.equal(got, want)
    c.check(got, window=50)
    c.cache.tables[0, first // page] = -1  # the one it does see
    kv.attention(c.cache, 0, c.batch, c.q.cuda(), window=50, bad=bad)
    assert int(bad) == 1


def test_slots_and_layers(kv):
    """Sequences in any slots of a cache, in a layer past the first."""
    c = Case(kv, [(2, 40), (1, 17), (3, 70)], 16, 2, 2, 64, BF16, seed=12)
    pool = torch.full((3, *c.book.pool.shape[1:]), math.nan, dtype=BF16)
    pool[2] = c.book.pool[0]
    order = [4, 0, 3]
    tables, lens = torch.full((6, c.book.table.shape[1]), -1, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    for b, s in enumerate(order):
        tables[s], lens[s] = c.book.table[b], c.book.lens[b]
    cache = kv.Cache(pool.cuda(), tables.cuda(), lens.cuda(), c.book.refs.cuda(), 16, 64)
    c.check(kv.attention(cache, 2, kv.Batch(_i32(c.starts), c.rows, 3, 70, _i32(order)), c.q.cuda()))


@pytest.mark.parametrize("dtype,in_dtype", [(BF16, F32), (F16, F32), (BF16, BF16), (F16, F16), (F16, BF16)])
@pytest.mark.parametrize("mode,rot", [(2, 64), (0, 64), (2, 32), (0, 32), (2, 24), (0, 10), (2, 6), (0, 64), (None, 0)])
def test_append(kv, dtype, in_dtype, mode, rot):
    """New tokens into whole and broken units of 16 places, rope in both layouts over the whole head and parts of it:
    each value rounded once (half a step of its type) from angles of positions far out."""
    d, page, kvh, heads = 64, 32, 2, 4
    new, lens = [1, 17, 40, 16, 3], [1, 200000, 45, 32, 90]
    rows, starts = sum(new), _starts(new)
    # a table wide enough for the long sequence, its page only where tokens are written
    g = torch.Generator().manual_seed(rot)
    cols = -(-200000 // page)
    table = torch.full((5, cols), -1, dtype=torch.int32)
    ids = iter(torch.randperm(40, generator=g).tolist())
    for b, (n, m) in enumerate(zip(new, lens)):
        for j in range((m - n) // page, -(-m // page)):
            table[b, j] = next(ids)
    before = torch.randn((1, 40, kvh, 2 * page * d), generator=g).to(dtype)
    cache = kv.Cache(before.cuda(), table.cuda(), _i32(lens), torch.ones(40, dtype=torch.int32, device="cuda"), page, d)
    batch = kv.Batch(_i32(starts), rows, 40, 200000)
    q, k, v = (torch.randn((rows, h, d), generator=g).to(in_dtype) for h in (heads, kvh, kvh))
    freqs = [1e4 ** (-2 * p / rot) for p in range(rot // 2)]
    r = kv.Rope(torch.tensor(freqs, dtype=torch.float64, device="cuda"), mode, 1.25) if mode is not None else None
    place = np.concatenate([np.arange(m - n, m) for n, m in zip(new, lens)])
    for pos in (None, place[::-1].copy()):
        bad = _flag()
        cache.pool.copy_(before)
        got = kv.append(cache, 0, batch, k.cuda(), v.cuda(), q.cuda(), r, None if pos is None else _i32(pos.tolist()), bad=bad)
        at = place if pos is None else pos
        wq, wk = (kv_ref.rope(x, at, freqs, mode, 1.25) if mode is not None else x.double() for x in (q, k))
        # the rounding, and sine and cosine in fp32 (2^-22 of the pair's length)
        tol = lambda w: torch.finfo(dtype).eps / 2 * w.abs() + 2.0 ** -22 * 1.25 * 8 + torch.finfo(dtype).smallest_normal  # noqa: E731
        assert bool(((got.cpu().double() - wq).abs() <= tol(wq)).all())
        pool, want = cache.pool.cpu(), before.clone()
        ki, vi = kv_ref.page_index(page, d)
        seq = np.concatenate([np.full(n, b) for b, n in enumerate(new)])
        for row in range(rows):
            held, t = int(table[seq[row], place[row] // page]), int(place[row] % page)
            for h in range(kvh):
                assert bool(((pool[0, held, h, ki[t]].double() - wk[row, h]).abs() <= tol(wk[row, h])).all())
                assert torch.equal(pool[0, held, h, vi[t]], v[row, h].to(dtype))
                want[0, held, h, ki[t]] = pool[0, held, h, ki[t]]
                want[0, held, h, vi[t]] = pool[0, held, h, vi[t]]
        assert torch.equal(pool, want) and int(bad) == 0  # nothing else was written


@pytest.mark.parametrize("mode,rot", [(2, 64), (0, 64), (2, 24), (2, 32)])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_append_in_place_and_strided(kv, mode, rot, dtype):
    """q turned in place; q, k and v as column slices of one wide buffer."""
    cache = kv.empty_cache(1, 4, 2, 64, 16, slots=2)
    cache.tables[:, 0], cache.tables[:, 1] = _i32([0, 2]), _i32([1, 3])
    cache.lens.copy_(_i32([9, 20]))
    batch = kv.Batch(_i32([0, 9, 14]), 14, 9, 20)
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((14, 4 * 64 + 2 * 128 + 16), generator=g).to(dtype).cuda()
    q, k, v = wide[:, :256], wide[:, 256:384], wide[:, 384:512]
    r = kv.Rope(torch.tensor([1e4 ** (-2 * p / rot) for p in range(rot // 2)], dtype=torch.float64, device="cuda"), mode)
    apart = kv.append(cache, 0, batch, k, v, q, r, q_dtype=dtype)
    pool = cache.pool.clone()
    rest = wide[:, 256:].clone()
    cache.pool.zero_()
    got = kv.append(cache, 0, batch, k, v, q, r, q_out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(q, apart) and torch.equal(cache.pool, pool) and torch.equal(wide[:, 256:], rest)
    # without q: the same pages
    cache.pool.zero_()
    assert kv.append(cache, 0, batch, k, v, rope=r) is None and torch.equal(cache.pool, pool)


@pytest.mark.parametrize("d,page,kvh,heads,mode,rot", [(64, 16, 16, 16, 2, 64), (96, 32, 5, 15, 2, 96), (96, 64, 3, 12, 0, 48), (128, 256, 8, 48, 2, 128),
                                                       (128, 64, 9, 27, 2, 40), (192, 128, 8, 24, 0, 192), (192, 16, 2, 30, 2, 64),
                                                       (256, 64, 7, 14, 2, 256), (256, 32, 11, 11, 0, 64)])
def test_append_of_every_width(kv, d, page, kvh, heads, mode, rot):
    """Several heads a workgroup, their last group ragged, for chunks that begin and end inside units of 16."""
    new, lens = [700, 1, 333, 16, 450], [1000, 33, 333, 48, 451]
    rows, starts = sum(new), _starts(new)
    g = torch.Generator().manual_seed(d + rot)
    count = [-(-m // page) for m in lens]
    ids = torch.randperm(sum(count) + 2, generator=g).int()
    table, at = torch.full((len(new), max(count)), -1, dtype=torch.int32), 0
    for b, n in enumerate(count):
        table[b, :n] = ids[at:at + n]
        at += n
    before = torch.randn((1, len(ids), kvh, 2 * page * d), generator=g).to(BF16)
    cache = kv.Cache(before.cuda(), table.cuda(), _i32(lens), torch.ones(len(ids), dtype=torch.int32, device="cuda"), page, d)
    q, k, v = (torch.randn((rows, h, d), generator=g) for h in (heads, kvh, kvh))
    freqs = [1e4 ** (-2 * p / rot) for p in range(rot // 2)]
    bad = _flag()
    got = kv.append(cache, 0, kv.Batch(_i32(starts), rows, max(new), max(lens)), k.cuda(), v.cuda(), q.cuda(),
                    kv.Rope(torch.tensor(freqs, dtype=torch.float64, device="cuda"), mode), bad=bad)
    place = np.concatenate([np.arange(m - n, m) for n, m in zip(new, lens)])
    seq = np.concatenate([np.full(n, b) for b, n in enumerate(new)])
    tol = lambda w: 2.0 ** -8 * w.abs() + 2.0 ** -22 * 8  # noqa: E731
    wq, wk = (kv_ref.rope(x, place, freqs, mode, 1.0) for x in (q, k))
    assert bool(((got.cpu().double() - wq).abs() <= tol(wq)).all()) and int(bad) == 0
    pool, want = cache.pool.cpu(), before.clone()
    ki, vi = kv_ref.page_index(page, d)
    held, t = table[torch.from_numpy(seq), torch.from_numpy(place // page)].long(), torch.from_numpy(place % page)
    at_k = held[:, None, None], torch.arange(kvh)[None, :, None], ki[t][:, None, :]
    assert bool(((pool[0][at_k].double() - wk).abs() <= tol(wk)).all())
    want[0][at_k] = pool[0][at_k]
    want[0][at_k[0], at_k[1], vi[t][:, None, :]] = v.to(BF16)
    assert torch.equal(pool, want)  # v's values, and nothing else


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_into_columns_of_the_same_buffer(kv, dtype):
    """q, k, v and the turned q side by side in one buffer's rows."""
    cache = kv.empty_cache(1, 4, 2, 64, 16, slots=2)
    cache.tables[:, 0], cache.tables[:, 1] = _i32([0, 2]), _i32([1, 3])
    cache.lens.copy_(_i32([9, 20]))
    batch = kv.Batch(_i32([0, 9, 14]), 14, 9, 20)
    wide = torch.randn((14, 256 + 2 * 128 + 256), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    q, k, v, out = wide[:, :256], wide[:, 256:384], wide[:, 384:512], wide[:, 512:]
    r = kv.Rope(torch.tensor([1e4 ** (-2 * p / 64) for p in range(32)], dtype=torch.float64, device="cuda"))
    want = kv.append(cache, 0, batch, k, v, q, r, q_dtype=dtype)
    pool, before = cache.pool.clone(), wide[:, :512].clone()
    cache.pool.zero_()
    kv.append(cache, 0, batch, k, v, q, r, q_out=out)
    assert torch.equal(out, want) and torch.equal(cache.pool, pool) and torch.equal(wide[:, :512], before)


def test_append_leaves_out_what_has_no_place(kv):
    cache = kv.empty_cache(1, 4, 1, 64, 16, slots=3)
    cache.tables[0, 0], cache.tables[1, 0], cache.tables[1, 1], cache.tables[2, 0] = 0, 1, 99, 3
    cache.lens.copy_(_i32([3, 20, 5]))
    cache.pool.fill_(5.0)
    x = torch.ones((5 + 8 + 2 + 1, 1, 64), device="cuda")
    bad = _flag()
    # 5 tokens in a sequence of 3 (two have no place), 8 of 20 with the last 4 on a page outside the pool, 2 fine; a row behind
    out = torch.full((16, 1, 64), 9.0, device="cuda")
    kv.append(cache, 0, kv.Batch(_i32([0, 5, 13, 15]), 16, 8, 20), x, 2 * x, q=x, q_out=out, bad=bad)
    assert int(bad) == 1 and bool((out[:15] == 1).all()) and bool((out[15] == 9).all())
    pool = cache.pool.cpu()
    for row, n, first in [([0], 3, 0), ([1], 16, 12), ([3], 5, 3)]:
        k, v = kv_ref.read_cache(pool, row, 16, 16, 64)
        want = torch.full((16, 1, 64), 5.0)
        want[first:n] = 1.0
        assert torch.equal(k.float(), want)
        want[first:n] = 2.0
        assert torch.equal(v.float(), want)
    assert bool((pool[0, 2] == 5).all())
    bad.zero_()
    kv.append(cache, 0, kv.Batch(_i32([0, 2]), 2, 2, 20, _i32([7])), x[:2], x[:2], bad=bad)  # a slot outside the tables
    assert int(bad) == 1 and torch.equal(cache.pool.cpu(), pool)


def _random_cache(kv, rng, slots, cols, pages, page, layers=2):
    """A cache whose counts are right: rows of pages of their own and of shared full pages."""
    tables = np.full((slots, cols), -1, dtype=np.int32)
    lens, refs = np.zeros(slots, dtype=np.int32), np.zeros(pages, dtype=np.int32)
    free = list(rng.permutation(pages))
    for s in range(slots):
        n = int(rng.integers(0, cols * page // 2))
        for j in range(-(-n // page)):
            if s and j < lens[s - 1] // page and rng.random() < 0.3:
                tables[s, j] = tables[s - 1, j]
            elif free:
                tables[s, j] = free.pop()
            else:
                n = j * page
                break
            refs[tables[s, j]] += 1
        lens[s] = n
    pool = torch.from_numpy(rng.standard_normal((layers, pages, 1, 2 * page * 64)).astype(np.float32)).to(BF16)
    dev = lambda a: torch.from_numpy(a.copy()).cuda()  # noqa: E731
    return kv.Cache(pool.cuda(), dev(tables), dev(lens), dev(refs), page, 64), pool, tables, lens, refs


@pytest.mark.parametrize("seed", range(24))
def test_assign(kv, seed):
    """Random steps against the entries done one after the other: forks, admissions, growth and frees, entries that
    name slots twice or not at all, chains of replaced slots, pools that run out."""
    rng = np.random.default_rng(seed)
    slots, cols, page = int(rng.integers(2, 40)), int(rng.integers(2, 9)), int(rng.choice([16, 32]))
    cache, pool, tables, lens, refs = _random_cache(kv, rng, slots, cols, int(rng.integers(4, slots * cols + 5)), page)
    n = int(rng.integers(1, slots + 1))
    dst = rng.permutation(slots)[:n].astype(np.int32)
    src = np.where(rng.random(n) < 0.4, dst, rng.integers(-1, slots, n)).astype(np.int32)
    src = np.where(rng.random(n) < 0.2, -1, src).astype(np.int32)
    grow = (rng.integers(0, cols * page // 2, n) * (rng.random(n) < 0.7)).astype(np.int32)
    if seed % 3 == 0:  # entries that cannot be done
        for a, values in ((dst, [dst[0], -1, slots, 1 << 30]), (src, [-2, slots, -(1 << 30)]), (grow, [-1, 1 << 30])):
            a[rng.integers(0, n)] = rng.choice(values)
    want = (tables.copy(), lens.copy(), refs.copy())
    copies, wrong = kv_ref.assign(*want, page, dst.tolist(), src.tolist(), grow.tolist())
    bad = _flag()
    kv.assign(cache, *(torch.from_numpy(a).cuda() for a in (dst, src, grow)), bad=bad)
    for name, got, w in zip(("tables", "lens", "refs"), (cache.tables, cache.lens, cache.refs), want):
        assert np.array_equal(got.cpu().numpy(), w), name
    for a, b in copies:
        pool[:, b] = pool[:, a]
    assert torch.equal(cache.pool.cpu(), pool)
    assert int(bad) == int(wrong)


def test_assign_many_entries_and_pages(kv):
    """More entries than a workgroup's threads, more pages than one pass."""
    rng = np.random.default_rng(5)
    slots, cols, page, pages = 3000, 4, 16, 9000
    cache, pool, tables, lens, refs = _random_cache(kv, rng, slots, cols, pages, page, layers=1)
    dst = rng.permutation(slots).astype(np.int32)
    src = np.where(np.arange(slots) < 1500, -1, dst).astype(np.int32)
    grow = rng.integers(0, 20, slots).astype(np.int32)
    want = (tables.copy(), lens.copy(), refs.copy())
    copies, wrong = kv_ref.assign(*want, page, dst.tolist(), src.tolist(), grow.tolist())
    bad = _flag()
    kv.assign(cache, *(torch.from_numpy(a).cuda() for a in (dst, src, grow)), bad=bad)
    for name, got, w in zip(("tables", "lens", "refs"), (cache.tables, cache.lens, cache.refs), want):
        assert np.array_equal(got.cpu().numpy(), w), name
    assert not copies and torch.equal(cache.pool.cpu(), pool) and int(bad) == int(wrong)


def test_assign_wishes_beyond_any_pool(kv):
    """Growth whose pages, summed over the entries, pass 32 bits: none fits, what needs none is done."""
    cols, n = 1 << 20, 2200
    tables = torch.full((n + 1, cols), -1, dtype=torch.int32, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = kv.Cache(torch.zeros((1, 8, 1, 2 * 16 * 64), dtype=BF16, device="cuda"), tables, torch.zeros(n + 1, **i32),
                     torch.zeros(8, **i32), 16, 64)
    cache.lens[n], cache.tables[n, 0], cache.refs[5] = 3, 5, 1
    grow = torch.full((n + 1,), 16 * cols, **i32)
    grow[0], grow[n] = 7 * 16, 4
    bad = _flag()
    order = torch.arange(n + 1, **i32)
    kv.assign(cache, order, order, grow, bad=bad)
    assert int(bad) == 1 and cache.lens[0] == 112 and cache.lens[n] == 7 and int(cache.lens[1:n].sum()) == 0
    assert cache.tables[0, :8].tolist() == [0, 1, 2, 3, 4, 6, 7, -1] and cache.refs.tolist() == [1] * 8
    assert int((tables >= 0).sum()) == 8


def test_assign_reports_wrong_counts(kv):
    """A released page that no count covers, a row's entry outside the pool: reported, and nothing outside is touched."""
    cache = kv.empty_cache(1, 4, 1, 64, 16, slots=3)
    cache.tables[0, 0], cache.tables[1, 0] = 2, 77
    cache.lens.copy_(_i32([5, 5, 0]))
    bad = _flag()
    kv.assign(cache, _i32([0]), _i32([-1]), _i32([0]), bad=bad)  # page 2 has no reference
    assert int(bad) == 1 and cache.refs.tolist() == [0, 0, 0, 0] and cache.lens.tolist() == [0, 5, 0]
    bad.zero_()
    kv.assign(cache, _i32([2]), _i32([1]), _i32([0]), bad=bad)  # the open page to copy is outside the pool
    assert int(bad) == 1 and cache.tables[2, 0] == 0 and cache.lens.tolist() == [0, 5, 5]


def test_assign_passes_over_pages_that_a_window_has_left(kv):
    """Rows whose first pages are given back (-1, as attention allows): forked, freed, replaced and grown without a
    report, with exact counts; a fork's open page that is missing, and a number outside the pool, are reported."""
    cache = kv.empty_cache(2, 8, 1, 64, 16, slots=4, columns=6)
    cache.pool.copy_(torch.randn(cache.pool.shape, generator=torch.Generator().manual_seed(2)))
    pool = cache.pool.clone()
    cache.tables[0, :5] = _i32([-1, -1, 4, 2, 7])
    cache.lens[0] = 70
    cache.refs[[4, 2, 7]] = 1

    def step(dst, src, grow, tables, lens, refs, wrong=0):
        bad = _flag()
        kv.assign(cache, _i32(dst), _i32(src), _i32(grow), bad=bad)
        assert int(bad) == wrong and cache.tables.tolist() == tables and cache.lens.tolist() == lens and cache.refs.tolist() == refs

    none, left = [-1] * 6, [-1, -1, 4, 2]
    step([1], [0], [1], [left + [7, -1], left + [0, -1], none, none], [70, 71, 0, 0], [1, 0, 2, 0, 2, 0, 0, 1])
    pool[:, 0] = pool[:, 7]
    assert torch.equal(cache.pool, pool)
    step([0], [-1], [0], [none, left + [0, -1], none, none], [0, 71, 0, 0], [1, 0, 1, 0, 1, 0, 0, 0])
    step([1, 2], [1, 1], [10, 0], [none, left + [0, 1], left + [3, -1], none], [0, 81, 71, 0], [1, 1, 2, 1, 2, 0, 0, 0])
    pool[:, 3] = pool[:, 0]
    step([1], [-1], [20], [none, [0, 1] + none[2:], left + [3, -1], none], [0, 20, 71, 0], [1, 1, 1, 1, 1, 0, 0, 0])
    # the open page given back as well: released without a word, but nothing to copy for a fork
    cache.tables[2, 4], cache.refs[3] = -1, 0
    step([3], [2], [0], [none, [0, 1] + none[2:], left + none[:2], left + [3, -1]], [0, 20, 71, 71], [1, 1, 2, 1, 2, 0, 0, 0], 1)
    step([2], [-1], [0], [none, [0, 1] + none[2:], none, left + [3, -1]], [0, 20, 0, 71], [1, 1, 1, 1, 1, 0, 0, 0])
    for wrong in (-2, 8):
        cache.tables[3, 0] = wrong
        step([2], [3], [0], [none, [0, 1] + none[2:], [wrong] + left[1:] + [5, -1], [wrong] + left[1:] + [3, -1]], [0, 20, 71, 71],
             [1, 1, 2, 1, 2, 1, 0, 0], 1)
        pool[:, 5] = pool[:, 3]
        step([2], [-1], [0], [none, [0, 1] + none[2:], none, [wrong] + left[1:] + [3, -1]], [0, 20, 0, 71],
             [1, 1, 1, 1, 1, 0, 0, 0], 1)
    assert torch.equal(cache.pool, pool)


@pytest.mark.parametrize("seed", range(10))
@pytest.mark.parametrize("inplace", [True, False])
def test_compact(kv, seed, inplace):
    rng = np.random.default_rng(seed)
    slots, cols, page = int(rng.integers(1, 60)), int(rng.integers(1, 9)), 16
    cache, pool, tables, lens, refs = _random_cache(kv, rng, slots, cols, int(rng.integers(1, slots * cols + 2000 * (seed % 2) + 9)), page)
    if seed % 4 == 3:  # entries that name nothing: beyond the pool, or a page without references
        tables[0, -1] = len(refs) + 3
        empty = np.flatnonzero(refs == 0)
        if len(empty):
            tables[-1, -1] = empty[-1]
        cache.tables.copy_(torch.from_numpy(tables))
    want_tables, want_refs, moves, live, wrong = kv_ref.compact(tables, refs)
    bad = _flag()
    new = {} if inplace else dict(refs=torch.full_like(cache.refs, 9), tables=torch.full_like(cache.tables, 9))
    got = kv.compact(cache, **new, bad=bad)
    assert int(got) == live and int(bad) == int(wrong)
    assert np.array_equal((cache.refs if inplace else new["refs"]).cpu().numpy(), want_refs)
    assert np.array_equal((cache.tables if inplace else new["tables"]).cpu().numpy(), want_tables)
    if not inplace:  # the old ones stay, and read the same
        assert np.array_equal(cache.refs.cpu().numpy(), refs) and np.array_equal(cache.tables.cpu().numpy(), tables)
    for a, b in moves:
        pool[:, b] = pool[:, a]
    assert torch.equal(cache.pool.cpu(), pool)


@pytest.mark.parametrize("live", [4000, 4097, 9000])
@pytest.mark.parametrize("inplace", [True, False])
def test_compact_of_many_pages(kv, live, inplace):
    """More pages than the plan keeps in shared memory, most of them in holes."""
    rng = np.random.default_rng(live)
    pages, page = 20000, 16
    ids = np.sort(rng.permutation(pages)[:live])
    tables = np.full((live // 50 + 1, 60), -1, dtype=np.int32)
    for s, part in enumerate(np.array_split(rng.permutation(ids), len(tables))):
        tables[s, :len(part)] = part
    refs = np.zeros(pages, dtype=np.int32)
    refs[ids] = rng.integers(1, 4, live)
    pool = torch.from_numpy(rng.integers(0, 1 << 15, (1, pages, 1, 2 * page * 64), dtype=np.int16)).view(BF16)
    dev = lambda a: torch.from_numpy(a.copy()).cuda()  # noqa: E731
    cache = kv.Cache(pool.cuda(), dev(tables), torch.zeros(len(tables), dtype=torch.int32, device="cuda"), dev(refs), page, 64)
    want_tables, want_refs, moves, n, wrong = kv_ref.compact(tables, refs)
    new = {} if inplace else dict(refs=torch.full_like(cache.refs, 9), tables=torch.full_like(cache.tables, 9))
    bad = _flag()
    assert int(kv.compact(cache, **new, bad=bad)) == n == live and not wrong and int(bad) == 0
    assert np.array_equal((cache.refs if inplace else new["refs"]).cpu().numpy(), want_refs)
    assert np.array_equal((cache.tables if inplace else new["tables"]).cpu().numpy(), want_tables)
    bits = pool.view(torch.int16)
    bits[:, [b for _, b in moves]] = bits[:, [a for a, _ in moves]]
    assert torch.equal(cache.pool.cpu().view(torch.int16), bits)


def test_batches_that_change_between_replays(kv):
    """A captured batch of chunks and single tokens, and a captured compaction: starts, lengths and tables are other ones
    at each replay, eager work runs in between."""
    heads, kvh, d, page = 8, 2, 128, 16
    cache = kv.empty_cache(1, 300, kvh, d, page, slots=4, columns=60)
    g = torch.Generator(device="cuda").manual_seed(0)
    cache.pool.copy_(torch.randn(cache.pool.shape, generator=g, device="cuda"))
    starts, rows = _i32([0, 0, 0, 0, 0]), 150
    batch = kv.Batch(starts, rows, 100, 900)
    q = torch.randn((rows, heads, d), generator=g, device="cuda").to(BF16)
    kv.assign(cache, _i32([0, 1, 2, 3]), _i32([-1] * 4), _i32([100, 500, 3, 800]))
    out = torch.full_like(q, 5.0)
    kv.attention(cache, 0, batch, q, out=out)
    torch.cuda.synchronize()
    stream, graph, tidy = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            kv.attention(cache, 0, batch, q, out=out)
        with torch.cuda.graph(tidy, stream=stream):
            live = kv.compact(cache)
    torch.cuda.synchronize()
    for step, new in enumerate([[0, 100, 0, 1], [1, 1, 3, 1], [50, 33, 2, 60], [0, 0, 0, 9], [100, 0, 1, 40]]):
        starts.copy_(_i32(_starts(new)))
        out.fill_(5.0)
        want = kv.attention(cache, 0, batch, q, out=torch.full_like(q, 5.0))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and bool((out[sum(new):] == 5).all()) and bool(out.isfinite().all())
        kv.assign(cache, _i32([step % 4, (step + 1) % 4]), _i32([-1, (step + 2) % 4]), _i32([0, 60]))
        torch.cuda.synchronize()
        tidy.replay()
        torch.cuda.synchronize()
        used = int((cache.refs > 0).sum())
        assert int(live) == used and bool((cache.refs[:used] > 0).all())
        after = kv.attention(cache, 0, batch, q, out=torch.full_like(q, 5.0))
        assert bool(after.isfinite().all())
        kv.assign(cache, _i32([step % 4]), _i32([-1]), _i32([int(np.random.default_rng(step).integers(100, 800))]))
    cache.check()


def test_calls_on_a_stream_and_in_a_graph(kv):
    """A decoding step (grow, append, attention) captured once on a stream of its own and replayed as the sequences
    grow, eager work between the replays: each replay gives what the same calls give eagerly on a second cache."""
    heads, kvh, d, page, slots = 4, 2, 64, 16, 3
    g = torch.Generator(device="cuda").manual_seed(0)

    def fresh():
        c = kv.empty_cache(1, 40, kvh, d, page, slots=slots, columns=12)
        c.pool.fill_(math.nan)
        kv.assign(c, _i32([0, 1, 2]), _i32([-1, -1, -1]), _i32([30, 5, 100]))
        n = 135
        x = torch.Generator(device="cuda").manual_seed(7)
        k, v = (torch.randn((n, kvh, d), generator=x, device="cuda") for _ in range(2))
        kv.append(c, 0, kv.Batch(_i32([0, 30, 35, 135]), n, 100, 192), k, v)
        return c

    rope = kv.Rope(torch.tensor(kv.rope_freqs(d, 1e4)[0], dtype=torch.float64, device="cuda"))
    same, one = _i32([0, 1, 2]), _i32([1, 1, 1])
    batch = kv.Batch(_i32([0, 1, 2, 3]), slots, 1, 12 * page)
    q, k, v = (torch.zeros((slots, h, d), device="cuda") for h in (heads, kvh, kvh))

    def step(c):
        kv.assign(c, same, same, one)
        return kv.attention(c, 0, batch, kv.append(c, 0, batch, k, v, q, rope))

    eager, graphed = fresh(), fresh()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(graphed)
    torch.cuda.synchronize()
    for _ in range(5):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        want = step(eager)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and bool(out.isfinite().all())
        assert torch.equal(graphed.tables, eager.tables) and torch.equal(graphed.lens, eager.lens)


def test_the_operators_together(kv):
    """As a server uses them: a prompt in chunks, a fork, tokens for parent and child, a freed sequence, compaction,
    more tokens. Every step's attention is that of plain keys and values kept beside."""
    heads, kvh, d, page = 4, 2, 64, 16
    c = kv.empty_cache(2, 24, kvh, d, page, slots=4, columns=8)
    c.pool.fill_(math.nan)
    rng = torch.Generator().manual_seed(3)
    freqs, mag = kv.rope_freqs(d, 1e4)
    rope = kv.Rope(torch.tensor(freqs, dtype=torch.float64, device="cuda"))
    kept = {}  # slot -> (k, v) of layer 1

    def tokens(slots, news):
        rows, starts = sum(news), _starts(news)
        kv.assign(c, _i32(slots), _i32(slots), _i32(news))
        q, k, v = (torch.randn((rows, h, d), generator=rng) for h in (heads, kvh, kvh))
        b = kv.Batch(_i32(starts), rows, max(news), 8 * page, _i32(slots))
        for layer in (0, 1):
            qt = kv.append(c, layer, b, k.cuda(), v.cuda(), q.cuda(), rope)
        got = kv.attention(c, 1, b, qt, out_dtype=F32).cpu()
        pool, tables = c.pool.cpu(), c.tables.cpu()
        for s, n, r in zip(slots, news, starts):
            k0, v0 = kept.get(s, (torch.zeros(0, kvh, d, dtype=torch.float64),) * 2)
            place = np.arange(len(k0), len(k0) + n)
            kept[s] = torch.cat([k0, kv_ref.rope(k[r:r + n], place, freqs, 2, 1.0)]), torch.cat([v0, v[r:r + n].double()])
            # what the cache holds of all of the sequence: each value rounded once, wherever its pages have been since
            held = kv_ref.read_cache(pool, tables[s], len(kept[s][0]), page, d, layer=1)
            for h, want in zip(held, kept[s]):
                assert bool(((h.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -22 * 8).all()), (s, n)
            out, spread, reach = kv_ref.attention(qt[r:r + n].cpu(), *held, 0.125)
            assert bool(((got[r:r + n].double() - out).abs() <= kv_ref.attention_bound(out, spread, reach, d, BF16, F32)).all()), (s, n)

    tokens([0], [37])
    tokens([0, 2], [20, 9])
    kv.assign(c, _i32([1, 3]), _i32([0, 2]), _i32([0, 0]))  # forks: 57 tokens (an open page), 9
    kept[1], kept[3] = kept[0], kept[2]
    tokens([1, 0, 3, 2], [1, 1, 5, 1])
    kv.assign(c, _i32([0, 2]), _i32([-1, -1]), _i32([0, 0]))
    del kept[0], kept[2]
    live = int(kv.compact(c))
    assert live == sum(-(-len(kept[s][0]) // page) for s in kept) == int((c.refs > 0).sum()) and int(c.tables.max()) == live - 1
    tokens([3, 1], [30, 2])
    tokens([1], [1])


def test_stack_with_attention(kv):
    """The stack runner's layers with attention, a prompt in chunks (the last one ragged) and then another: every chunk's
    O input against attention in 64 bits over the keys and values that the layer's own matmuls gave."""
    from ggml_xdna_amd import stack
    cfg = stack.StackConfig("tiny", 2, 256, 256, 128, 512, 8, 8, 8, 8, 300, 128, head_dim=64, rope_base=1e4)
    s = stack.Stack(cfg, seed=1, attention=True)
    freqs, _ = kv.rope_freqs(64, 1e4)
    seen = []
    plain_append, plain_attention = kv.append, kv.attention

    def append(cache, layer, batch, k, v, **more):
        q = plain_append(cache, layer, batch, k, v, **more)
        seen.append((layer, k.clone().cpu(), v.clone().cpu(), q.clone().cpu()))
        return q

    def attention(cache, layer, batch, q, **more):
        out = plain_attention(cache, layer, batch, q, **more)
        seen[-1] += (out.clone().cpu(),)
        return out

    try:
        kv.append, kv.attention = append, attention
        s.run_prompt()
        first = s.h[:44].clone()
        s.run_prompt()
        assert torch.equal(s.h[:44], first)  # a prompt starts anew
    finally:
        kv.append, kv.attention = plain_append, plain_attention
    # the second prompt's keys and values are still in the cache: token t of every chunk's attention
    pool, tables = s.cache.pool.cpu(), s.cache.tables.cpu()
    done = {0: 0, 1: 0}
    for layer, k, v, q, out in seen[6:]:
        n = len(k)
        place = np.arange(done[layer], done[layer] + n)
        done[layer] += n
        held = kv_ref.read_cache(pool, tables[0], done[layer], 64, 64, layer)
        turned = kv_ref.rope(k.view(n, 2, 64), place, freqs, 2, 1.0)
        assert bool(((held[0][-n:].double() - turned).abs() <= 2.0 ** -8 * turned.abs() + 2.0 ** -22 * 8).all())
        assert torch.equal(held[1][-n:], v.view(n, 2, 64).to(BF16))
        want, spread, reach = kv_ref.attention(q.view(n, 4, 64), *held, 0.125)
        bound = kv_ref.attention_bound(want, spread, reach, 64, BF16, F32)
        assert bool(((out.view(n, 4, 64).double() - want).abs() <= bound).all())
    assert [len(x[1]) for x in seen[:6:2]] == [128, 128, 44] and len(seen) == 12
