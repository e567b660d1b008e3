"""Attention over shared leading pages against the plain 64-bit form, a sequence at a time: groups of every size, shared
lengths around pages and tiles, masks, tables that agree for less than the group says or not at all."""
from __future__ import annotations

import math

import kv_ref
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


def _flag():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


class Case:
    """groups: lists of (new tokens, length) of sequences that name their first member's first `shared` pages."""

    def __init__(self, kv, groups, page=16, kv_heads=2, group=2, d=64, dtype=BF16, seed=0, max_shared=None):
        seqs = [s for _, members in groups for s in members]
        self.new, self.lens = [n for n, _ in seqs], [m for _, m in seqs]
        b = self.book = kv_ref.Book(self.lens, page, kv_heads, d, dtype, seed)
        at, starts = 0, [0]
        for pages, members in groups:
            for i in range(at + 1, at + len(members)):
                b.table[i, :pages] = b.table[at, :pages]
                t = min(pages * page, self.lens[i], self.lens[at])
                b.k[i][:t], b.v[i][:t] = b.k[at][:t], b.v[at][:t]
            at += len(members)
            starts.append(at)
        self.starts = [sum(self.new[:i]) for i in range(len(self.new) + 1)]
        self.rows, self.heads = self.starts[-1], kv_heads * group
        g = torch.Generator().manual_seed(seed + 1)
        self.q = (2.0 * torch.randn((self.rows, self.heads, d), generator=g)).to(dtype)
        b.pool.fill_(math.nan)
        b.fill()
        self.cache = b.cache(kv)
        self.batch = kv.Batch(_i32(self.starts), self.rows, max(self.new + [1]), max(self.lens + [1]))
        self.groups = kv.Groups(_i32(starts), max(self.lens) if max_shared is None else max_shared, always=True)

    def run(self, kv, **more):
        return kv.attention(self.cache, 0, self.batch, self.q.cuda(), groups=self.groups, **more)

    def check(self, got, causal=True, window=0, softcap=0.0, scale=None, unseen=None):
        b = self.book
        scale = 1.0 / math.sqrt(b.d) if scale is None else scale
        got = got.cpu().reshape(self.rows, self.heads, b.d)
        for i, n in enumerate(self.new):
            r = slice(self.starts[i], self.starts[i] + n)
            out, spread, reach = kv_ref.attention(self.q[r], b.k[i], b.v[i], scale, causal, window, softcap,
                                                  unseen=None if unseen is None else unseen[i])
            bound = kv_ref.attention_bound(out, spread, reach, b.d, b.dtype, got.dtype)
            off = (got[r].double() - out).abs()
            assert bool((off <= bound).all()), (i, n, b.lens[i], float((off / bound).max()))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,group,page", [(64, 1, 16), (64, 2, 32), (96, 3, 64), (128, 4, 64), (128, 6, 128), (192, 5, 16), (256, 8, 32),
                                          (128, 16, 16), (64, 33, 16)])
def test_groups(kv, dtype, d, group, page):
    """Every head width, page size and group shape; groups of one, a few and many sequences; own tokens from one to more
    than a unit; a group that shares nothing."""
    p = page
    groups = [(3, [(1, 3 * p + 1), (1, 3 * p + 7), (1, 5 * p)]), (2, [(1, 2 * p + 5)]), (0, [(1, 40), (1, 9)]),
              (7, [(1, 7 * p + 1 + 13 * i) for i in range(12)]), (1, [(2, p + 2), (1, p + 150)])]
    c = Case(kv, groups, page, 2 if group < 8 else 1, group, d, dtype, seed=d + group)
    bad = _flag()
    got = c.run(kv, bad=bad)
    assert got.dtype == dtype and got.shape == c.q.shape
    c.check(got)
    assert int(bad) == 0


@pytest.mark.parametrize("members,new", [(2, 1), (5, 3), (40, 1), (3, 17), (4, 40), (2, 90)])
@pytest.mark.parametrize("d,group", [(64, 4), (128, 4), (192, 3), (256, 2)])
def test_columns(kv, members, new, d, group):
    """From two columns of a group to several tiles of them; sequences of so many new tokens that they are chunks."""
    groups = [(9, [(new, 9 * 32 + new + 11 * i) for i in range(members)]), (0, [(1, 77)])]
    c = Case(kv, groups, 32, 2, group, d, BF16, seed=d + new)
    c.check(c.run(kv))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window,softcap,scale", [(0, 0.0, 0.3), (7, 0.0, None), (100, 5.0, None), (2000, 0.0, None), (0, 2.0, None),
                                                  (0, 100.0, None), (0, 0.0, 0.0), (0, 0.0, -0.2)])
def test_masks(kv, causal, window, softcap, scale):
    groups = [(6, [(1, 200), (3, 203), (1, 193)]), (10, [(20, 345), (9, 400), (70, 420)])]
    c = Case(kv, groups, 32, 2, 3, 64, BF16, seed=window)
    c.check(c.run(kv, scale=scale, causal=causal, window=window, softcap=softcap), causal, window, softcap, scale)


@pytest.mark.parametrize("page,max_shared", [(16, 0), (16, 15), (16, 16), (16, 100), (64, 63), (64, 64), (64, 10 ** 6), (256, 300)])
def test_what_is_shared_is_found(kv, page, max_shared):
    """Tables that agree for more than max_shared, and for less than the group's members hold; a member whose new tokens
    lie inside the shared pages, so that a row does not see all of them; a member that ends there."""
    groups = [(4, [(1, 4 * page + 3), (5, 4 * page + 1), (1, 4 * page), (3, 2 * page + 1), (1, page)]), (5, [(1, 6 * page), (6, 6 * page)])]
    c = Case(kv, groups, page, 2, 4, 64, BF16, seed=page, max_shared=max_shared)
    c.check(c.run(kv))


def test_tables_that_differ(kv):
    """Groups whose members' tables differ from some page on, at once, or by a page that is gone: each sequence gets
    its own tokens, the missing page is reported."""
    c = Case(kv, [(6, [(1, 120), (1, 119), (1, 130)]), (5, [(2, 100), (1, 95)])], 16, 2, 4, 64, BF16, seed=4)
    own = kv_ref.Book(c.lens, 16, 2, 64, BF16, 77)  # other keys for one member of the first group, from page 2 on
    spare = c.book.pages
    c.book.pool = torch.cat([c.book.pool, torch.full((1, 9, 2, 2 * 16 * 64), math.nan, dtype=BF16)], dim=1)
    c.book.refs = torch.cat([c.book.refs, torch.ones(9, dtype=torch.int32)])
    c.book.table[1, 2:8] = torch.arange(spare, spare + 6, dtype=torch.int32)
    c.book.k[1][32:], c.book.v[1][32:] = own.k[1][32:], own.v[1][32:]
    c.book.fill()
    c.cache = c.book.cache(kv)
    bad = _flag()
    c.check(c.run(kv, bad=bad))
    assert int(bad) == 0
    # page 1 of the second group is gone from both tables; of the first group from one
    c.cache.tables[3:5, 1] = -1
    c.cache.tables[2, 0] = 1 << 30
    unseen = [None, None, torch.arange(130) < 16, (torch.arange(100) // 16) == 1, (torch.arange(95) // 16) == 1]
    c.check(c.run(kv, bad=bad), unseen=unseen)
    assert int(bad) == 1


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16), (96, F16), (192, BF16)])
def test_long_prompts(kv, d, dtype):
    """Shared contexts long enough that their keys are split among workgroups, own ones of any length; the same bits
    from run to run."""
    groups = [(70, [(1, 70 * 64 + 1 + 37 * i) for i in range(9)]), (20, [(1, 1281), (2, 1400)]), (0, [(1, 2500)])]
    c = Case(kv, groups, 64, 2, 4, d, dtype, seed=d)
    got = c.run(kv, out_dtype=F32)
    c.check(got)
    for _ in range(3):
        assert torch.equal(c.run(kv, out_dtype=F32), got)


@pytest.mark.parametrize("count", [63, 64, 65, 300])
def test_many_groups_and_sequences(kv, count):
    """More groups and sequences than a wave's lanes and than a workgroup's threads; sequences without new tokens."""
    groups = []
    for i in range(count):
        members = [(0 if (i + j) % 7 == 3 else 1 + (i % 3), 33 + (5 * i + 3 * j) % 40) for j in range(1 + i % 3)]
        groups.append((i % 3, members))
    c = Case(kv, groups, 16, 1, 2, 64, BF16, seed=count)
    bad = _flag()
    c.check(c.run(kv, bad=bad))
    assert int(bad) == 0


def test_values_a_row_does_not_see(kv):
    """NaN and infinities in shared and own places: they reach the rows that see them and no other."""
    c = Case(kv, [(4, [(3, 80), (1, 70), (1, 64)])], 16, 2, 2, 64, F16, seed=6)
    want = c.run(kv).float().cpu()
    c.book.v[0][79, :, 5] = math.nan   # seen by sequence 0's last row alone
    c.book.v[1][66, :, 6] = math.inf
    c.book.fill()
    c.cache = c.book.cache(kv)
    got = c.run(kv).float().cpu()
    assert bool(got[2, :, 5].isnan().all()) and bool(got[3, :, 6].isinf().all())
    seen = torch.ones_like(got, dtype=torch.bool)
    seen[2, :, 5] = seen[3, :, 6] = False
    assert torch.equal(got[seen], want[seen])
    for b in range(3):
        c.book.v[b][10, 0, 7] = -math.inf  # shared: every row of the k/v head
    c.book.fill()
    c.cache = c.book.cache(kv)
    got = c.run(kv).float().cpu()
    assert bool((got[:, :2, 7] == -math.inf).all())


def test_rows_left_as_they_were(kv):
    """Rows behind the last sequence, sequences outside all groups, slots in another order, q and out as columns."""
    c = Case(kv, [(2, [(1, 50), (2, 40), (1, 35)]), (1, [(1, 20), (1, 30)])], 16, 2, 2, 64, BF16, seed=8)
    out = torch.full((c.rows + 3, 304), 7.0, dtype=BF16, device="cuda")
    q = torch.zeros((c.rows + 3, 512), dtype=BF16, device="cuda")
    q[:c.rows, 256:] = c.q.reshape(c.rows, 256).cuda()
    batch = kv.Batch(c.batch.starts, c.rows + 3, 2, 50)
    for starts in ([0, 3, 5], [1, 3], [0, 0, 5], [5, 5], [0, 2]):
        out.fill_(7.0)
        kv.attention(c.cache, 0, batch, q[:, 256:], out=out[:, 24:280], groups=kv.Groups(_i32(starts), 64, always=True))
        c.check(out[:c.rows, 24:280])
        assert bool((out[c.rows:] == 7).all()) and bool((out[:, :24] == 7).all()) and bool((out[:, 280:] == 7).all())
    order = [3, 0, 4, 2, 1]
    c2 = kv.Cache(c.cache.pool, c.cache.tables[order].contiguous(), c.cache.lens[order].contiguous(), c.cache.refs, 16, 64)
    slots = _i32([order.index(i) for i in range(5)])
    got = kv.attention(c2, 0, kv.Batch(c.batch.starts, c.rows, 2, 50, slots), c.q.cuda(), groups=c.groups)
    c.check(got)


def test_bad_groups_are_reported(kv):
    """Starts that go back or lie outside the batch: reported, those groups share nothing, the result is what it is."""
    c = Case(kv, [(2, [(1, 50), (1, 40), (1, 35)]), (2, [(1, 60), (1, 61)])], 16, 2, 2, 64, BF16, seed=9)
    for starts in ([0, 9], [-1, 3], [3, 0, 5], [2, 1], [0, 3, 2 ** 31 - 1], [-2 ** 31, 5]):
        bad = _flag()
        c.check(kv.attention(c.cache, 0, c.batch, c.q.cuda(), groups=kv.Groups(_i32(starts), 64, always=True), bad=bad))
        assert int(bad) == 1, starts


def test_bad_batches(kv):
    """A slot outside the tables, a length past the bounds: that sequence is left out and reported, its group goes on."""
    c = Case(kv, [(2, [(1, 50), (1, 40), (1, 35), (1, 36)])], 16, 2, 2, 64, BF16, seed=10)
    for slots, lens in (([0, 99, 2, 3], None), ([0, 1, 2, -1], None), ([0, 1, 2, 3], (2, 10 ** 6)), ([0, 1, 2, 3], (0, -5))):
        cache = c.book.cache(kv)
        if lens:
            cache.lens[lens[0]] = lens[1]
        bad = _flag()
        out = torch.full((4, 4, 64), 7.0, dtype=BF16, device="cuda")
        kv.attention(cache, 0, kv.Batch(c.batch.starts, 4, 1, 50, _i32(slots)), c.q.cuda(), out=out, groups=c.groups, bad=bad)
        gone = lens[0] if lens else [i for i in range(4) if not 0 <= slots[i] < 4][0]
        assert int(bad) == 1 and bool((out[gone] == 7).all())
        want = c.run(kv)
        rest = [i for i in range(4) if i != gone]
        out[gone] = want[gone]
        c.check(out)


def test_in_a_graph_with_forks(kv):
    """A captured decoding step (fork, append, attention by groups) replayed while lengths and shared pages change,
    against the same calls without groups, eager work between the replays."""
    heads, kvh, d, page = 8, 2, 64, 16
    cache = kv.empty_cache(1, 200, kvh, d, page, slots=8)
    g = torch.Generator(device="cuda").manual_seed(5)
    prompt = 100
    batch = kv.Batch(_i32([0, prompt]), prompt, prompt, prompt)
    kv.assign(cache, _i32([0]), _i32([-1]), _i32([prompt]))
    kv.append(cache, 0, batch, *(torch.randn((prompt, kvh * d), generator=g, device="cuda") for _ in range(2)))
    kv.assign(cache, _i32(list(range(1, 8))), _i32([0] * 7), _i32([0] * 7))
    step = kv.Batch(_i32(list(range(9))), 8, 1, 400)
    groups = kv.Groups(_i32([0, 8]), 400, always=True)
    q, k, v = (torch.randn((8, n * d), generator=g, device="cuda") for n in (heads, kvh, kvh))
    every, one = _i32(list(range(8))), _i32([1] * 8)
    out = torch.zeros((8, heads * d), device="cuda")
    space = torch.empty(kv.attention_workspace(cache, step, heads, groups), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kv.assign(cache, every, every, one)
        kv.append(cache, 0, step, k, v)
        kv.attention(cache, 0, step, q, out=out, groups=groups, workspace=space)
    for turn in range(40):
        for t in (q, k, v):
            t.normal_(generator=g)
        if turn == 20:  # the prompt's fourth page is replaced in some tables
            kv.assign(cache, _i32([3]), _i32([-1]), _i32([55]))
        graph.replay()
        want = kv.attention(cache, 0, step, q)
        torch.cuda.synchronize()
        # both forms round each weight once and differ in the order of their sums alone
        b = 2.0 ** -8 * 4.0 + 2.0 ** -10
        assert bool(((out - want).abs() <= b).all()), turn
    cache.check()


def test_groups_that_save_little_are_passed_over(kv):
    """By sizes and bounds: the sequences are then read one by one, bit for bit as without groups, and bad starts are
    still reported."""
    c = Case(kv, [(20, [(1, 100 + 3 * i) for i in range(6)])], 32, 2, 4, 128, BF16, seed=4)
    q, want = c.q.cuda(), kv.attention(c.cache, 0, c.batch, c.q.cuda())
    few = kv.Groups(c.groups.starts, 10 ** 4)
    assert torch.equal(kv.attention(c.cache, 0, c.batch, q, groups=few), want)
    assert kv.attention_workspace(c.cache, c.batch, 8, few) == kv.attention_workspace(c.cache, c.batch, 8)
    assert kv.attention_workspace(c.cache, c.batch, 8, c.groups) > kv.attention_workspace(c.cache, c.batch, 8)
    bad = _flag()
    assert torch.equal(kv.attention(c.cache, 0, c.batch, q, groups=kv.Groups(_i32([0, 99]), 64), bad=bad), want) and int(bad) == 1


def test_two_calls_at_once(kv):
    cs = [Case(kv, [(20, [(1, 700 + i) for i in range(6)])], 32, 2, 4, 128, BF16, seed=s) for s in (1, 2)]
    want = [c.run(kv, out_dtype=F32).clone() for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = []
    for _ in range(4):
        for c, st in zip(cs, streams):
            with torch.cuda.stream(st):
                got.append(c.run(kv, out_dtype=F32))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i % 2]) for i, a in enumerate(got))
