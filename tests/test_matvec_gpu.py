"""Products of a few rows with GGUF weights against their 64-bit forms (decode_ref): every type, row counts, sizes at
the edges of chunks, blocks and tiles, groups, residuals, GLUs, strides, streams and graphs."""
from __future__ import annotations

import math

import decode_ref
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [2, 3, 8, 12, 20, 23]


@pytest.fixture(scope="module")
def z(zest_gpu):
    return zest_gpu


def _x(m, k, seed=0, outliers=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=g)
    if outliers:
        x[:, torch.randperm(k, generator=g)[:max(1, k // 200)]] *= 30.0
    return x


def _check(got, wtype, x, raw, extra=None):
    y, bound = decode_ref.matvec(wtype, x.numpy(), raw)
    if extra is not None:
        y = y + extra.double().numpy()
        bound = bound + 2.0 ** -23 * (np.abs(y) + bound)
    off = np.abs(got.cpu().double().numpy() - y)
    assert (off <= bound).all(), float((off / bound).max())
    return y, bound


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9, 16])
def test_every_type_and_row_count(z, wtype, m):
    k, n = 1280, 83
    x, raw = _x(m, k, m), decode_ref.gguf(wtype, n, k)
    _check(z.matvec(wtype, x.cuda(), [torch.from_numpy(raw).cuda()], [n])[0], wtype, x, raw)


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("n,blocks", [(1, 1), (15, 2), (16, 3), (17, 1), (33, 5), (600, 7), (5000, 1), (31, 19), (64, 41), (9, 68)])
def test_sizes(z, wtype, n, blocks):
    """One row and more, K from one block on: numbers of chunks that no split divides."""
    values = decode_ref.BLOCKS[wtype][0]
    for k in {values * blocks, 256 * blocks}:
        if k * n > 1_500_000:
            continue
        for m in (1, 6):
            x, raw = _x(m, k, n), decode_ref.gguf(wtype, n, k, 1)
            _check(z.matvec(wtype, x.cuda(), [torch.from_numpy(raw).cuda()], [n])[0], wtype, x, raw)


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("m", [1, 7, 16])
def test_long_rows(z, wtype, m):
    """K past what shared memory holds of x at once (16 rows of 17408, one row of 131072)."""
    k = 131072 if m == 1 else 17408
    x, raw = _x(m, k, 5), decode_ref.gguf(wtype, 19, k, 2)
    _check(z.matvec(wtype, x.cuda(), [torch.from_numpy(raw).cuda()], [19])[0], wtype, x, raw)


def test_many_rows(z):
    """More tiles than workgroups, several rounds of them; an N that ends inside a tile."""
    k, n = 256, 70001
    for wtype, m in ((12, 1), (2, 4), (8, 16)):
        x, raw = _x(m, k, 6), decode_ref.gguf(wtype, n, k, 3)
        _check(z.matvec(wtype, x.cuda(), [torch.from_numpy(raw).cuda()], [n])[0], wtype, x, raw)


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("m,ns", [(5, [33001]), (16, [20015, 1, 17003])])
def test_tall_weights_by_more_rows(z, wtype, m, ns):
    """32 weight rows a wave: heights that end inside 32 and inside 16, a weight of one row between two of many."""
    k = 768
    x, raws = _x(m, k, 8), [decode_ref.gguf(wtype, n, k, 20 + i) for i, n in enumerate(ns)]
    got = z.matvec(wtype, x.cuda(), [torch.from_numpy(r).cuda() for r in raws], ns)
    for y, raw in zip(got, raws):
        _check(y, wtype, x, raw)


@pytest.mark.parametrize("wtype", TYPES)
@pytest.mark.parametrize("m", [1, 4, 11])
def test_group_residuals_and_strides(z, wtype, m):
    """Four weights of different heights on an x with a stride, one output in columns of a wider buffer whose rest
    stays, a residual of its own, one in place and none."""
    k, ns = 512, [40, 7, 129, 16]
    x = _x(m, k, 7)
    wide = torch.full((m, k + 36), math.nan)
    wide[:, 32:32 + k] = x
    raws = [decode_ref.gguf(wtype, n, k, 10 + i) for i, n in enumerate(ns)]
    res = torch.randn((m, 40), generator=torch.Generator().manual_seed(1))
    place = torch.randn((m, 129), generator=torch.Generator().manual_seed(2))
    buf = torch.full((m, 64), 7.0, device="cuda")
    outs = [torch.empty((m, 40), device="cuda"), buf[:, 3:10], place.cuda(), torch.empty((m, 16), device="cuda")]
    got = z.matvec(wtype, wide.cuda()[:, 32:32 + k], [torch.from_numpy(r).cuda() for r in raws], ns, outs=outs,
                   residuals=[res.cuda(), None, outs[2], None])
    for i, extra in enumerate((res, None, place, None)):
        _check(got[i], wtype, x, raws[i], extra)
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 10:] == 7).all())


@pytest.mark.parametrize("kind", range(5))
@pytest.mark.parametrize("wtype,m,f,k", [(12, 1, 50, 512), (2, 3, 16, 96), (8, 16, 33, 320), (23, 4, 130, 256), (3, 2, 2100, 64), (20, 8, 17, 64)])
def test_glu(z, kind, wtype, m, f, k):
    x = 0.5 * _x(m, k, kind, outliers=False)
    gate, up = (decode_ref.gguf(wtype, f, k, s) for s in (1, 2))
    got = z.matvec_glu(kind, wtype, x.cuda(), torch.from_numpy(gate).cuda(), torch.from_numpy(up).cuda(), f).cpu().double().numpy()
    (g, eg), (u, eu) = decode_ref.matvec(wtype, x.numpy(), gate), decode_ref.matvec(wtype, x.numpy(), up)
    off, bound = np.abs(got - decode_ref.glu(kind, g, u)), decode_ref.glu_bound(g, eg, u, eu)
    assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("wtype", TYPES)
def test_values_of_any_size(z, wtype):
    """Blocks of zeros, of one value, of the smallest and largest magnitudes side by side; codes at their ends. Magnitudes
    below 2^-100 of a block may count as zero."""
    k = 512
    x = torch.zeros((3, k))
    x[0, 5], x[0, 33] = 1.5, -2.0 ** -90
    x[1] = torch.randn(k, generator=torch.Generator().manual_seed(3)) * torch.exp2(torch.arange(k) // 32 * 8.0 - 60)
    x[2, 256:] = 1e30
    for fill in (0x00, 0xff, 0x77, 0x80):
        raw = decode_ref.gguf(wtype, 20, k, 4).reshape(20, -1, decode_ref.BLOCKS[wtype][1])
        raw[:, :, 4 if wtype in (3, 12, 23) else 2:] = fill
        raw = raw.reshape(20, -1)
        _check(z.matvec(wtype, x.cuda(), [torch.from_numpy(raw).cuda()], [20])[0], wtype, x, raw)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("wtype,m", [(12, 3), (2, 3), (8, 9)])
def test_nonfinite_rows(z, value, wtype, m):
    """A row with a NaN or an infinity is NaN in whole; the others are what they are without it."""
    k, n = 1024, 40
    x, raw = _x(m, k, 8), decode_ref.gguf(wtype, n, k, 5)
    w = torch.from_numpy(raw).cuda()
    want = z.matvec(wtype, x.cuda(), [w], [n])[0].clone()
    x[1, 700] = value
    got = z.matvec(wtype, x.cuda(), [w], [n])[0]
    assert bool(got[1].isnan().all())
    rest = [i for i in range(m) if i != 1]
    assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("wtype", [2, 8, 20])
def test_a_weight_s_infinite_scale(z, wtype):
    """An infinite or NaN scale makes its row what IEEE arithmetic makes it, and no other."""
    k, n = 64, 18
    x, raw = _x(1, k, 9).abs() + 0.1, decode_ref.gguf(wtype, n, k, 6)
    r = raw.reshape(n, 2, -1)
    r[3, 1, :2] = np.frombuffer(np.float16(np.inf).tobytes(), dtype=np.uint8)
    r[3, 1, 2:] = 0x99 if wtype != 8 else 1
    got = z.matvec(wtype, x.cuda(), [torch.from_numpy(raw).cuda()], [n])[0].cpu()
    assert not bool(got[0, 3].isfinite())
    rest = [i for i in range(n) if i != 3]
    _check(got[:, rest], wtype, x, raw[rest])


def test_unaligned_weights(z):
    """Rows at the least alignment that the header asks for."""
    for wtype, align in ((2, 2), (20, 2), (8, 2), (3, 4), (23, 8), (12, 16)):
        k, n = 768, 37
        raw = decode_ref.gguf(wtype, n, k, 7)
        buf = torch.zeros(raw.size + 256, dtype=torch.uint8, device="cuda")
        w = buf[align:align + raw.size]
        w.copy_(torch.from_numpy(raw.reshape(-1)))
        for m in (2, 9):
            x = _x(m, k, 3)
            _check(z.matvec(wtype, x.cuda(), [w], [n])[0], wtype, x, raw)


@pytest.mark.parametrize("m", [2, 13])
def test_bits_do_not_vary(z, m):
    """The same bits from run to run and on another stream."""
    k, n, wtype = 2560, 1000, 12
    x, raw = _x(m, k, 4).cuda(), torch.from_numpy(decode_ref.gguf(wtype, n, k, 8)).cuda()
    want = z.matvec(wtype, x, [raw], [n])[0].clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(5):
            assert torch.equal(z.matvec(wtype, x, [raw], [n])[0], want)


@pytest.mark.parametrize("m", [3, 16])
def test_in_graphs_and_at_once(z, m):
    """Captured with a workspace of its own, replayed with the program's work between, new x and weights; two graphs and
    an eager call with a workspace each run at once."""
    k, n, wtype = 1024, 3000, 2
    raws = [decode_ref.gguf(wtype, n, k, s) for s in (1, 2, 3)]
    xs = [_x(m, k, s).cuda() for s in (1, 2, 3)]
    ws = [torch.from_numpy(r).cuda() for r in raws]
    eager = [z.matvec(wtype, x, [w], [n])[0].clone() for x, w in zip(xs, ws)]
    bytes_ = z.matvec_workspace(wtype, m, k, [n])
    outs = [torch.zeros((m, n), device="cuda") for _ in range(3)]
    spaces = [torch.empty(max(16, bytes_), dtype=torch.uint8, device="cuda") for _ in range(3)]
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            z.matvec(wtype, xs[i], [ws[i]], [n], outs=[outs[i]], workspace=spaces[i])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            z.matvec(wtype, xs[2], [ws[2]], [n], outs=[outs[2]], workspace=spaces[2])
        torch.cuda.synchronize()
        assert all(torch.equal(o, e) for o, e in zip(outs, eager)), turn
        xs[0].copy_(xs[1] if turn % 2 else xs[2])
        eager[0] = z.matvec(wtype, xs[0], [ws[0]], [n])[0].clone()


def test_offsets_past_32_bits(z):
    """A weight of more than 4 GiB: its last rows."""
    k, n = 1 << 20, 8000
    row = decode_ref.gguf(2, 1, k, 9)
    w = torch.zeros((n, row.size), dtype=torch.uint8, device="cuda")
    w[-1] = torch.from_numpy(row[0]).cuda()
    w[-17] = w[-1]
    x = _x(1, k, 2)
    got = z.matvec(2, x.cuda(), [w.view(-1)], [n])[0]
    for i in (-1, -17):
        _check(got[:, [i]], 2, x, row)
    assert bool((got[0, :-17] == 0).all()) and bool((got[0, -16:-1] == 0).all())
