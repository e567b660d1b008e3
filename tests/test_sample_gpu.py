"""The next token's choice against its definition in whole numbers (decode_ref)."""
from __future__ import annotations

import math

import decode_ref
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def s(zest_gpu):
    from ggml_xdna_amd import sampling
    return sampling


def _logits(rows, vocab, dtype=torch.float32, spread=2.5, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn((rows, vocab), generator=g)
    x[:, :max(1, vocab // 50)] += spread
    return x[:, torch.randperm(vocab, generator=g)].to(dtype)


def _f(v):
    return None if v is None else torch.tensor(v, dtype=torch.float32, device="cuda")


def _i(v):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")


def _check(s, x, u, t=None, k=None, p=None, m=None, **more):
    tokens, probs = s.sample(x.cuda() if not x.is_cuda else x, _f(u), _f(t), _i(k), _f(p), _f(m), probs=True, **more)
    tokens, probs, rows = tokens.cpu().tolist(), probs.cpu().tolist(), x.double().cpu().numpy()
    for r in range(len(u)):
        stay, w = decode_ref.kept(rows[r], np.float32(t[r]) if t else 1.0, k[r] if k else 0, p[r] if p else 1.0, m[r] if m else 0.0)
        assert decode_ref.fits(tokens[r], probs[r], stay, w, u[r]), (r, tokens[r], probs[r], len(stay))
    return tokens


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 4097, 32003])
def test_every_parameter(s, dtype, vocab):
    rng = np.random.default_rng(vocab)
    n = 24
    x = _logits(n, vocab, dtype, seed=vocab)
    u = [float(v) for v in rng.random(n)]
    t = [float(v) for v in rng.choice([0.2, 0.7, 1.0, 1.5, 0.0], n)]
    k = [int(v) for v in rng.choice([0, 1, 2, 20, 200, vocab, 10 * vocab], n)]
    p = [float(v) for v in rng.choice([0.0, 0.3, 0.8, 0.95, 1.0, 2.0], n)]
    m = [float(v) for v in rng.choice([0.0, 0.01, 0.2, 1.0, 1.5, -1.0], n)]
    _check(s, x, u, t, k, p, m)
    _check(s, x, u)
    _check(s, x, u, t)
    _check(s, x, u, None, k)
    _check(s, x, u, None, None, p)
    _check(s, x, u, None, None, None, m)
    _check(s, x, u, t, k, None, m)


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 151936), (torch.bfloat16, 128256), (torch.float16, 262144)])
def test_large_vocabularies(s, dtype, vocab):
    x = _logits(6, vocab, dtype, seed=vocab)
    u = [0.0, 0.1, 0.5, 0.77, 0.999, 0.9999999]
    _check(s, x, u, [1.0] * 6)
    _check(s, x, u, [0.8] * 6, [50, 1, 20000, 5, 3000, 100000], [0.9, 0.9, 0.99, 0.5, 0.95, 0.7])
    _check(s, x, u, [1.2] * 6, None, [0.3, 0.9, 0.95, 0.99, 0.999, 0.9999])
    _check(s, x, u, None, None, None, [0.001, 0.01, 0.1, 0.2, 0.05, 0.5])


@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.1, 30.0, 1e4])
@pytest.mark.parametrize("vocab", [5000, 70000])
def test_flat_and_steep_rows(s, spread, vocab):
    """All logits equal, nearly so, or one above all: cuts among ties, and among very many logits."""
    for dtype in (torch.float32, torch.bfloat16):
        x = _logits(5, vocab, dtype, spread, seed=3)
        u = [0.0, 0.25, 0.5, 0.75, 0.99999]
        _check(s, x, u, None, [7, 64, 1000, 4999, 2500], None, None)
        _check(s, x, u, [2.0] * 5, None, [0.1, 0.5, 0.9, 0.99, 0.0])
        _check(s, x, u, None, [100, 3000, 4000, 10, 1], [0.5, 0.9, 0.3, 0.7, 0.9], [0.5, 0.0, 0.9, 0.1, 0.0])


def test_ties_go_to_the_lowest_index(s):
    x = torch.full((1, 300), -1.0)
    x[0, [7, 70, 200, 299]] = 3.0
    x[0, 100] = 5.0
    # five largest by rank: 100, 7, 70, 200, 299
    for k, want in ((1, [100]), (2, [7, 100]), (3, [7, 70, 100]), (4, [7, 70, 100, 200])):
        got = {_check(s, x, [u], None, [k])[0] for u in np.linspace(0, 0.9999, 60)}
        assert got == set(want)
    assert _check(s, x - 100 * (torch.arange(300) == 100), [0.9], [0.0])[0] == 7
    # minus zero is zero
    x = torch.tensor([[-0.0, 0.0, -0.0, -1.0]])
    assert {_check(s, x, [u], None, [2])[0] for u in (0.0, 0.3, 0.6, 0.99)} == {0, 1}


@pytest.mark.parametrize("vocab", [1000, 5000, 30000])
def test_masked_and_odd_logits(s, vocab):
    """-infinity and NaN are never taken, whatever u; +infinity takes all; a row of nothing gives -1."""
    x = torch.full((8, vocab), -math.inf)
    x[0, 321] = -5.0
    x[1, ::3] = math.nan
    x[1, 10::50] = 1.0
    x[2, 5] = x[2, vocab - 100] = math.inf
    x[2, 30:60] = 1e30
    x[4] = math.nan
    x[5, vocab - 1] = -3e38
    x[6, 0] = 3.4e38
    x[6, 1] = -3.4e38
    x[7] = torch.randn(vocab, generator=torch.Generator().manual_seed(1))
    x[7, ::2] = -math.inf
    for u in (0.0, 0.4, 0.6, 1.0 - 2.0 ** -24):
        for more in (dict(), dict(k=[vocab // 10] * 8), dict(p=[0.9] * 8), dict(m=[0.5] * 8), dict(p=[0.9] * 8, m=[1e-3] * 8), dict(t=[0.0] * 8), dict(t=[math.inf] * 8)):
            tokens = _check(s, x, [u] * 8, **more)
            assert tokens[0] == 321 and tokens[3] == tokens[4] == -1 and tokens[2] in (5, vocab - 100) and tokens[5] == vocab - 1 and tokens[6] <= 1
            assert tokens[7] % 2 == 1


@pytest.mark.parametrize("vocab", [777, 20001])
def test_odd_parameters(s, vocab):
    """NaN, infinite and negative parameters are read as the header says."""
    x = _logits(9, vocab, seed=5)
    nan, inf = math.nan, math.inf
    _check(s, x, [nan, -1.0, 1.0, 2.0, inf, -inf, 0.5, 0.5, 0.5])
    u = [0.6] * 9
    _check(s, x, u, [nan, -1.0, inf, 1e-30, 1e-45, 1e30, 0.0, -inf, 1.0])
    _check(s, x, u, None, [-5, 0, 1, vocab - 1, vocab, vocab + 1, 2 ** 31 - 1, -2 ** 31, 2])
    _check(s, x, u, None, None, [nan, -1.0, 0.0, 1e-45, 1.0, inf, -inf, 0.5, 2.0])
    _check(s, x, u, None, None, None, [nan, -1.0, 0.0, 1e-45, 1.0, inf, -inf, 0.5, 2.0])


@pytest.mark.parametrize("vocab", [777, 20001])
def test_tiny_temperatures(s, vocab):
    """Logits that lie closer than a histogram's narrowest bin, but far apart by their temperature."""
    x = 1e-42 * _logits(4, vocab, seed=6, spread=1.0)
    u = [0.0, 0.3, 0.6, 0.999]
    for t in (1e-45, 1e-43, 1e-42, 1e-30):
        _check(s, x, u, [t] * 4)
        _check(s, x, u, [t] * 4, [3, 50, 700, 5000])
        _check(s, x, u, [t] * 4, None, [0.1, 0.9, 0.99, 0.5])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_any_stride_and_alignment(s, dtype):
    wide = torch.full((7, 3001), math.inf, dtype=dtype)
    x = _logits(7, 2900, dtype, seed=8)
    for at in (1, 2, 3, 7):
        wide[:] = math.inf
        wide[:, at:at + 2900] = x
        _check(s, wide.cuda()[:, at:at + 2900], [0.1 * i for i in range(7)], [0.9] * 7, [40] * 7, [0.95] * 7, [0.01] * 7)
        _check(s, wide.cuda()[:, at:at + 2900], [0.1 * i for i in range(7)])


@pytest.mark.parametrize("rows,vocab", [(300, 500), (2000, 100), (65, 40000), (270, 8193), (257, 16385)])
def test_many_rows(s, rows, vocab):
    x = _logits(rows, vocab, seed=rows)
    u = [(i * 0.6180339887) % 1.0 for i in range(rows)]
    _check(s, x, u, [0.5 + (i % 5) * 0.3 for i in range(rows)], [(i * 7) % 60 for i in range(rows)], [1.0 - (i % 4) * 0.1 for i in range(rows)],
           [0.0 if i % 3 else 0.02 for i in range(rows)])


def test_draws_follow_the_distribution(s):
    """u over a fine grid takes each token for as much of it as its share."""
    x = _logits(1, 50, seed=2)
    n = 20000
    u = ((torch.arange(n) + 0.5) / n).cuda()
    tokens = s.sample(x.cuda().expand(n, 50).contiguous(), u, _f([0.8] * n), _i([12] * n), _f([0.9] * n)).cpu()
    stay, w = decode_ref.kept(x[0].double().numpy(), np.float32(0.8), 12, 0.9)
    for i, v in zip(stay, w):
        assert abs(int((tokens == i).sum()) - n * v / sum(w)) <= 1.01
    assert set(tokens.tolist()) <= set(stay)


def test_outputs_streams_and_graphs(s):
    """Tokens into the caller's tensor without probabilities; a captured draw replayed on new logits and numbers."""
    rows, vocab = 5, 20000
    xs = [_logits(rows, vocab, seed=i).cuda() for i in range(4)]
    us = [torch.rand(rows, generator=torch.Generator().manual_seed(i)).cuda() for i in range(4)]
    p, k = _f([0.9] * rows), _i([100] * rows)
    want = [s.sample(x, u, None, k, p).clone() for x, u in zip(xs, us)]
    x, u, out = xs[0].clone(), us[0].clone(), torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    space = torch.empty(s.workspace_bytes(rows, vocab), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.sample(x, u, None, k, p, out=out, workspace=space)
    for i in (0, 1, 2, 3, 1):
        x.copy_(xs[i])
        u.copy_(us[i])
        torch.cuda.synchronize()
        g.replay()
        assert torch.equal(out, want[i])
    with torch.cuda.stream(torch.cuda.Stream()):
        assert s.sample(x, u, None, k, p, out=out) is out and torch.equal(out, want[1])
