"""The decoding runner: matvec, append, attention by groups, matvec_glu, the logits and the choice of the next token, one
after the other as they are used, each call against its 64-bit form on what the call was given."""
from __future__ import annotations

import decode_ref
import kv_ref
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def st(zest_gpu):
    from ggml_xdna_amd import stack
    return stack


def _config(st, types=(12, 8, 12, 8), layers=2):
    return st.StackConfig("tiny", layers, 256, 256, 128, 512, *types, 0, 0, head_dim=64, rope_base=1e4)


def _start(st, cfg, answers, prompt, seed=1, page=16, vocab=700):
    d = st.Decode(cfg, vocab, answers, 160, seed=seed, page=page)
    d.groups = type(d.groups)(d.groups.starts, 160, always=True)  # (so few tokens would be read one by one)
    d.prompt(torch.randint(0, vocab, (prompt,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda())
    d.temperature.fill_(0.9)
    d.top_k.fill_(50)
    d.top_p.fill_(0.95)
    d.min_p.fill_(0.02)
    return d


@pytest.mark.parametrize("answers,prompt,types", [(1, 1, (12, 8, 12, 8)), (3, 40, (8, 12, 8, 12)), (6, 75, (12, 8, 12, 8)), (16, 33, (8, 8, 8, 8))])
def test_every_call_of_a_step(st, answers, prompt, types, monkeypatch):
    from ggml_xdna_amd import kv, sampling
    z, cfg = st.z, _config(st, types)
    d = _start(st, cfg, answers, prompt)
    calls = {"matvec": 0, "glu": 0, "attention": 0, "sample": 0}

    def close(got, want, bound):
        assert bool((np.abs(got.double().cpu().numpy() - want) <= bound).all())

    def matvec(wtype, x, weights, ns, outs=None, residuals=None):
        before = None if residuals is None else residuals[0].clone()
        got = matvec_(wtype, x, weights, ns, outs=outs, residuals=residuals)
        for w, n, y in zip(weights, ns, got):
            want, bound = decode_ref.matvec(wtype, x.cpu().numpy(), w.cpu().numpy().reshape(n, -1))
            if before is not None:  # one rounding of the sum
                want = want + before.double().cpu().numpy()
                bound = bound + 2.0 ** -24 * (np.abs(want) + bound)
            close(y, want, bound)
        calls["matvec"] += 1
        return got

    def matvec_glu(kind, wtype, x, gate, up, f):
        got = matvec_glu_(kind, wtype, x, gate, up, f)
        (g, eg), (u, eu) = (decode_ref.matvec(wtype, x.cpu().numpy(), w.cpu().numpy().reshape(f, -1)) for w in (gate, up))
        close(got, decode_ref.glu(kind, g, u), decode_ref.glu_bound(g, eg, u, eu))
        calls["glu"] += 1
        return got

    def attention(cache, layer, batch, q, out_dtype=None, groups=None):
        got = attention_(cache, layer, batch, q, out_dtype=out_dtype, groups=groups)
        pool, tables, lens = cache.pool.cpu(), cache.tables.cpu(), cache.lens.cpu()
        for i in range(answers):
            held = kv_ref.read_cache(pool, tables[i], int(lens[i]), 16, 64, layer)
            want, spread, reach = kv_ref.attention(q[i].cpu().view(1, 4, 64), *held, 0.125)
            # (joining a shared part and an own one rounds the factors of each once more)
            bound = kv_ref.attention_bound(want, spread, reach, 64, torch.bfloat16, torch.float32) + 2.0 ** -21 * (spread + want.abs())
            assert bool(((got[i].cpu().view(1, 4, 64).double() - want).abs() <= bound).all())
        assert len(set(tables[:, 0].tolist())) == (1 if prompt > 16 else answers)  # the prompt's pages are the answers' own
        calls["attention"] += 1
        return got

    def sample(logits, u, t, k, p, m, probs=None, out=None):
        sample_(logits, u, t, k, p, m, probs=probs, out=out)
        rows = logits.double().cpu().numpy()
        for r in range(answers):
            stay, w = decode_ref.kept(rows[r], np.float32(t[r].item()), int(k[r]), float(p[r]), float(m[r]))
            assert decode_ref.fits(int(out[r]), float(probs[r]), stay, w, float(u[r]))
        calls["sample"] += 1

    matvec_, matvec_glu_, attention_, sample_ = z.matvec, z.matvec_glu, kv.attention, sampling.sample
    monkeypatch.setattr(z, "matvec", matvec)
    monkeypatch.setattr(z, "matvec_glu", matvec_glu)
    monkeypatch.setattr(kv, "attention", attention)
    monkeypatch.setattr(sampling, "sample", sample)
    g = torch.Generator(device="cuda").manual_seed(answers)
    for _ in range(3):
        d.u.uniform_(generator=g)
        tokens = d.step()
        assert int(tokens.min()) >= 0 and int(tokens.max()) < d.vocab
    assert calls == {"matvec": 3 * (2 * 3 + 1), "glu": 3 * 2, "attention": 3 * 2, "sample": 3}
    assert d.cache.lens.tolist() == [prompt - 1 + 3] * answers
    d.cache.check()


def test_a_captured_step_is_the_eager_one(st):
    """Steps replayed from one graph, with eager work between them, against the same steps of another runner."""
    cfg = _config(st)
    a, b = (_start(st, cfg, 5, 50) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(3)
    us = torch.rand((30, 5), generator=g, device="cuda")
    eager = []
    for i in range(30):
        b.u.copy_(us[i])
        eager.append((b.step().clone(), b.probs.clone()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for i in range(30):
        a.u.copy_(us[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a.tokens, eager[i][0]) and torch.equal(a.probs, eager[i][1]), i
        us.sum().item()
    assert len({tuple(t.tolist()) for t, _ in eager}) > 20 and torch.equal(a.cache.lens, b.cache.lens)
    a.prompt(torch.arange(20, dtype=torch.int32, device="cuda"))  # another prompt, by the same graph
    b.prompt(torch.arange(20, dtype=torch.int32, device="cuda"))
    for i in range(4):
        for d in (a, b):
            d.u.copy_(us[i])
        graph.replay()
        want = b.step()
        torch.cuda.synchronize()
        assert torch.equal(a.tokens, want)
    a.cache.check()
    b.cache.check()


def test_a_runner_that_outgrows_its_cache_is_told(st):
    d = st.Decode(_config(st), 100, 2, 32, page=16)
    d.prompt(torch.zeros(31, dtype=torch.int32, device="cuda"))
    d.step()
    d.step()
    d.cache.check()
    d.step()
    with pytest.raises(st.z.ZestError, match="left out"):
        d.cache.check()
