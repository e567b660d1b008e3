"""The paged KV cache without a GPU: the surface of include/zest/kv.h, the
refusals of every entry point before anything reaches the GPU, the layout that
the kernels and the plain forms share, and rope's frequency table."""
from __future__ import annotations

import ctypes
import math
import re

import kv_ref
import numpy as np
import pytest
import torch
from helpers import ROOT, load_pkg


@pytest.fixture(scope="module")
def kv(zest):
    from ggml_xdna_amd import kv as m
    return m


def test_library_exports_the_cache_s_entry_points():
    z = load_pkg()
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "zest" / "kv.h").read_text(), flags=re.S)
    names = set(re.findall(r"\bZEST_API\s+[\w\s\*]+?\b(\w+)\s*\(", text))
    assert {"zest_kv_append", "zest_kv_attn", "zest_kv_assign", "zest_kv_compact"} <= names
    assert all(hasattr(z.lib(), n) for n in names) and names <= set(z.SIGNATURES)


@pytest.mark.parametrize("page,d", [(16, 64), (32, 96), (64, 128), (256, 64)])
def test_page_layout_is_a_bijection(page, d):
    k, v = kv_ref.page_index(page, d)
    assert torch.equal(torch.cat([k.reshape(-1), v.reshape(-1)]).sort().values, torch.arange(2 * page * d))
    # what the matrix instruction reads: 8 values of a token, 8 tokens of a column
    assert torch.equal(k[3, 8:16], k[3, 8] + torch.arange(8))
    assert [int(v[t, 5]) - int(v[4, 5]) for t in (4, 5, 6, 7, 12, 13, 14, 15)] == list(range(8))


def test_rope_freqs(kv):
    f, mag = kv.rope_freqs(8, 1e4)
    assert np.allclose(f, [1e4 ** (-p / 4) for p in range(4)], rtol=1e-15) and mag == 1.0
    # linear scaling, and a factor for each pair
    f, mag = kv.rope_freqs(8, 1e4, freq_scale=0.25, attn_factor=2.0, ff=[1.0, 2.0, 4.0, 8.0])
    assert np.allclose(f, [0.25 * 1e4 ** (-p / 4) / 2 ** p for p in range(4)], rtol=1e-15) and mag == 2.0
    # YaRN: pairs below the first correction dim keep their frequency, from the second on it is interpolated, between
    # them it moves linearly, and the magnitude grows with the scale
    f, mag = kv.rope_freqs(32, 1e6, freq_scale=0.25, ext_factor=1.0, corr=(4.0, 12.0))
    plain = np.array([1e6 ** (-2 * p / 32) for p in range(16)])
    mix = np.clip((np.arange(16) - 4) / 8, 0, 1)
    assert np.allclose(f, plain * (1 - 0.75 * mix), rtol=1e-14)
    assert mag == np.float32(1 + 0.1 * math.log(4.0))
    with pytest.raises(load_pkg().ZestError, match="n_dims"):
        kv.rope_freqs(7, 1e4)
    with pytest.raises(load_pkg().ZestError, match="base"):
        kv.rope_freqs(8, -1.0)


def test_entry_points_refuse_bad_arguments_before_the_gpu(kv):
    """Each call breaks one rule of its contract: it must be refused with its code and a message naming the call (the
    pointers are host memory, so no call here may launch)."""
    z = load_pkg()
    lib = z.lib()
    raw = ctypes.create_string_buffer(1 << 20)
    base = (ctypes.addressof(raw) + 255) & ~255
    E_ARG, E_UNSUPPORTED = -1, -3

    def cache(pool=base, pages=4, type=30, kv_heads=2, head_dim=64, page_tokens=16):
        return kv._Cache(pool, pages, type, kv_heads, head_dim, page_tokens)

    def batch(tables=base, lens=base, starts=base, slots=None, rows=4, seqs=2, table_rows=2, table_cols=2, max_new=4, max_len=32):
        return kv._Batch(tables, lens, starts, slots, rows, seqs, table_rows, table_cols, max_new, max_len)

    bad_caches = [(dict(pool=None), E_ARG), (dict(pool=base + 8), E_ARG), (dict(pages=0), E_ARG), (dict(pages=(1 << 24) + 1), E_ARG),
                  (dict(type=0), E_UNSUPPORTED), (dict(type=8), E_UNSUPPORTED), (dict(kv_heads=0), E_ARG), (dict(kv_heads=1025), E_ARG),
                  (dict(head_dim=80), E_UNSUPPORTED), (dict(head_dim=512), E_UNSUPPORTED), (dict(page_tokens=8), E_UNSUPPORTED),
                  (dict(page_tokens=48), E_UNSUPPORTED), (dict(page_tokens=512), E_UNSUPPORTED)]
    bad_batches = [(dict(tables=None), E_ARG), (dict(lens=None), E_ARG), (dict(starts=None), E_ARG), (dict(rows=0), E_ARG), (dict(rows=(1 << 27) + 1), E_ARG),
                   (dict(seqs=0), E_ARG), (dict(seqs=4097, slots=base), E_ARG), (dict(seqs=3), E_ARG), (dict(table_cols=0), E_ARG),
                   (dict(table_cols=1 << 27), E_ARG), (dict(max_new=0), E_ARG), (dict(max_new=5), E_ARG), (dict(max_len=-1), E_ARG), (dict(max_len=(1 << 30) + 1), E_ARG)]

    def append(c=None, b=None, rope=None, in_type=0, k=base, ldk=128, v=base, ldv=128, q=None, ldq=256, heads=4, q_out=None,
               ldo=256, to=0):
        return lib.zest_kv_append(ctypes.byref(c or cache()), ctypes.byref(b or batch()), ctypes.byref(rope) if rope else None, None,
                                  in_type, k, ldk, v, ldv, q, ldq, heads, q_out, ldo, to, None, None)

    def attn(c=None, b=None, q=base, qt=0, ldq=256, heads=4, scale=0.1, window=0, cap=0.0, out=base + 65536, ot=0, ldo=256,
             ws=base, size=1 << 30):
        return lib.zest_kv_attn(ctypes.byref(c or cache()), ctypes.byref(b or batch()), q, qt, ldq, heads, scale, 1, window, cap, out,
                                ot, ldo, ws, size, None, None)

    def assign(c=None, layers=1, stride=0, refs=base, tables=base, lens=base, rows=2, cols=2, dst=base, src=base, grow=base, n=2,
               scratch=base, size=1 << 20):
        return lib.zest_kv_assign(ctypes.byref(c or cache()), layers, stride, refs, tables, lens, rows, cols, dst, src, grow, n,
                                  scratch, size, None, None)

    def compact(c=None, layers=1, stride=0, refs=base, tables=base, rows=2, cols=2, ro=base, to=base, live=base, scratch=base,
                size=1 << 20):
        return lib.zest_kv_compact(ctypes.byref(c or cache()), layers, stride, refs, tables, rows, cols, ro, to, live, scratch, size,
                                   None, None)

    def refused(name, got, want):
        msg = lib.zest_last_error().decode()
        assert got == want and msg.startswith(name), (name, got, want, msg)

    for call, name in ((append, "zest_kv_append"), (attn, "zest_kv_attn"), (assign, "zest_kv_assign"), (compact, "zest_kv_compact")):
        for broken, code in bad_caches:
            refused(name, call(c=cache(**broken)), code)
        if call in (append, attn):
            for broken, code in bad_batches:
                refused(name, call(b=batch(**broken)), code)
    rope = lambda f=base, n=64, mode=2: kv._Rope(f, n, mode, 1.0)  # noqa: E731
    for broken, code in [(dict(k=None), E_ARG), (dict(v=None), E_ARG), (dict(in_type=8), E_UNSUPPORTED), (dict(ldk=124), E_ARG),
                         (dict(ldv=130), E_ARG), (dict(k=base + 4), E_ARG), (dict(rope=rope(f=None)), E_ARG),
                         (dict(rope=rope(f=base + 4)), E_ARG), (dict(rope=rope(n=63)), E_ARG), (dict(rope=rope(n=66)), E_ARG),
                         (dict(rope=rope(mode=1)), E_ARG), (dict(q=base, q_out=None), E_ARG), (dict(q=base, q_out=base, heads=0), E_ARG),
                         (dict(q=base, q_out=base, to=2), E_UNSUPPORTED), (dict(q=base, q_out=base + 8192, ldq=255), E_ARG),
                         (dict(q=base, q_out=base, to=30), E_ARG), (dict(q=base, q_out=base + 1024), E_ARG)]:
        refused("zest_kv_append", append(**broken), code)
    need = lib.zest_kv_attn_workspace(ctypes.byref(cache()), ctypes.byref(batch()), 4)
    assert need > 0
    for broken, code in [(dict(q=None), E_ARG), (dict(out=None), E_ARG), (dict(qt=2), E_UNSUPPORTED), (dict(ot=8), E_UNSUPPORTED),
                         (dict(ldq=252), E_ARG), (dict(ldo=258), E_ARG), (dict(q=base + 8), E_ARG), (dict(heads=3), E_ARG),
                         (dict(heads=0), E_ARG), (dict(heads=8192, ldq=1 << 20, ldo=1 << 20), E_ARG), (dict(scale=math.nan), E_ARG),
                         (dict(scale=math.inf), E_ARG), (dict(window=-1), E_ARG), (dict(cap=-1.0), E_ARG), (dict(cap=math.nan), E_ARG),
                         (dict(out=base), E_ARG), (dict(q=base + 65536, out=base + 65536), E_ARG), (dict(q=base + 65536 - 2048), E_ARG),
                         (dict(q=base + 65536, ldq=512, out=base + 65536 + 512, ldo=512), E_ARG), (dict(out=base + 32768 - 16), E_ARG),
                         (dict(c=cache(type=30, kv_heads=1), b=batch(rows=(1 << 27) - 16, max_new=1 << 20), heads=16, q=base + (1 << 42),
                               ldq=1024, out=base + (1 << 45), ldo=1024), E_ARG),
                         (dict(ws=None), E_ARG), (dict(ws=base + 8), E_ARG), (dict(size=need - 1), E_ARG)]:
        refused("zest_kv_attn", attn(**broken), code)
    # columns of one wider buffer: past that check, refused for the workspace
    attn(q=base + 65536, ldq=512, out=base + 65536 + 1024, ldo=512, ws=None)
    assert "workspace" in lib.zest_last_error().decode()
    attn(q=base + 65536 + 1024, ldq=512, out=base + 65536, ldo=512, ws=None)
    assert "workspace" in lib.zest_last_error().decode()
    need = lib.zest_kv_scratch_bytes(4, 2)
    for broken, code in [(dict(layers=0), E_ARG), (dict(layers=2, stride=8192), E_ARG), (dict(layers=2, stride=32776), E_ARG),
                         (dict(refs=None), E_ARG), (dict(tables=None), E_ARG), (dict(rows=0), E_ARG), (dict(rows=65537), E_ARG),
                         (dict(cols=0), E_ARG), (dict(scratch=None), E_ARG), (dict(scratch=base + 4), E_ARG), (dict(size=8), E_ARG)]:
        refused("zest_kv_assign", assign(**broken), code)
        refused("zest_kv_compact", compact(**broken), code)
    for broken, code in [(dict(lens=None), E_ARG), (dict(dst=None), E_ARG), (dict(src=None), E_ARG), (dict(grow=None), E_ARG),
                         (dict(n=0), E_ARG), (dict(n=65537), E_ARG), (dict(size=need - 1), E_ARG)]:
        refused("zest_kv_assign", assign(**broken), code)
    for broken, code in [(dict(ro=None), E_ARG), (dict(to=None), E_ARG), (dict(live=None), E_ARG)]:
        refused("zest_kv_compact", compact(**broken), code)


def test_append_refuses_an_output_that_overlaps_its_inputs(kv):
    """q, k and v of a call are read and q_out and the pages written in no order: a q_out over k, v or the pool, or over
    q without being q, is refused; columns of one wider buffer are not (no call here may launch: a rope without
    frequencies is refused after the overlaps)."""
    z = load_pkg()
    lib = z.lib()
    raw = ctypes.create_string_buffer(1 << 20)
    base = (ctypes.addressof(raw) + 255) & ~255
    pool = base + (1 << 19)  # 4 pages of 2 heads, 16 tokens of 64 values: 32 KB
    cache = kv._Cache(pool, 4, kv.TYPE_BF16, 2, 64, 16)
    batch = kv._Batch(base, base, base, None, 4, 2, 2, 2, 4, 32)
    none = kv._Rope(None, 64, 2, 1.0)
    ld = 1024  # fp32 values: q's 4 heads are 256 of a row, k's and v's 2 heads 128 each

    def said(q_out, ldo=ld, to=0, q=0, k=256 * 4, v=384 * 4):
        code = lib.zest_kv_append(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(none), None, 0, base + k, ld, base + v, ld,
                                  base + q, ld, 4, q_out, ldo, to, None, None)
        assert code == -1
        return lib.zest_last_error().decode()

    for fine in (said(base), said(base + 512 * 4), said(base + 768 * 4), said(base + 65536), said(pool + 32768), said(pool - 4 * ld * 4),
                 said(base + 65536, 256, kv.TYPE_BF16), said(pool + 32768, 256, kv.TYPE_F16), said(base, q=512 * 4)):
        assert "freqs" in fine
    for q_out, more, what in [(base + 256 * 4, {}, "k or v"), (base + 384 * 4, {}, "k or v"), (base + 496 * 4, {}, "k or v"),
                              (base + 240 * 4, {}, "q_out overlaps q"), (base, dict(q=512 * 4, k=0), "k or v"),
                              (base, dict(q=512 * 4, v=128 * 4), "k or v"), (base + 16, {}, "q_out overlaps q"),
                              (base + 512 * 4, dict(ldo=512), "overlaps"), (base + 1024, dict(to=30, ldo=256), "overlaps"),
                              (pool, {}, "the pool"), (pool + 32768 - 16, {}, "the pool"), (pool - 4 * ld * 4 + 3 * ld * 4, {}, "the pool"),
                              (pool - 16, dict(to=1, ldo=256), "the pool")]:
        assert what in said(q_out, **more), (q_out - base, more)


def test_attention_refuses_a_softcap_too_small_for_its_scale(kv):
    """Where their quotient passes 32 bits, a score of 0 would become NaN. (No call here may launch: the workspace is missing.)"""
    z = load_pkg()
    lib = z.lib()
    raw = ctypes.create_string_buffer(1 << 20)
    base = (ctypes.addressof(raw) + 255) & ~255
    cache, batch = kv._Cache(base, 4, kv.TYPE_BF16, 2, 64, 16), kv._Batch(base, base, base, None, 4, 2, 2, 2, 4, 32)

    def said(scale, cap):
        code = lib.zest_kv_attn(ctypes.byref(cache), ctypes.byref(batch), base + 65536, 0, 256, 4, scale, 1, 0, cap, base + 131072, 0, 256,
                                None, 0, None, None)
        assert code == -1
        return lib.zest_last_error().decode()

    for scale, cap in [(0.125, 1e-39), (-0.125, 1e-39), (1e20, 1e-20), (0.0, 1e-39)]:
        assert "softcap" in said(scale, cap)
    for scale, cap in [(0.125, 1e-38), (-0.125, 3e38), (0.0, 1e-37), (1e20, 0.0)]:
        assert "workspace" in said(scale, cap)


def test_package_refuses_tensors_that_do_not_fit(kv):
    z = load_pkg()
    pool = torch.zeros((2, 3, 1, 2 * 16 * 64), dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32)
    tables, lens, refs = torch.zeros((2, 2), **i32), torch.zeros(2, **i32), torch.zeros(3, **i32)
    cache = kv.Cache(pool, tables, lens, refs, 16, 64)
    for broken in [(pool.float(), tables, lens, refs), (pool[:, :, :, ::2], tables, lens, refs), (pool, tables.long(), lens, refs),
                   (pool, tables.T, lens, refs[:2]), (pool, tables, lens[:1], refs), (pool, tables, lens, refs[:2])]:
        with pytest.raises(z.ZestError):
            kv.Cache(*broken, 16, 64)
    with pytest.raises(z.ZestError, match="starts"):
        kv.Batch(torch.zeros(1, **i32), 1, 1, 1)
    with pytest.raises(z.ZestError, match="slots"):
        kv.Batch(torch.zeros(3, **i32), 1, 1, 1, slots=torch.zeros(1, **i32))
    batch = kv.Batch(torch.zeros(3, **i32), 2, 1, 1)
    x = torch.zeros((2, 1, 64))
    for call in (lambda: kv.attention(cache, 0, batch, x), lambda: kv.append(cache, 0, batch, x, x),
                 lambda: kv.assign(cache, lens, lens, lens), lambda: kv.compact(cache)):
        with pytest.raises(z.ZestError, match="not the current device"):
            call()


def test_a_cache_s_flag(kv):
    z = load_pkg()
    cache = kv.empty_cache(1, 3, 1, 64, 16, slots=2, device="cpu")
    cache.check()
    cache.bad[0] = 1
    with pytest.raises(z.ZestError, match="left out"):
        cache.check()
    cache.check()
    with pytest.raises(AttributeError):  # calls hold its address
        cache.bad = torch.zeros(1, dtype=torch.int32)


def test_bounds_that_32_bits_would_cut(kv):
    z = load_pkg()
    starts = torch.zeros(3, dtype=torch.int32)
    for max_new, max_len in [((1 << 32) + 1, 8), (1, (1 << 32) + 8), (-1, 8), (1, -1)]:
        with pytest.raises(z.ZestError, match="31 bits"):
            kv.Batch(starts, 2, max_new, max_len)
    assert kv.Batch(starts, 2, 1, 1 << 30).max_len == 1 << 30
