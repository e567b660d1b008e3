"""A decoding step's kernels without a GPU: the surface of include/zest/decode.h and of the shared attention, and the
refusals of every entry point before anything reaches the GPU."""
from __future__ import annotations

import ctypes
import re

import decode_ref
import numpy as np
import pytest
import torch
from helpers import ROOT, load_pkg

E_ARG, E_UNSUPPORTED = -1, -3


def _lib():
    return load_pkg().lib()


def _base():
    raw = ctypes.create_string_buffer(1 << 21)
    _base.keep = raw
    return (ctypes.addressof(raw) + 255) & ~255


def _refused(name, got, want):
    msg = _lib().zest_last_error().decode()
    assert got == want and msg.startswith(name), (name, got, want, msg)


def test_library_exports_the_entry_points():
    z = load_pkg()
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "zest" / "decode.h").read_text(), flags=re.S)
    names = set(re.findall(r"\bZEST_API\s+[\w\s\*]+?\b(\w+)\s*\(", text))
    assert {"zest_matvec", "zest_matvec_glu", "zest_sample"} <= names
    assert all(hasattr(z.lib(), n) for n in names) and names <= set(z.SIGNATURES)


@pytest.mark.parametrize("wtype", sorted(decode_ref.BLOCKS))
def test_weights_stand_for_what_the_oracle_says(oracle, wtype):
    k = 512
    raw = decode_ref.gguf(wtype, 5, k)
    a, b = decode_ref.parts(wtype, raw, k)
    want = oracle.dequant(wtype, raw, 5, k)
    assert np.allclose(a + b, want, rtol=2e-7, atol=1e-9)


def test_matvec_refuses():
    lib, base = _lib(), _base()
    x, w, y, r = base, base + (1 << 18), base + (1 << 19), base + (3 << 18)
    P, I = lambda *v: (ctypes.c_void_p * len(v))(*v), lambda *v: (ctypes.c_int64 * len(v))(*v)  # noqa: E731,E741

    def call(type=2, x=x, m=2, k=64, ldx=64, w=(w,), n=(8,), res=None, ldr=None, y=(y,), ldy=(8,), ws=base + (1 << 20), size=1 << 20, count=None):
        return lib.zest_matvec(type, x, m, k, ldx, len(w) if count is None else count, P(*w), I(*n), P(*res) if res else None,
                               I(*ldr) if ldr else None, P(*y), I(*ldy), ws, size, None)

    for broken, code in [(dict(type=0), E_UNSUPPORTED), (dict(type=13), E_UNSUPPORTED), (dict(type=-1), E_UNSUPPORTED), (dict(m=0), E_ARG), (dict(m=17), E_ARG), (dict(m=-1), E_ARG),
                         (dict(k=0), E_ARG), (dict(k=48), E_ARG), (dict(type=12, k=128), E_ARG), (dict(k=(1 << 20) + 32), E_ARG), (dict(x=None), E_ARG),
                         (dict(x=x + 4), E_ARG), (dict(ldx=60), E_ARG), (dict(ldx=66), E_ARG), (dict(ldx=1 << 31), E_ARG), (dict(w=(None,)), E_ARG), (dict(w=(w + 1,)), E_ARG),
                         (dict(type=3, w=(w + 2,)), E_ARG), (dict(type=23, k=256, ldx=256, w=(w + 4,)), E_ARG), (dict(type=12, k=256, ldx=256, w=(w + 8,)), E_ARG),
                         (dict(n=(0,)), E_ARG), (dict(n=((1 << 26) + 1,)), E_ARG), (dict(y=(None,)), E_ARG), (dict(y=(y + 2,)), E_ARG), (dict(ldy=(7,)), E_ARG),
                         (dict(count=0), E_ARG), (dict(w=(w,) * 5, n=(8,) * 5, y=tuple(y + 4096 * i for i in range(5)), ldy=(8,) * 5), E_ARG),
                         (dict(res=(r + 2,), ldr=(8,)), E_ARG), (dict(res=(r,), ldr=(7,)), E_ARG), (dict(res=(r,)), E_ARG),
                         (dict(m=9, ws=None), E_ARG), (dict(m=9, ws=base + (1 << 20) + 4), E_ARG), (dict(m=9, size=9 * 2 * 112 - 1), E_ARG)]:
        _refused("zest_matvec", call(**broken), code)
    # overlaps: of an output with x, a weight, another output, a residual that it is not
    two = dict(w=(w, w), n=(8, 8), ldy=(8, 8))
    for broken in (dict(y=(x,)), dict(y=(x + 60 * 4,)), dict(y=(w + 16,)), dict(y=(y, y + 4), **two), dict(y=(y, y), **two),
                   dict(res=(y + 4,), ldr=(8,)), dict(res=(y,), ldr=(9,)), dict(res=(None, y), ldr=(0, 8), y=(y, y + 4096), **two)):
        _refused("zest_matvec", call(**broken), E_ARG)
        assert "overlap" in lib.zest_last_error().decode(), broken
    # columns of one buffer, a residual in place: past that check, refused for the workspace
    wide = dict(w=(w, w), n=(8, 8), ldy=(16, 16), y=(y, y + 32))
    for fine in (dict(m=9, **wide), dict(m=9, res=(y,), ldr=(8,)), dict(m=9, res=(y + 32, y), ldr=(16, 16), **dict(wide, y=(y + 32, y)))):
        _refused("zest_matvec", call(ws=None, **fine), E_ARG)
        assert "workspace" in lib.zest_last_error().decode(), fine


def test_matvec_workspace_goes_by_sizes():
    lib = _lib()
    ws = lambda t, m, k, *n: lib.zest_matvec_workspace(t, m, k, len(n), (ctypes.c_int64 * len(n))(*n))  # noqa: E731
    assert ws(12, 1, 2560, 4096) == 0 and ws(12, 9, 2560, 4096) == 80 * 1664
    assert ws(12, 4, 5120, 17408, 17408) == 160 * 4 * 112  # as a GLU's
    assert [ws(0, 1, 256, 8), ws(12, 1, 128, 8), ws(12, 0, 256, 8), ws(12, 17, 256, 8), ws(12, 9, 256, 0), ws(12, 9, 256)] == [0] * 6


def test_matvec_glu_refuses():
    lib, base = _lib(), _base()
    w, y = base + (1 << 18), base + (1 << 19)

    def call(kind=2, type=2, x=base, m=2, k=64, ldx=64, gate=w, up=w + 4096, f=8, y=y, ldy=8, ws=base + (1 << 20), size=1 << 20):
        return lib.zest_matvec_glu(kind, type, x, m, k, ldx, gate, up, f, y, ldy, ws, size, None)

    for broken, code in [(dict(kind=5), E_UNSUPPORTED), (dict(kind=-1), E_UNSUPPORTED), (dict(type=1), E_UNSUPPORTED), (dict(m=0), E_ARG), (dict(m=17), E_ARG),
                         (dict(k=33), E_ARG), (dict(x=None), E_ARG), (dict(gate=None), E_ARG), (dict(up=None), E_ARG), (dict(up=w + 1), E_ARG), (dict(f=0), E_ARG),
                         (dict(y=None), E_ARG), (dict(ldy=4), E_ARG), (dict(y=base), E_ARG), (dict(y=w + 4096), E_ARG), (dict(m=16, ws=None), E_ARG), (dict(m=16, size=1), E_ARG)]:
        _refused("zest_matvec_glu", call(**broken), code)


def test_sample_refuses():
    lib, base = _lib(), _base()

    def call(logits=base, type=0, rows=2, vocab=20000, ld=20000, u=base, t=None, k=None, p=None, m=None, token=base, prob=None, ws=base + (1 << 20), size=1 << 20):
        return lib.zest_sample(logits, type, rows, vocab, ld, u, t, k, p, m, token, prob, ws, size, None)

    for broken, code in [(dict(type=2), E_UNSUPPORTED), (dict(type=8), E_UNSUPPORTED), (dict(logits=None), E_ARG), (dict(u=None), E_ARG), (dict(token=None), E_ARG),
                         (dict(rows=0), E_ARG), (dict(rows=65537), E_ARG), (dict(vocab=0), E_ARG), (dict(vocab=(1 << 18) + 1, ld=1 << 19), E_ARG), (dict(ld=19999), E_ARG),
                         (dict(ld=1 << 31), E_ARG), (dict(logits=base + 2), E_ARG), (dict(type=1, logits=base + 1), E_ARG), (dict(u=base + 2), E_ARG), (dict(t=base + 1), E_ARG),
                         (dict(k=base + 2), E_ARG), (dict(p=base + 3), E_ARG), (dict(m=base + 2), E_ARG), (dict(token=base + 2), E_ARG), (dict(prob=base + 2), E_ARG),
                         (dict(ws=None), E_ARG), (dict(ws=base + 8), E_ARG), (dict(size=8), E_ARG)]:
        _refused("zest_sample", call(**broken), code)
    assert lib.zest_sample_workspace(0, 5) == 0 and lib.zest_sample_workspace(1, 1 << 19) == 0 and lib.zest_sample_workspace(3, 1000) == 0
    assert 0 < lib.zest_sample_workspace(1, 20000) < lib.zest_sample_workspace(256, 20000) == lib.zest_sample_workspace(65536, 20000)


def test_shared_attention_refuses():
    z = load_pkg()
    from ggml_xdna_amd import kv
    lib, base = _lib(), _base()
    cache = kv._Cache(base, 4, 30, 2, 64, 16)
    batch = lambda **m: kv._Batch(*[dict(dict(tables=base, lens=base, starts=base, slots=None, rows=4, seqs=2, table_rows=2, table_cols=2, max_new=4, max_len=32), **m)[f]  # noqa: E731
                                    for f, _ in kv._Batch._fields_])

    def call(g=(base, 1, 32), b=None, heads=4, q=base, out=base + 65536, ws=base, size=1 << 20, c=cache):
        groups = ctypes.byref(kv._Groups(*g)) if g else None
        return lib.zest_kv_attn_shared(ctypes.byref(c), ctypes.byref(b or batch()), groups, q, 0, 256, heads, 0.1, 1, 0, 0.0, out, 0, 256, ws, size, None, None)

    need = lib.zest_kv_attn_shared_workspace(ctypes.byref(cache), ctypes.byref(batch()), ctypes.byref(kv._Groups(base, 1, 32)), 4)
    assert need > 0
    for broken in (dict(g=None), dict(g=(None, 1, 32)), dict(g=(base + 2, 1, 32)), dict(g=(base, 0, 32)), dict(g=(base, 2049, 32)), dict(g=(base, 1, -1)),
                   dict(g=(base, 1, (1 << 30) + 1)), dict(g=(base, 1, 32, 2)), dict(heads=3), dict(q=None), dict(out=base), dict(ws=None), dict(ws=base + 8), dict(size=need - 1),
                   dict(b=batch(max_new=0)), dict(b=batch(seqs=0)), dict(c=kv._Cache(base, 0, 30, 2, 64, 16))):
        _refused("zest_kv_attn", call(**broken), E_ARG)
    _refused("zest_kv_attn", call(c=kv._Cache(base, 4, 8, 2, 64, 16)), E_UNSUPPORTED)
    with pytest.raises(z.ZestError):
        kv.Groups(torch.zeros(1, dtype=torch.int32), 5)
    with pytest.raises(z.ZestError):
        kv.Groups(torch.zeros(2, dtype=torch.int64), 5)
    with pytest.raises(z.ZestError):
        kv.Groups(torch.zeros(2, dtype=torch.int32), -1)
    with pytest.raises(z.ZestError):
        kv.Groups(torch.zeros(2, dtype=torch.int32), 1 << 31)


def test_the_package_refuses(zest):
    """Tensors that are not on a GPU, not of the type or not of the sizes that the call says."""
    from ggml_xdna_amd import sampling
    x, w = torch.zeros((1, 64)), torch.zeros(8 * 36, dtype=torch.uint8)
    with pytest.raises(zest.ZestError, match="current device"):
        zest.matvec(2, x, [w], [8])
    with pytest.raises(zest.ZestError, match="current device"):
        zest.matvec_glu(2, 2, x, w, w, 8)
    with pytest.raises(zest.ZestError, match="current device"):
        sampling.sample(torch.zeros((1, 10)), torch.zeros(1))
