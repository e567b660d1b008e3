"""The paged KV cache (include/zest/kv.h): append with rope, attention of new
tokens over their sequences' pages, the scheduler's step over the page tables,
compaction of the pool.

Like the package's other calls these go straight to the HIP kernels, on torch's
current stream, with device memory owned by torch tensors; a call that cannot
be made raises ZestError. Nothing waits for the GPU, so a decoding loop (append
and attention of every layer, assign) can be captured in a HIP graph; only
attention's default workspace and outputs are allocated, from torch's allocator.

What a call leaves out because of what the tables, lengths, starts or entries on
the device hold, it reports in the flag it is given, else in the cache's, which
Cache.check() looks at. Rows of an output that it does not write (those of a
sequence left out, and those of no sequence) hold what they held: in an output
that the call made, anything.
"""
from __future__ import annotations

import ctypes
import math

import torch

import ggml_xdna_amd as z

TYPE_F16, TYPE_BF16 = 1, 30
ROPE_NORMAL, ROPE_NEOX = 0, 2

_TYPES = {torch.float32: z.TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}


class _Cache(ctypes.Structure):
    _fields_ = [("pool", ctypes.c_void_p), ("pages", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("type", "kv_heads",
                                                                                                    "head_dim", "page_tokens")]


class _Batch(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("tables", "lens", "starts", "slots")] + [("rows", ctypes.c_int64)] +
                [(n, ctypes.c_int32) for n in ("seqs", "table_rows", "table_cols", "max_new", "max_len")])


class _Rope(ctypes.Structure):
    _fields_ = [("freqs", ctypes.c_void_p), ("n_dims", ctypes.c_int32), ("mode", ctypes.c_int32), ("magnitude", ctypes.c_float)]


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise z.ZestError(what)


def _list(t, what: str, device, dim: int = 1):
    if t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous() or t.device != device:
        raise z.ZestError(f"{what}: a contiguous int32 tensor of {dim} dimension(s) on {device} wanted")
    return t


def _here(device) -> None:
    if device.type != "cuda" or device.index != torch.cuda.current_device():
        raise z.ZestError(f"the cache is on {device}, which is not the current device")


def _rows(t, what: str, rows: int, heads: int | None, dim: int, device):
    """A tensor [rows][heads][dim] or [rows][heads * dim], rows any stride apart; returns (type, pointer, stride, heads)."""
    # (the messages are made only when needed: these checks are a good part of a small call's time)
    shape, kind = t.shape, _TYPES.get(t.dtype)
    if kind is None or len(shape) not in (2, 3) or shape[0] != rows or t.device != device:
        raise z.ZestError(f"{what}: float32, float16 or bfloat16 rows, {rows} of them, on {device} wanted")
    stride = t.stride()
    if len(shape) == 3:
        have = shape[1]
        ok = shape[2] == dim and stride[2] == 1 and (stride[1] == dim or have == 1)
    else:
        have = shape[1] // dim
        ok = shape[1] % dim == 0 and stride[1] == 1
    if not ok or have <= 0 or (heads is not None and heads != have):
        raise z.ZestError(f"{what}: rows of {heads or 'whole'} heads of {dim} contiguous values wanted")
    # a single row's stride is not used
    return kind, t.data_ptr(), stride[0] if rows > 1 else have * dim, have


class Cache:
    """A paged cache over tensors that the program owns: pool [layers][pages][kv_heads][2 * page_tokens * head_dim] of
    float16 or bfloat16, tables [slots][columns], lens [slots] and refs [pages] of int32 (zest/kv.h says what they
    hold). empty_cache makes one of no sequences."""

    def __init__(self, pool, tables, lens, refs, page_tokens: int, head_dim: int):
        dev = pool.device
        _need(pool.dim() == 4 and pool.dtype in (torch.float16, torch.bfloat16) and pool.is_contiguous() and
              pool.shape[3] == 2 * page_tokens * head_dim and pool.numel() > 0,
              "pool: a contiguous [layers][pages][kv_heads][2 * page_tokens * head_dim] of float16 or bfloat16 wanted")
        self.pool, self.tables, self.device = pool, _list(tables, "tables", dev, 2), dev
        self.lens, self.refs = _list(lens, "lens", dev), _list(refs, "refs", dev)
        self.layers, self.pages, self.kv_heads = pool.shape[:3]
        _need(lens.numel() == tables.shape[0] and refs.numel() == self.pages, "lens: one a slot, refs: one a page, wanted")
        self.page_tokens, self.head_dim = page_tokens, head_dim
        self.layer_stride = pool.stride(0) * 2
        self._layer = [_Cache(pool.data_ptr() + i * self.layer_stride, self.pages, _TYPES[pool.dtype], self.kv_heads, head_dim,
                              page_tokens) for i in range(self.layers)]
        # where calls that are given no flag of their own report what they leave out
        self._bad = torch.zeros(1, dtype=torch.int32, device=dev)
        self._bad_at = self._bad.data_ptr()
        # assign's and compact's working memory: their calls change the cache, so they never run at once
        self._scratch = torch.empty(z.lib().zest_kv_scratch_bytes(self.pages, tables.shape[0]), dtype=torch.uint8, device=dev)
        self._home = torch.cuda.current_stream(dev).cuda_stream if dev.type == "cuda" else None

    @property
    def bad(self) -> torch.Tensor:
        return self._bad

    def check(self) -> None:
        """Raises ZestError where calls without a flag of their own have left something out since the last check (a page
        outside the pool, a slot outside the tables, a length past the bounds, a pool that ran out). Waits for the current
        stream."""
        if int(self.bad):
            self.bad.zero_()
            raise z.ZestError("a call left out what its tables, lengths, starts or entries name outside the cache or the bounds given")

    def _stream(self) -> int:
        """The current stream's handle. The cache's own memory was allocated on the stream it was made on: on another one
        it is marked as used there, so that dropping the cache does not hand it back under the work queued there."""
        handle = z._stream()
        if handle != self._home:
            stream = torch.cuda.current_stream(self.device)
            self._bad.record_stream(stream)
            self._scratch.record_stream(stream)
        return handle

    def _batch(self, b: "Batch") -> _Batch:
        if b.starts.device != self.device:
            raise z.ZestError("the batch and the cache are on different devices")
        return _Batch(self.tables.data_ptr(), self.lens.data_ptr(), b.starts.data_ptr(),
                      None if b.slots is None else b.slots.data_ptr(), b.rows, b.seqs, self.tables.shape[0],
                      self.tables.shape[1], b.max_new, b.max_len)


def empty_cache(layers: int, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64, slots: int = 64,
                columns: int | None = None, dtype=torch.bfloat16, device="cuda") -> Cache:
    """A cache of `slots` empty sequences of at most `columns` pages (all of the pool unless given)."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    i32 = dict(dtype=torch.int32, device=device)
    return Cache(torch.zeros((layers, pages, kv_heads, 2 * page_tokens * head_dim), dtype=dtype, device=device),
                 torch.full((slots, columns or pages), -1, **i32), torch.zeros(slots, **i32), torch.zeros(pages, **i32),
                 page_tokens, head_dim)


class Batch:
    """The sequences of a call: starts [seqs + 1] (int32, device), the rows of q, k, v and the output, bounds on a
    sequence's new tokens and length, and its slots (int32, device; the first ones unless given)."""

    def __init__(self, starts, rows: int, max_new: int, max_len: int, slots=None):
        self.starts, self.slots = _list(starts, "starts", starts.device), slots
        self.seqs, self.rows, self.max_new, self.max_len = starts.numel() - 1, rows, max_new, max_len
        _need(self.seqs > 0, "starts: one more entry than sequences wanted")
        _need(all(0 <= x < 1 << 31 for x in (max_new, max_len)), f"max_new={max_new}, max_len={max_len}: 31 bits wanted")
        if slots is not None:
            _need(_list(slots, "slots", starts.device).numel() == self.seqs, "slots: one a sequence wanted")


class Rope:
    """Rotary positions: freqs (float64, device), one a pair; mode ROPE_NORMAL or ROPE_NEOX; a magnitude."""

    def __init__(self, freqs, mode: int = ROPE_NEOX, magnitude: float = 1.0):
        _need(freqs.dtype == torch.float64 and freqs.dim() == 1 and freqs.is_contiguous() and freqs.numel() > 0,
              "freqs: a contiguous float64 tensor of one frequency a pair wanted")
        self.freqs, self.mode, self.magnitude = freqs, mode, magnitude
        self._c = _Rope(freqs.data_ptr(), 2 * freqs.numel(), mode, magnitude)


def rope_freqs(n_dims: int, freq_base: float, freq_scale: float = 1.0, ext_factor: float = 0.0, attn_factor: float = 1.0,
               corr: tuple[float, float] = (0.0, 0.0), ff=None) -> tuple[list[float], float]:
    """The frequencies and the magnitude that zest_rope's parameters stand for (host arithmetic)."""
    out, mag = (ctypes.c_double * max(1, n_dims // 2))(), ctypes.c_float()
    f = (ctypes.c_float * len(ff))(*ff) if ff is not None else None
    _need(ff is None or len(ff) == n_dims // 2, "ff: one factor a pair wanted")
    z.check(z.lib().zest_kv_rope_freqs(n_dims, freq_base, freq_scale, ext_factor, attn_factor, corr[0], corr[1], f, out,
                                       ctypes.byref(mag)), "zest_kv_rope_freqs")
    return list(out), mag.value


def _bad(bad, cache: Cache) -> int:
    if bad is None:
        return cache._bad_at
    _need(bad.dtype in (torch.int32, torch.uint32) and bad.device == cache.device and bad.numel() > 0,
          f"bad: an int32 tensor on {cache.device} wanted")
    return bad.data_ptr()


def append(cache: Cache, layer: int, batch: Batch, k, v, q=None, rope: Rope | None = None, pos=None, q_out=None, q_dtype=None,
           bad=None):
    """zest_kv_append: the batch's new k (turned by rope) and v into layer's pages. With q, its turned rows are returned
    (of q_dtype, the cache's type unless given; or in q_out)."""
    dev = cache.device
    _here(dev)
    if not 0 <= layer < cache.layers:
        raise z.ZestError(f"layer {layer} of {cache.layers}")
    d = cache.head_dim
    tk, pk, ldk, _ = _rows(k, "k", batch.rows, cache.kv_heads, d, dev)
    tv, pv, ldv, _ = _rows(v, "v", batch.rows, cache.kv_heads, d, dev)
    if tk != tv:
        raise z.ZestError("k and v of one type wanted")
    qa, oa, heads = (None, 0), (0, None, 0), 0
    if q is None:
        _need(q_out is None, "q_out: rows of q wanted with it")
    else:
        tq, pq, ldq, heads = _rows(q, "q", batch.rows, None, d, dev)
        if tq != tk:
            raise z.ZestError("q, k and v of one type wanted")
        if q_out is None:
            q_out = torch.empty_like(q, dtype=q_dtype or cache.pool.dtype, memory_format=torch.contiguous_format)
        elif q_dtype is not None and q_out.dtype != q_dtype:
            raise z.ZestError(f"q_out of {q_out.dtype}, q_dtype {q_dtype}")
        to, po, ldo, _ = _rows(q_out, "q_out", batch.rows, heads, d, dev)
        qa, oa = (pq, ldq), (to, po, ldo)
    if pos is not None:
        _need(_list(pos, "pos", dev).numel() == batch.rows, "pos: one a row wanted")
    if rope is not None and rope.freqs.device != dev:
        raise z.ZestError("the rope and the cache are on different devices")
    z.check(z.lib().zest_kv_append(ctypes.byref(cache._layer[layer]), ctypes.byref(cache._batch(batch)),
                                   ctypes.byref(rope._c) if rope is not None else None, z._ptr(pos), tk, pk, ldk, pv, ldv, *qa,
                                   heads, oa[1], oa[2], oa[0], _bad(bad, cache), cache._stream()), "zest_kv_append")
    return q_out


def attention_workspace(cache: Cache, batch: Batch, q_heads: int) -> int:
    """Bytes of attention's workspace, by the batch's sizes and bounds alone."""
    return z.lib().zest_kv_attn_workspace(ctypes.byref(cache._layer[0]), ctypes.byref(cache._batch(batch)), q_heads)


def attention(cache: Cache, layer: int, batch: Batch, q, scale: float | None = None, causal: bool = True, window: int = 0,
              softcap: float = 0.0, out=None, out_dtype=None, workspace=None, bad=None):
    """zest_kv_attn: attention of the batch's new tokens over layer's pages; returns out (of q's type and shape unless
    given). scale: 1 / sqrt(head_dim) unless given."""
    dev = cache.device
    _here(dev)
    if not 0 <= layer < cache.layers:
        raise z.ZestError(f"layer {layer} of {cache.layers}")
    if not 0 <= window < 1 << 31:  # ctypes would cut it to 32 bits
        raise z.ZestError(f"window={window}")
    d = cache.head_dim
    tq, pq, ldq, heads = _rows(q, "q", batch.rows, None, d, dev)
    if out is None:
        out = torch.empty_like(q, dtype=out_dtype, memory_format=torch.contiguous_format)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise z.ZestError(f"out of {out.dtype}, out_dtype {out_dtype}")
    to, po, ldo, _ = _rows(out, "out", batch.rows, heads, d, dev)
    lib = z.lib()
    c, b = ctypes.byref(cache._layer[layer]), ctypes.byref(cache._batch(batch))
    if workspace is None:
        workspace = torch.empty(lib.zest_kv_attn_workspace(c, b, heads), dtype=torch.uint8, device=dev)
    elif workspace.device != dev or not workspace.is_contiguous():
        raise z.ZestError(f"workspace: a contiguous tensor on {dev} wanted")
    z.check(lib.zest_kv_attn(c, b, pq, tq, ldq, heads, 1.0 / math.sqrt(d) if scale is None else scale, int(causal), window,
                                 softcap, po, to, ldo, workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                                 _bad(bad, cache), cache._stream()), "zest_kv_attn")
    return out


def assign(cache: Cache, dst, src, grow, bad=None) -> None:
    """zest_kv_assign: slot dst[i] becomes what src[i] was (-1: empty), grown by grow[i] tokens; int32 device tensors, at
    most one entry a slot."""
    dev = cache.device
    _here(dev)
    n = _list(dst, "dst", dev).numel()
    _need(_list(src, "src", dev).numel() == n and _list(grow, "grow", dev).numel() == n, "dst, src and grow of one length wanted")
    if n > cache.tables.shape[0]:
        raise z.ZestError(f"{n} entries for {cache.tables.shape[0]} slots")
    z.check(z.lib().zest_kv_assign(ctypes.byref(cache._layer[0]), cache.layers, cache.layer_stride, cache.refs.data_ptr(),
                                   cache.tables.data_ptr(), cache.lens.data_ptr(), cache.tables.shape[0], cache.tables.shape[1],
                                   dst.data_ptr(), src.data_ptr(), grow.data_ptr(), n, cache._scratch.data_ptr(),
                                   cache._scratch.numel(), _bad(bad, cache), cache._stream()), "zest_kv_assign")


def compact(cache: Cache, refs=None, tables=None, live=None, bad=None):
    """zest_kv_compact: the live pages moved to the front of the pool; returns their number (int32 [1], device). refs and
    tables: buffers for the new ones, the cache's own (in place) unless given."""
    dev = cache.device
    _here(dev)
    refs, tables = cache.refs if refs is None else refs, cache.tables if tables is None else tables
    _need(_list(refs, "refs", dev).numel() == cache.pages and _list(tables, "tables", dev, 2).shape == cache.tables.shape,
          "refs and tables of the cache's sizes wanted")
    live = torch.empty(1, dtype=torch.int32, device=dev) if live is None else _list(live, "live", dev)
    z.check(z.lib().zest_kv_compact(ctypes.byref(cache._layer[0]), cache.layers, cache.layer_stride, cache.refs.data_ptr(),
                                    cache.tables.data_ptr(), cache.tables.shape[0], cache.tables.shape[1], refs.data_ptr(),
                                    tables.data_ptr(), live.data_ptr(), cache._scratch.data_ptr(), cache._scratch.numel(),
                                    _bad(bad, cache), cache._stream()), "zest_kv_compact")
    return live
