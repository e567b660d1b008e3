"""The choice of the next token (include/zest/decode.h): temperature, top-k, top-p,
min-p and the draw, from given random numbers.

Straight to the HIP kernels, on torch's current stream, with device memory owned
by torch tensors; a call that cannot be made raises ZestError. Nothing waits for
the GPU, so a decoding loop can be captured in a HIP graph with it; only default
workspaces and outputs are allocated, from torch's allocator.
"""
from __future__ import annotations

import functools

import torch

import ggml_xdna_amd as z

_TYPES = {torch.float32: z.TYPE_F32, torch.float16: 1, torch.bfloat16: 30}




def _param(t, what: str, rows: int, dtype, device):
    if t is None:
        return None
    if t.dtype is not dtype or t.shape != (rows,) or t.device != device or not t.is_contiguous():
        raise z.ZestError(f"{what}: a contiguous {dtype} tensor of {rows} values on {device} wanted")
    return t.data_ptr()


@functools.lru_cache(maxsize=4096)
def workspace_bytes(rows: int, vocab: int) -> int:
    """Bytes of sample's workspace, 0: none is wanted."""
    return z.lib().zest_sample_workspace(rows, vocab)


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, probs=False, out=None, workspace=None):
    """zest_sample: the next token (int32) of each row of logits [rows][vocab] (float32, float16 or bfloat16, rows any
    stride apart) by u [rows], random numbers in [0, 1). temperature, top_p, min_p (float32) and top_k (int32): one a
    row, 1 and off unless given. probs: True, or a float32 tensor to write, also returns each token's probability
    among those that stayed. out: the tokens' tensor."""
    dev, f32, i32 = logits.device, torch.float32, torch.int32
    if dev.type != "cuda" or dev.index != torch._C._cuda_getDevice():
        raise z.ZestError(f"the logits are on {dev}, which is not the current device")
    kind, shape, stride = _TYPES.get(logits.dtype), logits.shape, logits.stride()
    if kind is None or len(shape) != 2 or (shape[1] > 1 and stride[1] != 1):
        raise z.ZestError("logits: float32, float16 or bfloat16 rows [rows][vocab] wanted")
    if u is None:
        raise z.ZestError("u: a random number a row wanted")
    rows, vocab = shape
    if out is None:
        out = torch.empty(rows, dtype=i32, device=dev)
    if probs is True:
        probs = torch.empty(rows, dtype=f32, device=dev)
    elif probs is False:
        probs = None
    if workspace is None:
        need = workspace_bytes(rows, vocab)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif workspace.device != dev or not workspace.is_contiguous():
        raise z.ZestError(f"workspace: a contiguous tensor on {dev} wanted")
    z.check(z.lib().zest_sample(logits.data_ptr(), kind, rows, vocab, stride[0] if rows > 1 else vocab, _param(u, "u", rows, f32, dev),
                                _param(temperature, "temperature", rows, f32, dev), _param(top_k, "top_k", rows, i32, dev),
                                _param(top_p, "top_p", rows, f32, dev), _param(min_p, "min_p", rows, f32, dev),
                                _param(out, "out", rows, i32, dev), _param(probs, "probs", rows, f32, dev),
                                None if workspace is None else workspace.data_ptr(),
                                0 if workspace is None else workspace.numel() * workspace.element_size(), z._stream()), "zest_sample")
    return out if probs is None else (out, probs)
