"""Attention over packed prompts (include/holo_b200.h, cuda_attention_packed)
on torch tensors.

The reference forwards a prompt one position at a time (src/ai/llm.c:1049);
here whole prompts of different lengths are rows of one call.  The arithmetic
is the library's (csrc/packed_attn.cu); work is enqueued on torch's current
stream.
"""
from __future__ import annotations

import struct

import torch

from . import load, DT_F32, DT_F16, DT_BF16, HOLO_OK

DTYPES = {torch.float32: DT_F32, torch.float16: DT_F16, torch.bfloat16: DT_BF16}
LEGACY_STREAM = 1   # cudaStreamLegacy: torch's default stream has the handle 0, which the library takes for its own
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # absent from builds of torch without CUDA
_device = getattr(torch._C, "_cuda_getDevice", None)


def stream_of(index: int) -> int:
    """The handle of torch's current stream on CUDA device `index`, which has
    to be the current device (the library's state belongs to it)."""
    if index < 0 or index != _device():
        raise ValueError(f"tensors on device {index}: the current CUDA device is needed")
    return _raw_stream(index) or LEGACY_STREAM


_LIB = None


def _lib():
    global _LIB
    _LIB = load()
    return _LIB


def check(rc: int, what: str):
    """Raise on an error status, and clear it."""
    if rc != HOLO_OK:
        lib = load()
        msg = lib.cuda_last_status_string().decode(errors="replace")
        lib.cuda_clear_status()
        raise RuntimeError(f"{what}: status {rc} ({msg})")


# holo_packed_desc: type, n_heads, n_kv_heads, head_dim, n_seqs, total, scale, the strides of q, k, v and out, stream.  Packed
# into bytes, which takes half the time of a ctypes structure: a short call is the host's.
_packed_desc = struct.Struct("@6if8qP").pack


def row_stride(t, heads: int, hd: int, what: str) -> int:
    """Elements between the rows of t [rows][heads][hd] whose heads are
    adjacent; 0, dense, where one row or none leaves it open."""
    if t.is_contiguous():
        return 0
    s = t.stride()
    rows = t.shape[0]
    if (heads > 1 and s[1] != hd) or s[2] != 1 or (rows > 1 and s[0] < heads * hd):
        raise ValueError(f"{what}: strides {s} of {tuple(t.shape)}: the heads of a row have to be adjacent, and rows apart")
    return s[0] if rows > 1 else 0


DENSE = (0,) * 8


def _strides(t, what: str):
    """Elements between the rows and between the heads of t [rows][heads][head_dim]."""
    if t.is_contiguous():
        return 0, 0
    rows, heads, hd = t.shape
    s = t.stride()
    if s[2] != 1 or (rows > 1 and s[0] < hd) or (heads > 1 and s[1] < hd):
        raise ValueError(f"{what}: strides {s} of {tuple(t.shape)}: the values of a head have to be adjacent, and heads apart")
    return s[0] if rows > 1 else 0, s[1] if heads > 1 else 0


def attention_packed(q, k, v, cu_seqlens, out=None, lse=None, scale: float = 0.0):
    """Causal attention of packed prompts: q [total][n_heads][head_dim], k and
    v [total][n_kv_heads][head_dim] (float16 or bfloat16, any strides between
    rows and heads), cu_seqlens int32 [n_seqs + 1] on the device.  Returns out
    (made when None; it overlaps none of the others); lse, when given, is float32 [n_heads][total] and gets
    each row's log-sum-exp.  scale 0: 1 / sqrt(head_dim)."""
    shape, kv_shape = q.shape, k.shape
    total, n_heads, hd = shape
    if kv_shape != v.shape or len(kv_shape) != 3 or kv_shape[0] != total or kv_shape[2] != hd:
        raise ValueError(f"attention_packed: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != shape:
        raise ValueError(f"attention_packed: out {tuple(out.shape)} for q {tuple(q.shape)}")
    dtype = q.dtype
    if dtype not in DTYPES or k.dtype != dtype or v.dtype != dtype or out.dtype != dtype:
        raise TypeError(f"attention_packed: q {q.dtype}, k {k.dtype}, v {v.dtype}, out {out.dtype}: one type is needed")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or not cu_seqlens.is_contiguous():
        raise TypeError("attention_packed: cu_seqlens is a contiguous int32 vector")
    index = q.get_device()
    if k.get_device() != index or v.get_device() != index or out.get_device() != index or cu_seqlens.get_device() != index:
        raise ValueError("attention_packed: the tensors are on different devices")
    if lse is not None:
        if lse.dtype != torch.float32 or lse.shape != (n_heads, total) or not lse.is_contiguous():
            raise TypeError("attention_packed: lse is a contiguous float32 [n_heads][total]")
        if lse.get_device() != index:
            raise ValueError("attention_packed: the tensors are on different devices")
        lse = lse.data_ptr()
    dense = q.is_contiguous() and k.is_contiguous() and v.is_contiguous() and out.is_contiguous()
    strides = DENSE if dense else (*_strides(q, "attention_packed: q"), *_strides(k, "attention_packed: k"),
                                   *_strides(v, "attention_packed: v"), *_strides(out, "attention_packed: out"))
    d = _packed_desc(DTYPES[dtype], n_heads, kv_shape[1], hd, cu_seqlens.numel() - 1, total, scale, *strides, stream_of(index))
    rc = (_LIB or _lib()).cuda_attention_packed(d, out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                cu_seqlens.data_ptr(), lse)
    if rc:
        check(rc, "cuda_attention_packed")
    return out
