"""Attention between a layer's projections, on device pointers: new keys and
values into a paged cache (`append`), one new token per sequence (`decode`),
prompts, prompt chunks and drafts (`prompt`).  The C declarations and every
contract are in include/colizig_hip.h; q, k, v and out are rows as
moe.matmul_fp8_dev_multi gives them and moe.matmul_fp8_dev takes them.

The objects here hold device addresses, not the memory: the caller keeps it.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib
from .moe import _check

TYPES = {"f32": 0, "bf16": 1, "e4m3": 2}


def KvCache(k_ptr: int, v_ptr: int, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: str,
            k_scale: int | None = None, v_scale: int | None = None, strides=(0, 0, 0)) -> _lib.KvCache:
    """A paged cache over device memory; strides: page, head, token in elements (zeros: [page][head][slot][dim])."""
    return _lib.KvCache(k_ptr, v_ptr, k_scale, v_scale, *strides, pages, page_size, kv_heads, head_dim, TYPES[dtype])


def Batch(len_ptr: int, pages_ptr: int, n: int, rows: int, max_pages: int, row0: int | None = None) -> _lib.AttnBatch:
    """The sequences of a call: device int32 arrays of lengths, page numbers and, for more than one row each, first rows."""
    return _lib.AttnBatch(row0, len_ptr, pages_ptr, n, rows, max_pages)


def Rotation(table_ptr: int | None, positions: int, dims: int, q_norm: int | None = None, k_norm: int | None = None,
             eps: float = 1e-6) -> _lib.Rotation:
    """Norm weights and rotation table (rope_table, uploaded) of q and k."""
    return _lib.Rotation(table_ptr, q_norm, k_norm, positions, dims, eps)


def rope_table(positions: int, dims: int, theta: float) -> np.ndarray:
    """f32 [positions][dims]: cos(p / theta^(2i/dims)) for i < dims/2, then the sines; angles in 64 bits."""
    inv = float(theta) ** (-np.arange(0, dims, 2, dtype=np.float64) / dims)
    ang = np.arange(positions, dtype=np.float64)[:, None] * inv
    return np.concatenate([np.cos(ang), np.sin(ang)], axis=1).astype(np.float32)


def append(cache, batch, dtype: str, q: int | None, k: int, v: int, q_out: int | None, q_heads: int, rotation=None,
           strides=(0, 0, 0, 0), stream=None) -> None:
    """colizig_hip_attn_append; strides of q, k, v and q_out from row to row in elements (0: dense)."""
    rot = None if rotation is None else ctypes.byref(rotation)
    _check("colizig_hip_attn_append", _lib.hip().colizig_hip_attn_append(
        ctypes.byref(cache), ctypes.byref(batch), TYPES[dtype], q, strides[0], k, strides[1], v, strides[2], q_out,
        strides[3], q_heads, rot, stream))


def work_bytes(cache, batch, q_heads: int) -> int:
    """Scratch of a `decode` or `prompt` call with these sizes."""
    return _lib.hip().colizig_hip_attn_work_bytes(ctypes.byref(cache), ctypes.byref(batch), q_heads)


def decode(cache, batch, dtype: str, q: int, out: int, q_heads: int, scale: float, work: int, work_size: int,
           strides=(0, 0), stream=None) -> None:
    """colizig_hip_attn_decode: one new token per sequence."""
    _check("colizig_hip_attn_decode", _lib.hip().colizig_hip_attn_decode(
        ctypes.byref(cache), ctypes.byref(batch), TYPES[dtype], q, strides[0], out, strides[1], q_heads, scale, work,
        work_size, stream))


def prompt(cache, batch, dtype: str, q: int, out: int, q_heads: int, scale: float, work: int, work_size: int,
           strides=(0, 0), stream=None) -> None:
    """colizig_hip_attn_prompt: causal attention of packed sequences' new tokens."""
    _check("colizig_hip_attn_prompt", _lib.hip().colizig_hip_attn_prompt(
        ctypes.byref(cache), ctypes.byref(batch), TYPES[dtype], q, strides[0], out, strides[1], q_heads, scale, work,
        work_size, stream))
