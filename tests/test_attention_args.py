"""Refusals of the attention entry points, all decided on the host: no device
is touched and none is needed.  The rotation table against 64 bits."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from colizig_amd import _lib, attn

A = 1 << 20  # addresses that no call gets far enough to use


def cache(**kw):
    a = dict(k_ptr=A, v_ptr=A, pages=8, page_size=16, kv_heads=4, head_dim=128, dtype="bf16")
    a.update(kw)
    return attn.KvCache(**a)


def batch(decode=True, **kw):
    a = dict(len_ptr=A, pages_ptr=A, n=3, rows=3, max_pages=2, row0=None if decode else A)
    a.update(kw)
    return attn.Batch(**a)


def attend(fn="colizig_hip_attn_decode", c=None, b=None, dtype=0, q=A, out=A, heads=32, scale=0.1, work=A, size=1 << 40,
           sq=0, so=0):
    c = cache() if c is None else c
    b = batch(fn.endswith("decode")) if b is None else b
    rc = getattr(_lib.hip(), fn)(ctypes.byref(c), ctypes.byref(b), dtype, q, sq, out, so, heads, scale, work, size, None)
    return rc, _lib.last_error()


def append(c=None, b=None, dtype=0, q=A, k=A, v=A, qo=A, heads=32, rot=None, strides=(0, 0, 0, 0)):
    c = cache() if c is None else c
    b = batch() if b is None else b
    rc = _lib.hip().colizig_hip_attn_append(ctypes.byref(c), ctypes.byref(b), dtype, q, strides[0], k, strides[1], v,
                                            strides[2], qo, strides[3], heads, None if rot is None else ctypes.byref(rot),
                                            None)
    return rc, _lib.last_error()


SIZES = [
    (dict(c=cache(head_dim=96)), "head_dim"),
    (dict(c=cache(head_dim=0)), "head_dim"),
    (dict(c=cache(page_size=0)), "page_size"),
    (dict(c=cache(page_size=24)), "page_size"),
    (dict(c=cache(pages=0)), "pages"),
    (dict(c=cache(kv_heads=0)), "q_heads"),
    (dict(c=cache(kv_heads=5)), "q_heads"),
    (dict(dtype=2), "rows are"),
    (dict(dtype=1, c=cache(dtype="f32")), "caches are"),
    (dict(heads=33), "q_heads"),
]


@pytest.mark.parametrize("kw,why", SIZES)
def test_sizes_and_types(kw, why):
    for call in (attend, lambda **k: attend("colizig_hip_attn_prompt", **k), append):
        rc, msg = call(**kw)
        assert rc == -1 and why in msg, msg


@pytest.mark.parametrize("b,why", [
    (dict(n=0, rows=0), "at least 1"), (dict(rows=4), "one row per sequence"), (dict(max_pages=0), "at least 1"),
    (dict(max_pages=(1 << 26) + 1), "2^30"), (dict(n=1 << 28, rows=1 << 28), "too many"),
])
def test_batches(b, why):
    for call in (attend, append):
        rc, msg = call(b=batch(**b))
        assert rc == -1 and why in msg, msg


def test_row0_says_which_form():
    assert attend(b=batch(False))[0] == -1
    rc, msg = attend("colizig_hip_attn_prompt", b=batch(True))
    assert rc == -1 and "row0" in msg


def test_null_structs():
    h = _lib.hip()
    b, c = batch(), cache()
    assert h.colizig_hip_attn_decode(None, ctypes.byref(b), 0, A, 0, A, 0, 32, 0.1, A, 1 << 40, None) == -1
    assert h.colizig_hip_attn_decode(ctypes.byref(c), None, 0, A, 0, A, 0, 32, 0.1, A, 1 << 40, None) == -1
    assert h.colizig_hip_attn_append(None, None, 0, A, 0, A, 0, A, 0, A, 0, 32, None, None) == -1
    assert h.colizig_hip_attn_work_bytes(None, None, 32) == 0


def test_work_bytes():
    assert attn.work_bytes(cache(), batch(), 32) > 0
    assert attn.work_bytes(cache(), batch(False, rows=900), 32) > 0
    assert attn.work_bytes(cache(head_dim=80), batch(), 32) == 0
    assert attn.work_bytes(cache(), batch(), 0) == 0
    with pytest.raises(Exception):
        attn.decode(cache(), batch(), "f32", A, A, 32, float("nan"), A, 1 << 40)


def test_not_initialised_is_refused():
    if _lib.hip().colizig_cuda_init() == 0:
        pytest.skip("a GPU is present")
    for call in (attend, lambda: attend("colizig_hip_attn_prompt"), append):
        rc, msg = call()
        assert rc == -1 and "not initialised" in msg


@pytest.mark.gpu
@pytest.mark.parametrize("kw,why", [
    (dict(c=cache(k_ptr=None)), "null"), (dict(c=cache(v_ptr=A + 8)), "aligned"),
    (dict(c=cache(strides=(0, 0, 64))), "stride"), (dict(c=cache(strides=(8192, 2048, 132))), "stride"),
    (dict(c=cache(strides=(0, 2048, 128))), "stride"), (dict(c=cache(strides=(8192, 2048, (1 << 24) + 128))), "stride"),
    (dict(c=cache(strides=(1 << 41, 2048, 128))), "stride"),
    (dict(b=batch(len_ptr=None)), "null"), (dict(b=batch(pages_ptr=None)), "null"), (dict(b=batch(len_ptr=A + 2)), "aligned"),
    (dict(q=None), "missing"), (dict(out=A + 4), "aligned"), (dict(sq=32 * 128 - 4), "stride"),
    (dict(so=32 * 128 + 2), "stride"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(heads=0), "q_heads"), (dict(work=None), "scratch"), (dict(work=A + 8), "scratch"), (dict(size=1), "scratch"),
])
def test_pointers_and_strides(gpu, kw, why):
    rc, msg = attend(**kw)
    assert rc == -1 and why in msg, msg


@pytest.mark.gpu
@pytest.mark.parametrize("kw,why", [
    (dict(q=None), "together"), (dict(qo=None), "together"), (dict(heads=0), "together"), (dict(k=None), "missing"),
    (dict(v=A + 8), "aligned"), (dict(strides=(0, 500, 0, 0)), "stride"), (dict(strides=(0, 0, 514, 0)), "stride"),
    (dict(rot=attn.Rotation(A, 0, 128)), "rotation"), (dict(rot=attn.Rotation(A, 9, 24)), "rotation"),
    (dict(rot=attn.Rotation(A, 9, 144)), "rotation"), (dict(rot=attn.Rotation(A + 4, 9, 128)), "aligned"),
    (dict(rot=attn.Rotation(None, 0, 0, q_norm=A, eps=-1.0)), "eps"),
    (dict(rot=attn.Rotation(None, 0, 0, k_norm=A, eps=float("nan"))), "eps"),
])
def test_append_arguments(gpu, kw, why):
    rc, msg = append(**kw)
    assert rc == -1 and why in msg, msg


def test_rope_table():
    t = attn.rope_table(70000, 64, 1e6)
    p = np.array([0, 1, 4095, 69999])
    inv = [1e6 ** (-2 * i / 64) for i in range(32)]
    ref = np.array([[np.cos(float(a) * w) for w in inv] + [np.sin(float(a) * w) for w in inv] for a in p])
    assert t.dtype == np.float32 and t.shape == (70000, 64)
    assert np.abs(t[p] - ref).max() <= 2.0 ** -24  # half a step below 1, angles to 64 bits
