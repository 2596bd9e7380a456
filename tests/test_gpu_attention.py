"""Attention over a paged cache (colizig_hip_attn_append, _decode, _prompt)
against 64 bits, with bounds from the roundings that each result goes through
(tests/attn_helpers.py).  Unused slots, pages and scratch hold NaN."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from colizig_amd import _lib, attn, moe, synth
from tests import attn_helpers as H
from tests.helpers import deq_f64

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f32", "bf16"), ("f32", "e4m3"), ("bf16", "bf16"), ("bf16", "e4m3")]


@pytest.fixture
def dev(gpu):
    d = H.Dev()
    yield d
    _lib.hip().colizig_hip_sync()
    d.free()


def say(*a):
    print(*a, flush=True)


# ---- append -------------------------------------------------------------------
def _append(p: H.Problem, dev: H.Dev, in_place=False, keys_only=False):
    p.upload(dev)
    dk, dv = dev.put(p.kx), dev.put(p.vx)
    rope = dev.put(p.rope) if p.rope is not None else None
    qn, kn = (dev.put(p.q_norm), dev.put(p.k_norm)) if p.q_norm is not None else (None, None)
    rot = attn.Rotation(rope.ptr if rope else None, 0 if rope is None else p.rope.shape[0], p.dims,
                        q_norm=qn.ptr if qn else None, k_norm=kn.ptr if kn else None, eps=p.eps)
    sq, sk = p.row_stride(p.hq), p.row_stride(p.hk)
    q, qo = (None, None) if keys_only else (p.dq.ptr, p.dq.ptr if in_place else p.dout.ptr)
    attn.append(p.cache, p.batch, p.rows_t, q, dk.ptr, dv.ptr, qo, p.hq, rot, strides=(sq, sk, sk, sq))
    rc = _lib.hip().colizig_hip_sync()
    assert rc == 0, _lib.last_error()
    return ((p.dq if in_place else p.dout).download(np.empty_like(p.out0)), p.dk.download(np.empty_like(p.k)),
            p.dv.download(np.empty_like(p.v)))


def _turned(p: H.Problem, x, w, pos):
    """Rows [t][heads][d] normalised and rotated in 64 bits, and what f32 steps may have done to them."""
    e = np.zeros_like(x)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + p.eps) * w.astype(np.float64)
        e = (p.d + 8) * H.U32 * np.abs(x)  # the sum of squares, mean, root, quotient and two products
    if p.dims:
        h = p.dims // 2
        t = p.rope[pos].astype(np.float64)[:, None]
        c, s = t[..., :h], t[..., h:]
        a, b = x[..., :h].copy(), x[..., h:p.dims].copy()
        ea, eb = e[..., :h].copy(), e[..., h:p.dims].copy()
        x, e = x.copy(), e.copy()
        x[..., :h], x[..., h:p.dims] = a * c - b * s, b * c + a * s
        m = (np.abs(a) + np.abs(b)) * 4 * H.U32
        e[..., :h], e[..., h:p.dims] = ea * abs(c) + eb * abs(s) + m, eb * abs(c) + ea * abs(s) + m
    return x, e


def _held_ok(got, ref, err, t):
    """Values as type t holds them, ref being off by err before that rounding."""
    step = {"f32": H.U32, "bf16": H.U16, "e4m3": H.U8}[t] * (np.abs(ref) + err)
    if t == "e4m3":
        step = np.maximum(step, 2.0 ** -10) + 2 * H.U32 * np.abs(ref)
        ref = np.clip(ref, -448, 448)
    return np.abs(got - ref) <= err + step + 1e-37


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("heads,page,layout,pad,dims,norm,new,past", [
    ((32, 4, 128), 16, "heads", 0, None, True, [1], [0]),
    ((32, 4, 128), 64, "slots", 64, None, True, [1, 1, 1, 0, 1], [0, 15, 16, 4, 700]),
    ((6, 2, 64), 48, "heads", 16, 32, False, [5, 0, 130, 1], [0, 3, 47, 96]),
    ((3, 1, 256), 32, "slots", 0, 64, True, [33, 64], [31, 0]),
    ((5, 5, 64), 16, "heads", 0, 0, False, [17, 2], [1, 14]),
])
def test_append(dev, rows, cache, heads, page, layout, pad, dims, norm, new, past):
    say("append", rows, cache, heads, page, layout, new)
    p = H.Problem(rows, cache, heads, new, [a + b for a, b in zip(new, past)], page, layout, pad, extra_rows=3, seed=5,
                  dims=dims, norm=norm)
    k0, v0 = p.k.copy(), p.v.copy()
    q, k, v = _append(p, dev)
    last = p.row0[-1]
    pos = np.concatenate([np.arange(L - n, L) for n, L in zip(p.new, p.len)]).astype(int)
    part = lambda a, h: H.decode(a[:last, :h * p.d].reshape(last, h, p.d), rows)
    ref, err = _turned(p, part(p.q, p.hq), p.q_norm, pos)
    assert _held_ok(part(q, p.hq), ref, err, rows).all()
    assert np.array_equal(q[last:].view(np.uint8), p.out0[last:].view(np.uint8)), "rows behind the last sequence"
    if pad:
        assert np.array_equal(np.ascontiguousarray(q[:, p.hq * p.d:]).view(np.uint8),
                              np.ascontiguousarray(p.out0[:, p.hq * p.d:]).view(np.uint8))
    for name, got, was, x, w, i in (("k", k, k0, p.kx, p.k_norm, 0), ("v", v, v0, p.vx, None, 1)):
        ref, err = _turned(p, part(x, p.hk), w, pos) if i == 0 else (part(x, p.hk), 0.0)
        sc = p.scale[i][:, None].astype(np.float64)
        ref, err = ref / sc, err / sc
        for b in range(p.n):
            r, n, L = p.row0[b], p.new[b], p.len[b]
            held = H.decode(p.get(got, b, L)[L - n:], cache)
            assert _held_ok(held, ref[r:r + n], (err if np.isscalar(err) else err[r:r + n]) if i == 0 else 0.0, cache).all(), name
            # put the old tokens back: everything else has its old bits
            p.set(got, b, L - n, p.get(was, b, L)[L - n:])
        assert np.array_equal(got.view(np.uint8), was.view(np.uint8)), f"{name}: bits beside the new tokens"


def test_append_in_place_and_keys_only(dev):
    say("append: q rotated in place, and keys alone")
    p = H.Problem("f32", "bf16", (8, 2, 128), [9, 4], [9, 30], seed=6)
    q, k, v = _append(p, dev)
    p2 = H.Problem("f32", "bf16", (8, 2, 128), [9, 4], [9, 30], seed=6)
    q2, k2, v2 = _append(p2, dev, in_place=True)
    assert np.array_equal(q, q2) and np.array_equal(k, k2) and np.array_equal(v, v2)
    p3 = H.Problem("f32", "bf16", (8, 2, 128), [9, 4], [9, 30], seed=6)
    q3, k3, v3 = _append(p3, dev, keys_only=True)
    assert np.array_equal(q3.view(np.uint32), p3.out0.view(np.uint32))
    assert np.array_equal(k, k3) and np.array_equal(v, v3)


def test_append_e4m3_saturates_and_keeps_nan(dev):
    say("append: values past the E4M3 range, NaN")
    p = H.Problem("f32", "e4m3", (2, 2, 64), [4], [4], seed=7, dims=0, norm=False)
    p.vx[0, 0], p.vx[1, 1], p.vx[2, 2], p.vx[3, 3] = 1e9, -np.inf, np.nan, 1e-9
    _, _, v = _append(p, dev)
    got = H.decode(p.get(v, 0, 4), "e4m3").reshape(4, -1)
    assert got[0, 0] == 448 and got[1, 1] == -448 and np.isnan(got[2, 2]) and got[3, 3] == 0
    assert np.isfinite(np.delete(got.ravel(), 2 * 128 + 2)).all()


def test_append_padding_rows(dev):
    """Rows at negative positions (a padded batch): nothing is written for them."""
    say("append: padding rows")
    p = H.Problem("f32", "bf16", (8, 2, 64), [1, 1, 1], [7, 1, 20], seed=8)
    p.len[1] = 0
    k0 = p.k.copy()
    q, k, _ = _append(p, dev)
    assert np.array_equal(q[1].view(np.uint32), p.out0[1].view(np.uint32))
    pg, sl = p.where(1, np.arange(1))
    assert np.array_equal(k[pg, :, sl], k0[pg, :, sl])
    assert not np.isnan(q[0]).any() and not np.isnan(q[2]).any()


def test_append_norm_alone_first_rows_and_no_scales(dev):
    """A norm of k alone without a rotation, sequences that start behind row 0
    (the rows before them stay), an E4M3 cache without scales."""
    say("append: k's norm alone, rows before the first sequence, no scales")
    p = H.Problem("f32", "e4m3", (4, 2, 64), [3, 2], [3, 20], seed=9, dims=0, extra_rows=4)
    p.upload(dev)
    p.scale[:] = 1.0
    p.cache.k_scale = p.cache.v_scale = None
    p.drow0.upload(p.row0 + 4)
    dk, dv, kn = dev.put(p.kx), dev.put(p.vx), dev.put(p.k_norm)
    rot = attn.Rotation(None, 0, 0, k_norm=kn.ptr, eps=p.eps)
    k0 = p.k.copy()
    attn.append(p.cache, p.batch, "f32", p.dq.ptr, dk.ptr, dv.ptr, p.dout.ptr, p.hq, rot)
    assert _lib.hip().colizig_hip_sync() == 0
    q, k = p.dout.download(np.empty_like(p.out0)), p.dk.download(np.empty_like(p.k))
    assert np.array_equal(q[:4].view(np.uint32), p.out0[:4].view(np.uint32))
    assert np.array_equal(q[4:9], p.q[4:9])
    for b in range(2):
        r, n, L = p.row0[b] + 4, p.new[b], p.len[b]
        x = p.kx[r:r + n].reshape(n, 2, 64).astype(np.float64)
        ref, err = _turned(p, x, p.k_norm, None)
        assert _held_ok(H.decode(p.get(k, b, L)[L - n:], "e4m3"), ref, err, "e4m3").all()
        assert np.array_equal(p.get(k, b, L)[:L - n], p.get(k0, b, L)[:L - n])
    p.k, p.v = k, p.dv.download(np.empty_like(p.v))
    p.row0 = p.row0 + 4
    p.scale_qk = 0.125
    size = attn.work_bytes(p.cache, p.batch, p.hq)
    work = dev.put(np.zeros(size, np.uint8))
    p.dout.upload(p.out0)
    attn.prompt(p.cache, p.batch, "f32", p.dq.ptr, p.dout.ptr, p.hq, 0.125, work.ptr, size)
    got = p.fetch()
    assert np.array_equal(got[:4].view(np.uint32), p.out0[:4].view(np.uint32))
    p.check(got, rows=set(range(4, 9)))


# ---- one token ------------------------------------------------------------------
@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("heads,page,layout,pad,lens", [
    ((32, 4, 128), 16, "heads", 0, [1]),
    ((32, 4, 128), 64, "heads", 64, [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 300]),
    ((12, 12, 64), 48, "slots", 0, [100, 0, 47, 48, 49]),
    ((16, 2, 256), 32, "slots", 16, [257, 31, 1]),
    ((40, 1, 128), 16, "heads", 0, [511, 20]),
    ((21, 3, 64), 128, "heads", 0, [5000, 3]),
])
def test_decode(dev, rows, cache, heads, page, layout, pad, lens):
    say("decode", rows, cache, heads, page, layout, lens)
    p = H.Problem(rows, cache, heads, [1] * len(lens), lens, page, layout, pad, seed=11)
    p.check(p.attend(dev, decode_form=True))


@pytest.mark.parametrize("rows,cache", [("f32", "bf16"), ("bf16", "e4m3"), ("f32", "f32")])
def test_decode_long(dev, rows, cache):
    """Parts over a long cache, a short sequence beside it."""
    say("decode of 40,001 tokens", rows, cache)
    p = H.Problem(rows, cache, (8, 2, 128), [1, 1, 1], [40001, 5, 9000], 64, seed=12)
    p.check(p.attend(dev, decode_form=True))


def test_decode_many_sequences(dev):
    """More sequences than the chip has workgroups."""
    say("decode of 700 sequences")
    rng = np.random.default_rng(3)
    p = H.Problem("f32", "bf16", (8, 2, 64), [1] * 700, list(rng.integers(0, 80, 700)), seed=13)
    p.check(p.attend(dev, decode_form=True))


# ---- prompts ----------------------------------------------------------------------
@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("heads,page,layout,pad,new,past", [
    ((32, 4, 128), 16, "heads", 0, [1], [0]),
    ((8, 1, 128), 64, "heads", 0, [3, 0, 70, 1, 17], [0, 4, 0, 130, 63]),
    ((4, 4, 64), 48, "slots", 16, [130, 65], [0, 300]),
    ((6, 2, 64), 16, "heads", 0, [64, 129, 2], [64, 1, 700]),
    ((4, 2, 256), 32, "slots", 0, [40, 33], [0, 95]),
    ((40, 8, 128), 128, "heads", 64, [50], [11]),
])
def test_prompt(dev, rows, cache, heads, page, layout, pad, new, past):
    say("prompt", rows, cache, heads, page, layout, new, past)
    p = H.Problem(rows, cache, heads, new, [a + b for a, b in zip(new, past)], page, layout, pad, extra_rows=5, seed=21)
    p.check(p.attend(dev))


@pytest.mark.parametrize("rows,cache", TYPES)
def test_prompt_long(dev, rows, cache):
    """A prompt over many tiles, checked at some rows."""
    say("prompt of 1500 tokens", rows, cache)
    p = H.Problem(rows, cache, (8, 2, 128), [1500, 301], [1500, 301], 64, seed=22)
    rows_ = set(np.random.default_rng(0).integers(0, 1801, 60)) | {0, 1, 1498, 1499, 1500, 1800}
    p.check(p.attend(dev), rows=rows_)


@pytest.mark.parametrize("rows,cache", TYPES)
def test_prompt_draft(dev, rows, cache):
    """A few tokens on long caches: the parts over the cache's length are joined."""
    say("draft of 5 tokens on 9,000", rows, cache)
    p = H.Problem(rows, cache, (8, 2, 128), [5, 2, 1], [9000, 61, 4097], 32, seed=23)
    p.check(p.attend(dev))


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("heads,new,past", [
    ((8, 2, 128), [1], [3000]), ((8, 2, 128), [7, 1], [2500, 300]), ((8, 2, 128), [150], [0]), ((8, 2, 128), [200], [2200]),
    ((4, 4, 64), [300], [2100]), ((4, 2, 256), [140], [2100]), ((16, 2, 64), [60], [100]),
])
def test_rising_scores(dev, rows, cache, heads, new, past):
    """Scores that spread over many powers of e and grow with the position, so
    that a row's largest rises again and again: every kernel and tile size (one
    token, few rows, 64- and 128-row tiles, parts) scales down what it holds."""
    say("rising scores", rows, cache, heads, new, past)
    p = H.Problem(rows, cache, heads, new, [a + b for a, b in zip(new, past)], 32, q_scale=3.0, seed=28)
    for b in range(p.n):
        k = H.decode(p.get(p.k, b, p.len[b]), cache)
        k *= (0.2 + 2.0 * np.arange(p.len[b]) / p.len[b])[:, None, None]
        p.set(p.k, b, 0, H.encode(k, cache))
    total = p.row0[-1]
    sel = None if total < 40 else set(np.random.default_rng(1).integers(0, total, 40)) | {0, total - 1}
    p.check(p.attend(dev, decode_form=max(new) == 1 and len(new) == 1), rows=sel)


def test_prompt_rows_before_the_start(dev):
    """More rows than tokens: rows at negative positions see nothing and give zeros."""
    say("prompt: rows without a key")
    p = H.Problem("f32", "bf16", (4, 2, 64), [4, 3], [6, 3], seed=24)
    p.len[0] = 2
    got = p.attend(dev)
    assert not got[:2, :4 * 64].any()
    p.check(got)
    # whole tiles of them, in each tile size
    for cache in ("bf16", "f32"):
        for heads, n in (((4, 1, 64), 300), ((32, 2, 256), 700)):
            p = H.Problem("f32", cache, heads, [n, 2], [n, 2], seed=29)
            p.len[0] = 20
            got = p.attend(dev)
            assert not got[:n - 20, :heads[0] * heads[2]].any()
            p.check(got, rows=set(range(n - 25, n + 2)))


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_masked_keys_do_not_reach_earlier_rows(dev, rows, cache, bad):
    """A later token's key and value that are not finite leave the rows before
    it their bits; the rows that see them are not finite."""
    if cache == "e4m3" and bad == "inf":
        pytest.skip("E4M3 has no infinity")
    say("not finite in masked places", rows, cache, bad)
    a = H.Problem(rows, cache, (8, 2, 128), [200], [230], seed=25)
    ra = a.attend(dev)
    b = H.Problem(rows, cache, (8, 2, 128), [200], [230], seed=25)
    x = {"nan": H.NAN[cache], "inf": {"f32": np.float32(np.inf), "bf16": np.uint16(0x7F80)}.get(cache)}[bad]
    at = 100  # position; row 70 is the first that sees it
    for c, cols in ((b.k, slice(0, 8)), (b.v, slice(None))):
        t = b.get(c, 0, 230).copy()
        t[at, :, cols] = x
        b.set(c, 0, 0, t)
    rb = b.attend(dev)
    bits = lambda v: np.ascontiguousarray(v).view(np.uint8)
    assert np.array_equal(bits(ra[:70]), bits(rb[:70]))
    assert not np.isfinite(H.decode(rb[70:], rows)).any()


@pytest.mark.parametrize("rows,cache", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
def test_infinite_values(dev, rows, cache):
    """An infinite value of a visible token is an infinity in the rows that see it, at its number alone."""
    say("infinite values", rows, cache)
    a = H.Problem(rows, cache, (4, 2, 64), [40], [40], seed=26)
    ra = a.attend(dev)
    b = H.Problem(rows, cache, (4, 2, 64), [40], [40], seed=26)
    t = b.get(b.v, 0, 40).copy()
    t[30, 1, 5] = {"f32": np.float32(-np.inf), "bf16": np.uint16(0xFF80)}[cache]
    b.set(b.v, 0, 0, t)
    rb = H.decode(b.attend(dev), rows).reshape(40, 4, 64)
    ra = H.decode(ra, rows).reshape(40, 4, 64)
    assert (rb[30:, 2:, 5] == -np.inf).all()
    rb[30:, 2:, 5] = ra[30:, 2:, 5] = 0
    assert np.array_equal(ra, rb)


def test_scales(dev):
    """A scale of 0, a negative one, and one that makes the softmax a choice of the largest."""
    for scale in (0.0, -0.5, 40.0):
        say("scale", scale)
        p = H.Problem("f32", "bf16", (4, 2, 64), [33, 1], [60, 90], seed=27)
        p.check(p.attend(dev, scale=scale))


# ---- places, streams, graphs --------------------------------------------------------
def test_far_pages(dev):
    """Pages whose elements are past 2^32 from the cache's start."""
    say("pages past 2^32 elements")
    p = H.Problem("f32", "e4m3", (8, 2, 128), [1, 40], [60, 40], seed=31)
    stride = (1 << 32) // 4
    size = p.hk * p.page * p.d
    assert p.pages * stride > 1 << 32
    p.attend(dev, launch=False)
    big = moe.DeviceBuffer((p.pages - 1) * stride + 2 * size)
    try:
        for c, off in ((p.k, 0), (p.v, size)):
            for i in range(p.pages):
                page = np.ascontiguousarray(c[i])
                assert _lib.hip().colizig_hip_memcpy_htod(big.ptr + i * stride + off, page.ctypes.data, size) == 0
        p.cache.k, p.cache.v = big.ptr, big.ptr + size
        p.cache.page_stride, p.cache.head_stride, p.cache.token_stride = stride, p.page * p.d, p.d
        p.call()
        p.check(p.fetch())
    finally:
        big.free()


def test_out_may_be_q(dev):
    say("out in q's place")
    for form, new, lens in ((True, [1, 1], [5000, 40]), (False, [3, 200], [5000, 200])):
        p = H.Problem("f32", "bf16", (8, 2, 128), new, lens, seed=32)
        want = p.attend(dev, decode_form=form)
        attn_fn = attn.decode if form else attn.prompt
        attn_fn(p.cache, p.batch, "f32", p.dq.ptr, p.dq.ptr, p.hq, p.scale_qk, p.work.ptr, p.work.nbytes)
        assert _lib.hip().colizig_hip_sync() == 0
        assert np.array_equal(p.dq.download(np.empty_like(p.q)), want)


def test_same_bits_again_and_on_other_streams(dev):
    """Three calls in flight on three streams, each with its scratch: the bits of each call alone."""
    torch = pytest.importorskip("torch")
    say("streams")
    ps = [H.Problem("f32", "bf16", (8, 2, 128), [1, 1], [9000, 3], seed=33),
          H.Problem("bf16", "bf16", (8, 2, 128), [100, 3], [100, 5000], seed=34),
          H.Problem("f32", "f32", (8, 2, 128), [6], [7000], seed=35)]
    want = [p.attend(dev, decode_form=i == 0) for i, p in enumerate(ps)]
    streams = [torch.cuda.Stream() for _ in ps]
    for _ in range(3):
        for p, st in zip(ps, streams):
            p.call(st.cuda_stream)
    torch.cuda.synchronize()
    for p, w in zip(ps, want):
        assert np.array_equal(p.fetch().view(np.uint8), w.view(np.uint8))


def test_captured_calls(dev):
    """Decode, prompt and append captured into graphs and replayed with eager
    work between the replays, lengths and inputs changing in place: each
    replay has the bits of an eager call on the same inputs."""
    torch = pytest.importorskip("torch")
    say("graphs")
    ps = [H.Problem("f32", "bf16", (8, 2, 128), [1, 1], [6000, 500], seed=36),
          H.Problem("f32", "e4m3", (8, 2, 128), [40, 3], [40, 5000], seed=37)]
    graphs = []
    for i, p in enumerate(ps):
        p.attend(dev, decode_form=i == 0, launch=False)
        p.xk, p.xv = dev.put(p.kx), dev.put(p.vx)
        p.append = lambda st, p=p: attn.append(p.cache, p.batch, "f32", p.dq.ptr, p.xk.ptr, p.xv.ptr, p.dq.ptr, p.hq,
                                               None, stream=st)
        st = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            p.append(torch.cuda.current_stream().cuda_stream)
            p.call(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    rng = np.random.default_rng(9)
    for it in range(4):
        lens = [[6000 - 1777 * it, 500 - 100 * it], [40, 5000 - 1300 * it]]
        for p, ln in zip(ps, lens):
            p.dlen.upload(np.array(ln, np.int32))
            p.dq.upload(rng.normal(size=p.q.shape).astype(np.float32))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [p.fetch() for p in ps]
        for i, p in enumerate(ps):
            p.dout.upload(p.out0)
            p.append(None)
            p.call()
            w = p.fetch()
            assert np.isfinite(w).all()
            assert np.array_equal(got[i].view(np.uint32), w.view(np.uint32)), (it, i)


def test_bad_pages_and_lengths_are_reported(dev):
    """What the device arrays hold is checked by the kernels: the next sync says so, once."""
    say("bad pages and lengths")
    hip = _lib.hip()
    for form in (True, False):
        p = H.Problem("f32", "bf16", (8, 2, 128), [1, 1], [40, 20], seed=41)
        p.attend(dev, decode_form=form, launch=False)
        bad = p.table.copy()
        bad[1, 1] = p.pages
        p.dtable.upload(bad)
        p.call()
        assert hip.colizig_hip_sync() == -5 and "page" in _lib.last_error()
        assert hip.colizig_hip_sync() == 0
        p.dtable.upload(p.table)
        p.dlen.upload(np.array([40, p.width * p.page + 1], np.int32))
        p.table[1] = np.where(p.table[1] < 0, 0, p.table[1])
        p.dtable.upload(p.table)
        p.call()
        assert hip.colizig_hip_sync() == -5 and "lengths" in _lib.last_error()
        p.dlen.upload(np.array([40, 20], np.int32))
        p.call()
        p.check(p.fetch())
    # append: a bad page is not written, a position past the table is not appended
    p = H.Problem("f32", "bf16", (8, 2, 128), [1, 1], [40, 20], seed=42)
    p.rope = p.rope[:30]
    p.upload(dev)
    dk, dv, rope = dev.put(p.kx), dev.put(p.vx), dev.put(p.rope)
    rot = attn.Rotation(rope.ptr, 30, p.dims)
    bad = p.table.copy()
    bad[1, 1] = -1
    p.dtable.upload(bad)
    attn.append(p.cache, p.batch, "f32", p.dq.ptr, dk.ptr, dv.ptr, p.dout.ptr, p.hq, rot)
    assert hip.colizig_hip_sync() == -5
    assert "page" in _lib.last_error() and "position" in _lib.last_error()
    assert np.array_equal(p.dk.download(np.empty_like(p.k)), p.k)


def test_rows_that_overlap_are_reported(dev):
    """row0 that falls: cut to what is there, reported, nothing out of bounds (the rows' results are invalid)."""
    say("falling row0")
    hip = _lib.hip()
    for new, lens in (([3] * 9, [500] * 9), ([40] * 9, [900] * 9), ([300] * 6, [3000] * 6)):
        p = H.Problem("f32", "bf16", (8, 2, 64), new, lens, 64, seed=43)
        p.attend(dev, launch=False)
        total = int(p.row0[-1])
        p.drow0.upload(np.array([0 if b % 2 == 0 else total for b in range(p.n + 1)], np.int32))
        p.call()
        assert hip.colizig_hip_sync() == -5 and "rows" in _lib.last_error()
        dk, dv = dev.put(p.kx), dev.put(p.vx)
        attn.append(p.cache, p.batch, "f32", p.dq.ptr, dk.ptr, dv.ptr, p.dout.ptr, p.hq)
        assert hip.colizig_hip_sync() in (0, -5)
        p.upload(dev)
        p.call()
        assert hip.colizig_hip_sync() in (0, -5)


@pytest.mark.parametrize("heads", [(8, 2, 64), (40, 1, 64)])
def test_thousands_of_sequences(dev, heads):
    """More sequences than workgroups, each a workgroup's own: no search for its place."""
    say("5,000 sequences", heads)
    rng = np.random.default_rng(4)
    n = 5000
    p = H.Problem("f32", "bf16", heads, [1] * n, list(rng.integers(0, 40, n)), seed=14)
    sel = set(rng.integers(0, n, 200)) | {0, n - 1}
    p.check(p.attend(dev, decode_form=True), rows=sel)
    new = list(rng.integers(0, 4, 600))
    p = H.Problem("bf16", "e4m3", heads, new, [a + int(b) for a, b in zip(new, rng.integers(0, 90, 600))], seed=15)
    p.check(p.attend(dev))


# ---- all of it together ---------------------------------------------------------------
def test_projections_append_prompt_decode(dev, oracle_lib):
    """A layer's attention as a program runs it: FP8 q, k and v projections,
    append (norm and rotation), a prompt, then two tokens one by one, each
    through the o projection; against the same in 64 bits.  The bar: the
    projections' 1e-5, twice, and the cache's BF16 steps where it has them."""
    say("projections, append, prompt, two tokens")
    hid, hq, hk, d, page, T = 512, 8, 2, 64, 16, 45
    rng = np.random.default_rng(50)
    moe.set_vram_budget(1 << 30)
    try:
        shapes = [(hq * d, hid), (hk * d, hid), (hk * d, hid), (hid, hq * d)]
        mats, keys = [], []
        for role, (O, I) in enumerate(shapes):
            w, s = synth.block_quantize(rng.normal(0, 0.05, size=(O, I)).astype(np.float32))
            keys.append(moe.Fp8Matrix.attn_key(31, role))
            moe.matrix_load(keys[-1], w, s)
            mats.append(deq_f64(w, s))
        x = rng.normal(size=(T, hid)).astype(np.float32)
        table = rng.permutation(6).astype(np.int32)[None, :4].copy()
        rope = attn.rope_table(64, d, 1e4)
        norm = (1 + 0.1 * rng.normal(size=(2, d))).astype(np.float32)
        kc, vc = dev.put(np.full((6, hk, page, d), np.nan, np.float32)), dev.put(np.full((6, hk, page, d), np.nan, np.float32))
        cache = attn.KvCache(kc.ptr, vc.ptr, 6, page, hk, d, "f32")
        dt, dr, dn, dx = dev.put(table), dev.put(rope), dev.put(norm), dev.put(x)
        rot = attn.Rotation(dr.ptr, 64, d, q_norm=dn.ptr, k_norm=dn.ptr + 4 * d)
        qkv = dev.put(np.zeros((T, (hq + 2 * hk) * d), np.float32))
        q, k, v = (dev.put(np.zeros((T, h * d), np.float32)) for h in (hq, hk, hk))
        o, y = dev.put(np.zeros((T, hq * d), np.float32)), dev.put(np.zeros((T, hid), np.float32))
        got = []
        for first, last in ((0, T - 2), (T - 2, T - 1), (T - 1, T)):
            S = last - first
            dl, d0 = dev.put(np.array([last], np.int32)), dev.put(np.array([0, S], np.int32))
            moe.matmul_fp8_dev_multi([q.ptr, k.ptr, v.ptr], dx.ptr + first * hid * 4, S, hid,
                                     [hq * d, hk * d, hk * d], keys[:3])
            batch = attn.Batch(dl.ptr, dt.ptr, 1, S, 4, row0=None if S == 1 else d0.ptr)
            attn.append(cache, batch, "f32", q.ptr, k.ptr, v.ptr, q.ptr, hq, rot)
            size = attn.work_bytes(cache, batch, hq)
            work = dev.put(np.zeros(size, np.uint8))
            (attn.decode if S == 1 else attn.prompt)(cache, batch, "f32", q.ptr, o.ptr, hq, d ** -0.5, work.ptr, size)
            moe.matmul_fp8_dev(y.ptr, o.ptr, S, hq * d, hid, keys[3])
            assert _lib.hip().colizig_hip_sync() == 0
            got.append(y.download(np.empty((T, hid), np.float32))[:S].copy())
        got = np.concatenate(got)
        X = x.astype(np.float64)
        Q, K, V = ((X @ m.T).reshape(T, -1, d) for m in mats[:3])
        t = rope.astype(np.float64)[:T, None]

        def turn(z, w):
            z = z / np.sqrt((z * z).mean(-1, keepdims=True) + 1e-6) * w.astype(np.float64)
            a, b, c, s = z[..., :32], z[..., 32:], t[..., :32], t[..., 32:]
            return np.concatenate([a * c - b * s, b * c + a * s], -1)

        Q, K = turn(Q, norm[0]), turn(K, norm[1])
        out = np.zeros((T, hq, d))
        for h in range(hq):
            a = Q[:, h] @ K[:, h // 4].T * d ** -0.5
            a[np.triu_indices(T, 1)] = -np.inf
            p = np.exp(a - a.max(1, keepdims=True))
            out[:, h] = (p / p.sum(1, keepdims=True)) @ V[:, h // 4]
        ref = out.reshape(T, -1) @ mats[3].T
        err = np.linalg.norm(got - ref, axis=1) / np.linalg.norm(ref, axis=1)
        say(f"  rel L2 {err.max():.2e}")
        assert err.max() < 2e-5
    finally:
        moe.set_vram_budget(0)
