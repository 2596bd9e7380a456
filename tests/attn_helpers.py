"""Problems for the attention tests: packed sequences over a shuffled paged
cache whose unused slots hold NaN, and the operators in 64 bits with bounds on
what rounding may do to each result (not collected as tests).

Rounding: a step to bf16 is off by at most 2^-8 of the value, to f32 2^-24, to
E4M3 2^-4 (2^-10 of the scale below 2^-6 scales)."""
from __future__ import annotations

import numpy as np

from colizig_amd import attn, moe
from tests.helpers import e4m3_f64

U32, U16, U8 = 2.0 ** -24, 2.0 ** -8, 2.0 ** -4
NP = {"f32": np.float32, "bf16": np.uint16, "e4m3": np.uint8}
NAN = {"f32": np.float32(np.nan), "bf16": np.uint16(0x7FC1), "e4m3": np.uint8(0x7F)}
_E4M3 = e4m3_f64(np.arange(256))


def bf16_bits(x) -> np.ndarray:
    """f32 -> nearest BF16 bits (ties to even)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(np.asarray(x, np.float32)), np.uint16(0x7FC0), r)


def e4m3_bits(x) -> np.ndarray:
    """Nearest E4M3 byte of finite x, saturating; ties to the even one."""
    x = np.asarray(x, np.float64)
    grid = _E4M3[:127]  # 0 .. 448, rising; byte = index
    a = np.minimum(np.abs(x), 448.0)
    hi = np.clip(np.searchsorted(grid, a), 1, 126)
    up = (grid[hi] - a < a - grid[hi - 1]) | ((grid[hi] - a == a - grid[hi - 1]) & (hi % 2 == 0))
    b = np.where(a <= 0, 0, np.where(up, hi, hi - 1)).astype(np.uint8)
    return np.where(x < 0, b | 0x80, b).astype(np.uint8)


def encode(x, t: str) -> np.ndarray:
    return {"f32": lambda v: np.asarray(v, np.float32), "bf16": bf16_bits, "e4m3": e4m3_bits}[t](x)


def decode(b, t: str) -> np.ndarray:
    if t == "f32":
        return np.asarray(b, np.float64)
    if t == "bf16":
        return (np.asarray(b).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return _E4M3[b]


class Dev:
    """Device copies of host arrays, freed together."""

    def __init__(self):
        self.bufs = []

    def put(self, a: np.ndarray) -> moe.DeviceBuffer:
        a = np.ascontiguousarray(a)
        b = moe.DeviceBuffer(max(16, a.nbytes))
        if a.nbytes:
            b.upload(a)
        self.bufs.append(b)
        return b

    def free(self):
        for b in self.bufs:
            b.free()
        self.bufs = []


class Problem:
    """Sequences of new[b] rows on len[b] cached tokens.  `layout`: "heads"
    ([page][head][slot][dim]) or "slots" ([page][slot][head][dim]); `pad`:
    extra numbers between rows of q, k, v and out."""

    def __init__(self, rows, cache, heads, new, lens, page=16, layout="heads", pad=0, extra_rows=0, seed=0, theta=1e4,
                 dims=None, norm=True, q_scale=1.5):
        self.rows_t, self.cache_t, self.page, self.layout, self.pad = rows, cache, page, layout, pad
        self.hq, self.hk, self.d = heads
        self.new, self.len = list(new), list(lens)
        self.n, self.t = len(new), sum(new) + extra_rows
        rng = self.rng = np.random.default_rng(seed)
        need = [max(1, -(-v // page)) for v in lens]
        self.width, self.pages = max(need) + 1, sum(need) + 2
        ids = rng.permutation(self.pages)
        self.table = np.full((self.n, self.width), -1, np.int32)
        at = 0
        for b, c in enumerate(need):
            self.table[b, :c] = ids[at:at + c]
            at += c
        self.row0 = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.scale = (rng.uniform(0.01, 0.02, (2, self.hk)) if cache == "e4m3" else np.ones((2, self.hk))).astype(np.float32)
        shape = (self.pages, self.hk, page, self.d) if layout == "heads" else (self.pages, page, self.hk, self.d)
        self.shape = shape
        self.k, self.v = (np.full(shape, NAN[cache], NP[cache]) for _ in range(2))
        for b in range(self.n):
            for c, s in ((self.k, 0), (self.v, 1)):
                x = rng.normal(size=(self.len[b], self.hk, self.d))
                if cache == "e4m3":
                    x = x / self.scale[s][:, None]
                self.set(c, b, 0, encode(x, cache))
        self.q = self.row_tensor(self.hq, q_scale)
        self.kx, self.vx = self.row_tensor(self.hk, 2.0), self.row_tensor(self.hk, 1.0)
        self.dims = self.d if dims is None else dims
        self.rope = attn.rope_table(max(self.len) + 1, self.dims, theta) if self.dims else None
        self.q_norm, self.k_norm = ((1 + 0.1 * rng.normal(size=(2, self.d))).astype(np.float32) if norm else (None, None))
        self.eps = 1e-6

    def row_tensor(self, heads, std):
        return encode(self.rng.normal(size=(self.t, heads * self.d + self.pad)) * std, self.rows_t)

    def where(self, b, pos):
        pos = np.asarray(pos)
        return self.table[b, pos // self.page], pos % self.page

    def set(self, c, b, first, x):
        """Tokens first.. of sequence b in cache array c: x [tokens][heads][dim]."""
        p, s = self.where(b, np.arange(first, first + len(x)))
        if self.layout == "heads":
            c[p, :, s] = x
        else:
            c[p, s] = x

    def get(self, c, b, length):
        p, s = self.where(b, np.arange(length))
        return c[p, :, s] if self.layout == "heads" else c[p, s]

    # -- on the device --
    def strides(self):
        d, hk, pg = self.d, self.hk, self.page
        return (0, 0, 0) if self.layout == "heads" else (pg * hk * d, d, hk * d)

    def upload(self, dev: Dev, decode_form=False):
        self.dk, self.dv = dev.put(self.k), dev.put(self.v)
        sc = dev.put(self.scale[0]), dev.put(self.scale[1])
        e = self.cache_t == "e4m3"
        self.cache = attn.KvCache(self.dk.ptr, self.dv.ptr, self.pages, self.page, self.hk, self.d, self.cache_t,
                                  k_scale=sc[0].ptr if e else None, v_scale=sc[1].ptr if e else None,
                                  strides=self.strides())
        self.dlen, self.dtable = dev.put(np.array(self.len, np.int32)), dev.put(self.table)
        self.drow0 = dev.put(self.row0)
        self.batch = attn.Batch(self.dlen.ptr, self.dtable.ptr, self.n, self.t, self.width,
                                row0=None if decode_form else self.drow0.ptr)
        self.dq = dev.put(self.q)
        self.out0 = np.full((self.t, self.hq * self.d + self.pad), NAN[self.rows_t], NP[self.rows_t])
        self.dout = dev.put(self.out0)

    def row_stride(self, heads):
        return heads * self.d + self.pad

    def attend(self, dev: Dev, decode_form=False, scale=None, stream=None, launch=True):
        """Uploads and runs one attention call; the whole out tensor."""
        self.upload(dev, decode_form)
        self.scale_qk = self.d ** -0.5 if scale is None else scale
        size = attn.work_bytes(self.cache, self.batch, self.hq)
        assert size > 0
        self.work = dev.put(np.full(size, 0xFF, np.uint8))
        self.call = lambda st=None: (attn.decode if decode_form else attn.prompt)(
            self.cache, self.batch, self.rows_t, self.dq.ptr, self.dout.ptr, self.hq, self.scale_qk, self.work.ptr, size,
            strides=(self.row_stride(self.hq),) * 2, stream=st)
        if launch:
            self.call(stream)
            return self.fetch()

    def fetch(self):
        from colizig_amd import _lib
        rc = _lib.hip().colizig_hip_sync()
        assert rc == 0, (rc, _lib.last_error())
        return self.dout.download(np.empty_like(self.out0))

    # -- in 64 bits --
    def reference(self, rows=None):
        """(out, bound) [t][hq][d] in 64 bits: NaN rows are not written.
        `rows`: only these (others come back NaN)."""
        out = np.full((self.t, self.hq, self.d), np.nan)
        bound = np.zeros_like(out)
        q = decode(self.q[:, :self.hq * self.d].reshape(self.t, self.hq, self.d), self.rows_t)
        g = self.hq // self.hk
        for b in range(self.n):
            L = self.len[b]
            k = decode(self.get(self.k, b, L), self.cache_t) * self.scale[0][:, None].astype(np.float64)
            v = decode(self.get(self.v, b, L), self.cache_t) * self.scale[1][:, None].astype(np.float64)
            for i in range(self.new[b]):
                r = self.row0[b] + i
                if rows is not None and r not in rows:
                    continue
                n = L - self.new[b] + i + 1
                if n <= 0:
                    out[r] = 0
                    continue
                kk, vv = np.repeat(k[:n], g, 1), np.repeat(v[:n], g, 1)
                s = np.einsum("hd,jhd->hj", q[r], kk) * self.scale_qk
                a = np.einsum("hd,jhd->hj", np.abs(q[r]), np.abs(kk)).max(1) * abs(self.scale_qk)
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                out[r] = np.einsum("hj,jhd->hd", p, vv)
                # a score is off by its products' and sums' roundings (d + 16 of them on sums of at most a), by the
                # scale's and the exponent's argument (8 on 2 a); a weight by that, the exponential's few steps and a
                # rescaling a tile; sums over n keys, numerator and denominator, by n + 16 steps each at most
                ds = ((self.d + 16) + 16) * U32 * a
                e = 2 * (ds + 16 * U32) + 2 * (n + 16) * U32
                if self.rows_t == "bf16":
                    e = e + 2 * U16  # the weights' rounding for their products, and the denominator's
                bound[r] = e[:, None] * np.einsum("hj,jhd->hd", p, np.abs(vv))
        bound += (U16 if self.rows_t == "bf16" else 4 * U32) * np.abs(np.nan_to_num(out)) * 1.01 + 1e-37
        return out, bound

    def check(self, got, rows=None, label=""):
        """`got` (the whole out tensor) against the reference; padding columns and rows behind the last untouched."""
        ref, bound = self.reference(rows)
        last = self.row0[-1]
        w = self.hq * self.d
        bits = lambda a: np.ascontiguousarray(a).view(np.uint8)
        assert np.array_equal(bits(got[last:]), bits(self.out0[last:])), "rows behind the last sequence"
        if self.pad:
            assert np.array_equal(bits(got[:, w:]), bits(self.out0[:, w:])), "between rows"
        val = decode(got[:last, :w].reshape(last, self.hq, self.d), self.rows_t)
        sel = np.arange(last) if rows is None else np.array(sorted(rows))
        d = np.abs(val[sel] - ref[sel])
        ok = d <= bound[sel]
        worst = np.nanmax(d / bound[sel]) if d.size else 0.0
        print(f"  {label} rel L2 {np.linalg.norm(val[sel] - ref[sel]) / max(np.linalg.norm(ref[sel]), 1e-30):.2e}, "
              f"worst {worst:.3f} of its bound", flush=True)
        assert ok.all(), (label, np.argwhere(~ok)[:5], val[sel][~ok][:5], ref[sel][~ok][:5])
