"""The attention operators between a layer's q, k, v and o projections, as
cases that can be timed and checked: new keys and values (normalised and
rotated) going into a paged cache, one new token per sequence attending over
that cache, and a prompt's or a prompt chunk's tokens attending causally.

Where `own` is false, `run` computes them in plain torch operations in 32
bits; where it is true, it makes the calls of colizig_amd.attn that a program
makes.  Both work on the same state.

The benchmark's attention shape is 32 query heads and 4 key heads of 128
(q rows 4096 wide, k and v rows 512); the other layouts are generic: one key
head per query head, one key head for all, and heads of 64 and 256.
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e6
F8_MAX = 448.0

_ROWS = {"f32": torch.float32, "bf16": torch.bfloat16}
_CACHE = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
_SIZE = {"f32": 4, "bf16": 2, "e4m3": 1}


def _case(op, rows, cache, heads, n, new, past, page=64, ragged=False, **more) -> dict:
    """heads: (query heads, key heads, head dimension); n sequences of `new`
    tokens each on top of `past` cached ones (upper ends where ragged)."""
    return dict(op=op, rows=rows, cache=cache, q_heads=heads[0], kv_heads=heads[1], dim=heads[2], n=n, new=new,
                past=past, page=page, ragged=ragged, **more)


BENCH = (32, 4, 128)


def listed() -> list[dict]:
    return [
        # the token just decoded goes into the cache: latency is all
        _case("append", "f32", "bf16", BENCH, 1, 1, 1021, name="append_1"),
        # a server's decode batch into an 8-bit cache
        _case("append", "f32", "e4m3", BENCH, 61, 1, 250, page=16, ragged=True, name="append_batch_e4m3"),
        # several prompts of different lengths at once
        _case("append", "bf16", "bf16", BENCH, 5, 4096, 0, ragged=True, name="append_prompts"),
        # one conversation, its next token: little to read, latency counts
        _case("decode", "f32", "bf16", BENCH, 1, 1, 576, name="decode_1_short"),
        # one very long document
        _case("decode", "f32", "bf16", BENCH, 1, 1, 131070, name="decode_1_long"),
        # a decode batch of conversations of very different lengths
        _case("decode", "bf16", "bf16", BENCH, 32, 1, 16000, ragged=True, name="decode_ragged"),
        # a large batch on an 8-bit cache
        _case("decode", "f32", "e4m3", BENCH, 128, 1, 8191, page=16, ragged=True, name="decode_batch_e4m3"),
        # a short prompt by itself, rows as the f32 projections give them
        _case("prompt", "f32", "bf16", BENCH, 1, 500, 0, name="prompt_short"),
        # a long prompt whose program works in bf16
        _case("prompt", "bf16", "bf16", BENCH, 1, 8192, 0, name="prompt_long_bf16"),
        # prompts of different lengths packed into one call, f32 rows
        _case("prompt", "f32", "bf16", BENCH, 7, 2311, 0, ragged=True, name="prompt_packed"),
        # the next chunk of a long prompt whose start is cached in 8 bits
        _case("prompt", "bf16", "e4m3", BENCH, 1, 777, 20000, name="prompt_chunk_e4m3"),
        # a draft of a few tokens checked against a long f32 cache
        _case("prompt", "f32", "f32", BENCH, 3, 6, 9000, page=32, ragged=True, name="prompt_draft_f32"),
    ]


_LAYOUTS = [BENCH, BENCH, (16, 2, 256), (40, 8, 128), (12, 12, 64), (8, 1, 128), (28, 4, 64)]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt"])
    rows, cache = rng.choice([("f32", "bf16"), ("bf16", "bf16"), ("f32", "e4m3"), ("bf16", "e4m3"), ("f32", "f32")])
    heads = rng.choice(_LAYOUTS)
    page = rng.choice([16, 32, 48, 64, 128])
    ragged = rng.random() < 0.7
    n = _log_int(rng, 1, 100)
    if op == "decode":
        # keys and values of all sequences: at most 2^29 bytes, about the largest listed decode case
        most = (1 << 28) // (n * heads[1] * heads[2] * _SIZE[cache])
        return _case(op, rows, cache, heads, n, 1, _log_int(rng, 1, max(2, min(131070, most))), page, ragged)
    if op == "append":
        if rng.random() < 0.4:
            return _case(op, rows, cache, heads, n, 1, _log_int(rng, 1, 600), page, ragged)
        new = _log_int(rng, 2, 4096)
        n = max(1, min(n, 10000 // (_SIZE[rows] * new)))
        return _case(op, rows, cache, heads, n, new, rng.choice([0, 0, _log_int(rng, 1, 500)]), page, ragged)
    new = _log_int(rng, 2, 8191)
    past = rng.choice([0, 0, _log_int(rng, 1, 20000)])
    pairs = (1 << 37) // (heads[0] * heads[2])  # new x keys over all sequences: the longest listed prompt's products
    while new * (new + past) > pairs:
        new, past = max(2, new * 3 // 4), past * 3 // 4
    n = max(1, min(n, pairs // (new * (new + past))))
    return _case(op, rows, cache, heads, n, new, past, page, ragged)


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and cached tokens (new ones included) of each sequence."""
    n, new, past = case["n"], case["new"], case["past"]
    if not case["ragged"]:
        return [new] * n, [new + past] * n
    rng = random.Random("%d %d %d %d" % (n, new, past, case["page"]))
    qs = [new] + [rng.randint(max(1, new // 16), new) for _ in range(n - 1)]
    ps = [past] + [rng.randint(past // 16, past) for _ in range(n - 1)]
    return qs, [q + p for q, p in zip(qs, ps)]


# ---- inputs -------------------------------------------------------------------
def _inputs(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, cache = _ROWS[case["rows"]], _CACHE[case["cache"]]
    hq, hk, d, page, n = case["q_heads"], case["kv_heads"], case["dim"], case["page"], case["n"]
    qs, ls = _lengths(case)
    t = sum(qs)
    need = [-(-v // page) for v in ls]
    pages, width = sum(need) + 3, max(need)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)  # pages are handed out in any order
    table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    scale = 0.01 + 0.01 * torch.rand(2, hk, generator=g, device="cuda")
    s = dict(table=table, k_scale=scale[0], v_scale=scale[1], rows=t, width=width, pages=pages, n=n)
    for name, sc in (("k", scale[0]), ("v", scale[1])):
        c = torch.empty(pages, hk, page, d, dtype=cache, device="cuda")
        for i in range(0, pages, 1024):  # bounds the f32 copy
            x = randn(min(1024, pages - i), hk, page, d)
            c[i:i + 1024] = (x / sc[:, None, None]).clamp(-F8_MAX, F8_MAX).to(cache) if case["cache"] == "e4m3" else x.to(cache)
        s[name + "_cache"] = c
    s["row0"] = torch.tensor([sum(qs[:b]) for b in range(n + 1)], dtype=torch.int32, device="cuda")
    s["len"] = torch.tensor(ls, dtype=torch.int32, device="cuda")
    s["q"] = (1.5 * randn(t, hq, d)).to(rows)
    s["most_new"], s["most_len"] = max(qs), max(ls)
    if case["op"] == "append":
        s["k"], s["v"] = (2 * randn(t, hk, d)).to(rows), randn(t, hk, d).to(rows)
        s["q_norm"], s["k_norm"] = 1 + 0.1 * randn(d), 1 + 0.1 * randn(d)
        ang = _angles(max(ls), d, "cuda")
        s["rope"] = torch.cat([ang.cos(), ang.sin()], 1).float()
    s["out"] = torch.zeros_like(s["q"])
    return s


def _angles(positions: int, dims: int, device) -> torch.Tensor:
    """Rotation angles [positions][dims / 2] in 64 bits."""
    inv = THETA ** (-torch.arange(0, dims, 2, dtype=torch.float64, device=device) / dims)
    return torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv


_stream = None


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        global _stream
        from colizig_amd import attn, moe
        if _stream is None:
            moe.init()
            _stream = torch.cuda.Stream()
        e4m3 = case["cache"] == "e4m3"
        s["cache"] = attn.KvCache(s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), s["pages"], case["page"],
                                  case["kv_heads"], case["dim"], case["cache"],
                                  k_scale=s["k_scale"].data_ptr() if e4m3 else None,
                                  v_scale=s["v_scale"].data_ptr() if e4m3 else None)
        decode = case["op"] == "decode"
        s["batch"] = attn.Batch(s["len"].data_ptr(), s["table"].data_ptr(), s["n"], s["rows"], s["width"],
                                row0=None if decode else s["row0"].data_ptr())
        if case["op"] == "append":
            s["rotation"] = attn.Rotation(s["rope"].data_ptr(), s["rope"].shape[0], case["dim"],
                                          q_norm=s["q_norm"].data_ptr(), k_norm=s["k_norm"].data_ptr(), eps=EPS)
        else:
            size = attn.work_bytes(s["cache"], s["batch"], case["q_heads"])
            s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
    return s


def run(s: dict):
    case = s["case"]
    if own:
        from colizig_amd import attn
        st = _stream.cuda_stream
        if case["op"] == "append":
            attn.append(s["cache"], s["batch"], case["rows"], s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                        s["out"].data_ptr(), case["q_heads"], s["rotation"], stream=st)
            return dict(q=s["out"], k=s["k_cache"], v=s["v_cache"])
        call = attn.decode if case["op"] == "decode" else attn.prompt
        call(s["cache"], s["batch"], case["rows"], s["q"].data_ptr(), s["out"].data_ptr(), case["q_heads"],
             case["dim"] ** -0.5, s["work"].data_ptr(), s["work"].numel(), stream=st)
        return s["out"]
    return _append(s) if case["op"] == "append" else _attend(s)


# ---- the plain form -------------------------------------------------------------
def _places(s: dict, page: int):
    """Sequence, position and cache place (page, slot) of every row."""
    r = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(s["row0"][1:].contiguous().long(), r, right=True)
    pos = (s["len"][b] - (s["row0"][b + 1] - s["row0"][b])).long() + r - s["row0"][b]
    return b, pos, s["table"][b, pos // page].long(), pos % page


def _turned(x, w, rope, pos):
    """Rows [T][heads][d] normalised, weighted, and rotated in halves."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    h = x.shape[-1] // 2
    c, sn = rope[pos, None, :h], rope[pos, None, h:]
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _held(x, scale, dtype):
    """Rows [T][heads][d] as the cache holds them."""
    if dtype == torch.float8_e4m3fn:
        return (x / scale[:, None]).clamp(-F8_MAX, F8_MAX).to(dtype)
    return x.to(dtype)


def _bits(t):
    """E4M3 values as their bytes: torch indexes those."""
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _append(s: dict):
    kc, vc = s["k_cache"], s["v_cache"]
    _, pos, page, slot = _places(s, s["case"]["page"])
    k = _held(_turned(s["k"], s["k_norm"], s["rope"], pos), s["k_scale"], kc.dtype)
    v = _held(s["v"].float(), s["v_scale"], vc.dtype)
    _bits(kc)[page, :, slot] = _bits(k)
    _bits(vc)[page, :, slot] = _bits(v)
    s["out"].copy_(_turned(s["q"], s["q_norm"], s["rope"], pos))
    return dict(q=s["out"], k=kc, v=vc)


def _gathered(cache, table, scale, length: int):
    """A cache's first `length` keys (or values) of every sequence as f32 [n][heads][length][d]."""
    x = _bits(cache)[table.long()].view(cache.dtype).float()          # [n][pages][heads][page][d]
    if cache.dtype == torch.float8_e4m3fn:
        x = x * scale[:, None, None]
    n, w, h, p, d = x.shape
    return x.transpose(1, 2).reshape(n, h, w * p, d)[:, :, :length]


def _attend(s: dict):
    case = s["case"]
    hq, hk, d, n = case["q_heads"], case["kv_heads"], case["dim"], s["n"]
    group, most, length = hq // hk, s["most_new"], s["most_len"]
    new = s["row0"][1:] - s["row0"][:-1]
    i = torch.arange(most, device="cuda")
    there = i < new[:, None]                                          # [n][most]
    row = torch.where(there, s["row0"][:-1, None] + i, 0)
    sees = torch.where(there, (s["len"] - new)[:, None] + i + 1, 0)   # keys each row sees
    q = s["q"].float()[row].view(n, most, hk, group, d).permute(0, 2, 1, 3, 4).reshape(n, hk, most * group, d)
    k = _gathered(s["k_cache"], s["table"], s["k_scale"], length)
    v = _gathered(s["v_cache"], s["table"], s["v_scale"], length)
    key = torch.arange(length, device="cuda")
    # slots behind a sequence's end hold anything: no key there counts
    v = v.masked_fill((key >= s["len"][:, None])[:, None, :, None], 0.0)
    a = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(d ** -0.5)
    dark = (key >= sees[:, :, None]).repeat_interleave(group, 1)[:, None]
    a.masked_fill_(dark, -math.inf)
    a.sub_(a.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    o = torch.matmul(a, v.contiguous()) / a.sum(-1, keepdim=True).clamp(min=1e-38)
    o = o.view(n, hk, most, group, d).permute(0, 2, 1, 3, 4).reshape(n, most, hq, d)
    s["out"][row[there].long()] = o[there].to(s["out"].dtype)
    return s["out"]


# ---- what a pass cannot do without ----------------------------------------------
def work(case: dict) -> dict:
    qs, ls = _lengths(case)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    r, c, t = _SIZE[case["rows"]], _SIZE[case["cache"]], sum(qs)
    if case["op"] == "append":
        # a position's cosines and sines are read once, however many sequences are there
        return dict(bytes=t * d * (2 * hq * r + 2 * hk * (r + c)) + 4 * d * max(qs) + 8 * d,
                    flops=t * d * (8 * hq + 8 * hk))
    pairs = sum(q * (l - q) + q * (q + 1) // 2 for q, l in zip(qs, ls))
    return dict(bytes=2 * t * hq * d * r + 2 * sum(ls) * hk * d * c, flops=4 * pairs * hq * d)


# ---- the same in 64 bits ----------------------------------------------------------
def _slots(s: dict, case: dict, b: int, first: int, last: int):
    at = torch.arange(first, last, device="cuda")
    return s["table"][b].long()[at // case["page"]], at % case["page"]


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    qs, ls = _lengths(case)
    hk, d = case["kv_heads"], case["dim"]
    group = case["q_heads"] // hk
    e4m3 = case["cache"] == "e4m3"
    if case["op"] == "append":
        return _exact_append(s, case, qs, ls)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    r0 = 0
    for b, (new, length) in enumerate(zip(qs, ls)):
        page, slot = _slots(s, case, b, 0, length)
        hidden = torch.arange(length, device="cuda") > torch.arange(length - new, length, device="cuda")[:, None]
        for h in range(hk):
            k = _bits(s["k_cache"])[page, h, slot].view(s["k_cache"].dtype).double()
            v = _bits(s["v_cache"])[page, h, slot].view(s["v_cache"].dtype).double()
            if e4m3:
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            kt = k.T.contiguous()
            for x in range(h * group, (h + 1) * group):
                a = (s["q"][r0:r0 + new, x].double() @ kt) / math.sqrt(d)
                out[r0:r0 + new, x] = torch.softmax(a.masked_fill(hidden, -math.inf), 1) @ v
        r0 += new
    return out


def _exact_append(s, case, qs, ls):
    """Cache and query rows: what rounding to the cache's type leaves is what the cache holds."""
    d, h = case["dim"], case["dim"] // 2
    ang = s["rope"].double()  # the table is an input, in f32

    def turned(x, w, pos):
        x = x.double()
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + EPS) * w.double()
        z = torch.complex(x[..., :h], x[..., h:]) * torch.complex(ang[pos, :h], ang[pos, h:])[:, None]
        return torch.cat([z.real, z.imag], -1)

    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    r0 = 0
    for b, (new, length) in enumerate(zip(qs, ls)):
        pos = torch.arange(length - new, length, device="cuda")
        page, slot = _slots(s, case, b, length - new, length)
        rows = slice(r0, r0 + new)
        q[rows] = turned(s["q"][rows], s["q_norm"], pos)
        k, v = turned(s["k"][rows], s["k_norm"], pos), s["v"][rows].double()
        if case["cache"] == "e4m3":
            k, v = _to_e4m3(k / s["k_scale"].double()[:, None]), _to_e4m3(v / s["v_scale"].double()[:, None])
        kc[page, :, slot], vc[page, :, slot] = k, v
        r0 += new
    return dict(q=q, k=kc, v=vc)


def _to_e4m3(x):
    """Nearest E4M3 value (ties to even), saturating, in 64 bits: 3 bits after the first, steps of 2^-9 below 2^-6."""
    x = x.clamp(-F8_MAX, F8_MAX)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step
