// cz_attn.hip - attention over a paged key-value cache: new keys and values into
// the cache, one new token per sequence, and prompts.
//
// A sequence's new tokens are the last of its len tokens: row i of new rows sits
// at position len - new + i and sees the positions up to its own.
#include "cz_attn.h"

#include <algorithm>
#include <type_traits>

namespace cz {
namespace {

__device__ __forceinline__ void flag(uint32_t *err, AttnError what) {
    __hip_atomic_store(err + what, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// What saturates to an E4M3 number: rounding to nearest follows.  A NaN stays one.
__device__ __forceinline__ float e4m3_range(float x) { return x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f); }

template <uint32_t T>
__device__ __forceinline__ float load1(const void *p, uint64_t i) {
    if constexpr (T == kF32) return ((const float *)p)[i];
    if constexpr (T == kBF16) return __uint_as_float((uint32_t)((const uint16_t *)p)[i] << 16);
    if constexpr (T == kE4M3) return __builtin_amdgcn_cvt_f32_fp8(((const uint8_t *)p)[i], 0);
}
// Rows and length of sequence b, checked: 0 <= r0 <= r1 <= rows, 0 <= len <=
// max_pages * page_size.  What is outside is flagged and cut.
struct Seq {
    int32_t r0, nq, len;
};
__device__ __forceinline__ Seq sequence(const AttnCache &c, uint32_t b) {
    Seq s;
    int32_t r0 = c.row0 ? c.row0[b] : (int32_t)b, r1 = c.row0 ? c.row0[b + 1] : (int32_t)b + 1, len = c.len[b];
    const int32_t most = (int32_t)(c.max_pages * c.page_size);
    if (r0 < 0 || r1 < r0 || r1 > (int32_t)c.rows || len < 0 || len > most) {
        flag(c.err, kAttnBadLength);
        r0 = min(max(r0, 0), (int32_t)c.rows);
        r1 = min(max(r1, r0), (int32_t)c.rows);
        len = min(max(len, 0), most);
    }
    s.r0 = r0;
    s.nq = r1 - r0;
    s.len = len;
    return s;
}


typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
#define CZ_LDS __attribute__((address_space(3)))

// bf16 terms of a number: three hold every bit of an f32, each the upper half of
// what the ones before leave; bf16 and E4M3 numbers are one.
template <uint32_t T>
constexpr int kTerms = T == kF32 ? 3 : 1;
template <uint32_t T>
constexpr int kSize = T == kF32 ? 4 : T == kBF16 ? 2 : 1;

// x in N terms: one or two round to nearest (8 and 16 bits).  In three, infinities have no lower terms (inf - inf);
// a NaN stays one in some term.
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf8 (&t)[N]) {
    if constexpr (N == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[0][i] = (__bf16)x[i];
    } else if constexpr (N == 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            t[0][i] = (__bf16)x[i];
            t[1][i] = (__bf16)(x[i] - (float)t[0][i]);
        }
    } else {
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = __builtin_amdgcn_perm(__float_as_uint(r[2 * i + 1]), __float_as_uint(r[2 * i]), 0x07060302u);
            t[n] = __builtin_bit_cast(bf8, w);
            if (n + 1 < N)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float lo = r[i] - __uint_as_float(__float_as_uint(r[i]) & 0xffff0000u);
                    r[i] = __builtin_isinf(r[i]) ? 0.0f : lo;
                }
        }
    }
}

__device__ __forceinline__ bf8 e4m3x8(uint32_t a, uint32_t b) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    const bf2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)a, 1.0f, false);
    const bf2 p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)a, 1.0f, true);
    const bf2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b, 1.0f, false);
    const bf2 p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)b, 1.0f, true);
    return bf8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// 8 numbers of type T in memory order, raw and as terms.
template <uint32_t T>
struct Eight;
template <>
struct Eight<kF32> {
    u32x4 a, b;
    __device__ __forceinline__ void load(const uint8_t *p) {
        a = *(const u32x4 *)p;
        b = *(const u32x4 *)(p + 16);
    }
    __device__ __forceinline__ void load_once(const uint8_t *p) {
        a = __builtin_nontemporal_load((const u32x4 *)p);
        b = __builtin_nontemporal_load((const u32x4 *)(p + 16));
    }
    __device__ __forceinline__ void zero() { a = b = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = __uint_as_float(a[i]);
            x[4 + i] = __uint_as_float(b[i]);
        }
    }
    __device__ __forceinline__ void terms(bf8 (&t)[3]) const {
        float x[8];
        floats(x);
        split8<3>(x, t);
    }
};
template <>
struct Eight<kBF16> {
    u32x4 a;
    __device__ __forceinline__ void load(const uint8_t *p) { a = *(const u32x4 *)p; }
    __device__ __forceinline__ void load_once(const uint8_t *p) { a = __builtin_nontemporal_load((const u32x4 *)p); }
    __device__ __forceinline__ void zero() { a = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(a[i] << 16);
            x[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void terms(bf8 (&t)[1]) const { t[0] = __builtin_bit_cast(bf8, a); }
};

// threadIdx.x as a value that the compiler knows nothing of: what rare or final code
// derives from it is worked out there, not held in registers through the loops.
__device__ __forceinline__ uint32_t thread_id() {
    uint32_t t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// Numbers of type T in a word that are not finite become 0; whether there were any.
template <uint32_t T>
__device__ __forceinline__ bool clean(uint32_t &w) {
    uint32_t bad;
    if constexpr (T == kF32) {
        bad = (w & 0x7f800000u) == 0x7f800000u ? ~0u : 0u;
    } else if constexpr (T == kBF16) {
        bad = ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
    } else {
        // 0x7f and 0xff: the sum carries into the sign bit where the low bits are all set
        bad = ((w & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u) >> 7;
        bad *= 0xffu;
    }
    w &= ~bad;
    return bad != 0;
}

// What a lane loads at a time: 8 numbers, of an E4M3 cache 16 so that it is 16 bytes.
// load_once: of data that nobody reads again (keeps the caches for what is; 533 MB of
// BF16 keys and values of one token go from 101 to 92 us with it).
template <uint32_t T>
struct Piece {
    static constexpr int N = 8;
    Eight<T> e;
    __device__ __forceinline__ void load(const uint8_t *p) { e.load(p); }
    __device__ __forceinline__ void load_once(const uint8_t *p) { e.load_once(p); }
    __device__ __forceinline__ void zero() { e.zero(); }
    __device__ __forceinline__ bool clean() {
        bool any = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w = e.a[i];
            any |= cz::clean<T>(w);
            e.a[i] = w;
            if constexpr (T == kF32) {
                w = e.b[i];
                any |= cz::clean<T>(w);
                e.b[i] = w;
            }
        }
        return any;
    }
    __device__ __forceinline__ void terms(int, bf8 (&t)[kTerms<T>]) const { e.terms(t); }
};
template <>
struct Piece<kE4M3> {
    static constexpr int N = 16;
    u32x4 a;
    __device__ __forceinline__ void load(const uint8_t *p) { a = *(const u32x4 *)p; }
    __device__ __forceinline__ void load_once(const uint8_t *p) { a = __builtin_nontemporal_load((const u32x4 *)p); }
    __device__ __forceinline__ void zero() { a = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ bool clean() {
        bool any = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w = a[i];
            any |= cz::clean<kE4M3>(w);
            a[i] = w;
        }
        return any;
    }
    __device__ __forceinline__ void terms(int half, bf8 (&t)[1]) const { t[0] = e4m3x8(a[2 * half], a[2 * half + 1]); }
};

// 8 numbers rounded to type T, 16-byte aligned (E4M3: 8).
template <uint32_t T>
__device__ __forceinline__ void store8(uint8_t *p, const float (&y)[8]) {
    if constexpr (T == kF32) {
        *(f32x4 *)p = f32x4{y[0], y[1], y[2], y[3]};
        *(f32x4 *)(p + 16) = f32x4{y[4], y[5], y[6], y[7]};
    } else if constexpr (T == kBF16) {
        bf8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (__bf16)y[i];
        *(bf8 *)p = v;
    } else {
        u32x2 w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float *x = y + 4 * i;
            int v = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(x[0]), e4m3_range(x[1]), 0, false);
            w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(x[2]), e4m3_range(x[3]), v, true);
        }
        *(u32x2 *)p = w;
    }
}

__device__ __forceinline__ void floats8(const float *p, float (&x)[8]) {
    const f32x4 a = *(const f32x4 *)p, b = *(const f32x4 *)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = a[i];
        x[4 + i] = b[i];
    }
}

// ---- append -------------------------------------------------------------------
// Head vectors (the query's into q_out, then the keys, then the values) over groups
// of D / 8 lanes, 8 neighbouring numbers a lane, so that a vector moves in 16-byte
// pieces.  A norm's sum goes over the group's lanes; a rotation's other half is
// dims / 16 lanes away.  A workgroup takes TB rows: the three lookups one after the
// other (sequence, length, page and angles) cost it some microseconds whatever it
// moves, and a group's angles and weights serve all its vectors of the row.  Below
// kAppendBlockRows rows a workgroup takes one pass over one row, and a row is spread
// over blockIdx.y.
//
// Bound: HBM for prompts, those look-ups for few rows.  14,588 BF16 rows of 32 + 2 x 4
// heads of 128 (301 MB) 69 us, 4.4 TB/s, where a large copy moves 5.2; one row 3.5 us.
// Eight rows a workgroup 76 us; a workgroup a row with its passes one after the other
// 164 us.
template <uint32_t R, uint32_t C, int D, int TB>
__global__ __launch_bounds__(256) void k_append(AppendArgs A) {
    constexpr uint32_t LV = D / 8, GROUPS = 256 / LV, STEP = GROUPS / TB, UNROLL = TB == 1 ? 1 : 4;
    const uint32_t lane = threadIdx.x & 63, gl = threadIdx.x % LV, gv = threadIdx.x / LV;
    const uint32_t heads = A.q_heads + 2 * A.c.kv_heads, t0 = blockIdx.x * TB, t = t0 + gv % TB;
    const uint32_t xs = gv / TB + blockIdx.y * STEP, xstep = STEP * gridDim.y;
    Eight<R> in[UNROLL];
    auto load = [&](uint32_t x0) {
#pragma unroll
        for (uint32_t u = 0; u < UNROLL; ++u) {
            const uint32_t x = x0 + u * xstep;
            in[u].zero();
            if (x >= heads || t >= A.c.rows) continue;
            const bool isq = x < A.q_heads, isk = x < A.q_heads + A.c.kv_heads;
            const uint32_t h = isq ? x : isk ? x - A.q_heads : x - A.q_heads - A.c.kv_heads;
            const uint64_t at = (uint64_t)t * (isq ? A.q_stride : isk ? A.k_stride : A.v_stride) + h * D + gl * 8;
            in[u].load_once((const uint8_t *)(isq ? A.q : isk ? A.k : A.v) + at * kSize<R>);
        }
    };
    load(xs);
    // the row's sequence: as many as end at or before it
    uint32_t b = 0;
    if (A.c.row0) {
        for (uint32_t b0 = 0; b0 < A.c.n; b0 += 64) {
            const int32_t e = b0 + lane < A.c.n ? A.c.row0[b0 + lane + 1] : 0x7fffffff;
#pragma unroll
            for (uint32_t i = 0; i < TB; ++i) {
                const uint32_t k = __popcll(__ballot(e <= (int32_t)(t0 + i)));
                b += gv % TB == i ? k : 0;
            }
        }
    } else {
        b = t;
    }
    Seq s{0, 0, 0};
    if (b < A.c.n && t < A.c.rows) s = sequence(A.c, b);
    const int32_t pos = s.len - s.nq + ((int32_t)t - s.r0);
    bool here = pos >= 0 && (int32_t)t >= s.r0 && (int32_t)t < s.r0 + s.nq;
    if (here && A.rope && (uint32_t)pos >= A.positions) {
        flag(A.c.err, kAttnBadPosition);
        here = false;
    }
    bool paged = false;
    uint64_t to = 0;
    const uint32_t half = A.dims / 2, d0 = gl * 8;
    const bool turns = A.rope && d0 < A.dims, lower = d0 < half;
    float cs[8], sn[8], wq[8], wk[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        cs[i] = wq[i] = wk[i] = 1.0f;
        sn[i] = 0.0f;
    }
    if (here) {
        const uint32_t pi = (uint32_t)pos / A.c.page_size, page = (uint32_t)A.c.table[(uint64_t)b * A.c.max_pages + pi];
        // the lane's angles: numbers d < dims/2 turn with d + dims/2
        if (turns) {
            const float *p = A.rope + (uint64_t)pos * A.dims + (lower ? d0 : d0 - half);
            floats8(p, cs);
            floats8(p + half, sn);
            if (lower)
#pragma unroll
                for (int i = 0; i < 8; ++i) sn[i] = -sn[i];
        }
        paged = page < A.c.pages;
        if (!paged) flag(A.c.err, kAttnBadPage);
        to = page * A.c.page_stride + (pos - pi * A.c.page_size) * A.c.token_stride;
    }
    if (A.q_norm) floats8(A.q_norm + d0, wq);
    if (A.k_norm) floats8(A.k_norm + d0, wk);
    const int other = (int)((turns ? (lower ? lane + half / 8 : lane - half / 8) : lane) * 4);

    for (uint32_t x0 = xs; x0 < heads; x0 += UNROLL * xstep) {  // (the bound is over a group: its lanes stay together)
        if (x0 != xs) load(x0);
#pragma unroll
        for (uint32_t u = 0; u < UNROLL; ++u) {
            const uint32_t x = x0 + u * xstep;
            const bool isq = x < A.q_heads, isk = !isq && x < A.q_heads + A.c.kv_heads;
            float y[8];
            in[u].floats(y);
            if (isq ? A.q_norm != nullptr : isk && A.k_norm) {
                float ss = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(y[i], y[i], ss);
#pragma unroll
                for (int m = LV / 2; m; m >>= 1) ss += __shfl_xor(ss, m);
                const float r = __builtin_amdgcn_rsqf(__builtin_fmaf(ss, 1.0f / D, A.eps));
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = y[i] * r * (isq ? wq[i] : wk[i]);
            }
            if (A.rope && (isq || isk)) {
                float z[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    z[i] = __int_as_float(__builtin_amdgcn_ds_bpermute(other, __float_as_int(y[i])));
                if (turns)
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(z[i], sn[i], y[i] * cs[i]);
            }
            if (x >= heads || !here) continue;
            if (isq) {
                store8<R>((uint8_t *)A.q_out + ((uint64_t)t * A.q_out_stride + x * D + d0) * kSize<R>, y);
                continue;
            }
            if (!paged) continue;
            const uint32_t h = x - A.q_heads - (isk ? 0 : A.c.kv_heads);
            if (C == kE4M3 && (isk ? A.c.k_scale : A.c.v_scale)) {
                const float sc = (isk ? A.c.k_scale : A.c.v_scale)[h];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = y[i] / sc;
            }
            store8<C>((uint8_t *)(isk ? A.c.k : A.c.v) + (to + h * A.c.head_stride + d0) * kSize<C>, y);
        }
    }
}

// ---- attention ------------------------------------------------------------------
// Rows of a key head: row r of a sequence's tile list is token r / group, query
// head h * group + r % group, so the query heads of a key head share its loads.
//
// Both kernels work on S^T = K Q^T and O^T = V^T P^T: the scores' result layout
// (a lane holds one row and 4 keys in a run) is the second product's operand
// layout once its keys are counted in that order, so weights go from one matrix
// instruction to the next in registers; V's side of it, 4 keys of one number, is
// what the transposing LDS read gives.
//
// f32 accuracy on the bf16 matrix cores: an f32 is the sum of three bf16 numbers, so
// q and the weights of f32 rows are three terms each and every product is exact (an
// f32 cache's keys and values are three terms too, and of the nine products of two
// numbers the six above 2^-24 are taken); sums are f32.  Nearer to 64 bits than f32
// products and sums are: 3.6e-7 for 6.2e-7 over packed prompts.
// 8 query numbers as terms, negated where `flip` is the sign bit.
template <uint32_t R>
__device__ __forceinline__ void query8(const void *q, uint64_t at, uint32_t flip, bf8 (&t)[kTerms<R>]) {
    Eight<R> e;
    e.load((const uint8_t *)q + at * kSize<R>);
    if constexpr (R == kF32) {
        e.a ^= flip;
        e.b ^= flip;
    } else {
        e.a ^= flip | flip >> 16;
    }
    e.terms(t);
}

// The terms' products whose weight is above 2^-24 of the whole.
template <int NA, int NB, typename V, typename M>
__device__ __forceinline__ V product(const bf8 (&a)[NA], const bf8 (&b)[NB], V c, M &&mfma) {
    // the smallest first
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
        for (int i = 0; i < NA; ++i)
            if (s - i >= 0 && s - i < NB) c = mfma(a[i], b[s - i], c);
    return c;
}

// Where 16-byte piece `chunk` of bf16 row `key` sits in an LDS tile of D numbers a
// row: the pieces of a row are permuted by the key, so that what the LDS serves at
// once falls on different banks: 8 keys at one piece (a read of K), and 4 keys at 4
// pieces, or 8 at 2 (the transposing reads of V).  Keys 8 apart are permuted alike:
// one address serves both.
template <int D>
__device__ __forceinline__ uint32_t lds_at(uint32_t key, uint32_t chunk) {
    const uint32_t f = D == 64 ? (key & 2) << 1 | (key & 4) >> 1 : (key & 3) << 2 | (key & 4) >> 1;
    return key * (D * 2) + ((chunk ^ f) << 4);
}

// A sequence that is the same for the whole wave, in scalar registers.
__device__ __forceinline__ Seq uniform(const Seq &s) {
    return Seq{__builtin_amdgcn_readfirstlane(s.r0), __builtin_amdgcn_readfirstlane(s.nq),
               __builtin_amdgcn_readfirstlane(s.len)};
}

// Sums over the lanes up to each one.
template <typename T>
__device__ __forceinline__ T wave_scan(T x) {
    auto step = [&](auto ctrl, auto mask) {
        x += __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl(), mask(), 0xf, false));
    };
    step(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // from 1 lane below in a row of 16,
    step(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});  // 2,
    step(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});  // 4,
    step(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});  // 8,
    step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // rows 0 and 2 into 1 and 3,
    step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // the lower half into the upper
    return x;
}
template <typename T>
__device__ __forceinline__ T lane_of(T x, int lane) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}

// The scratch: a line for how the work was divided, then the parts' sums.
constexpr uint32_t kPlanFloats = 64;
constexpr uint32_t kWhole = 0xffffffffu;  // no parts

// One part of the work: keys of a row tile of a key head.
struct Item {
    uint32_t b, rt, h, part, parts, slot;
    int32_t r0, nq, len;
};

// A share of a call's work: all tiles' units of `unit` keys, in the order sequence,
// tile (the last first), key head, unit, dealt out evenly to `slots` workgroups
// whatever the lengths are; a tile that several of them share is joined from their
// sums.  slots = 0: a tile is one unit, and each workgroup takes one.
struct Place {
    uint32_t b, j, h, tiles, units, unit0;  // tile j of the sequence's, unit unit0 of its units
    Seq s;
    uint32_t start;  // number of the tile's first unit
};
template <int BM>
__device__ __forceinline__ uint32_t tiles_of(const Seq &s, uint32_t group) { return ((uint32_t)s.nq * group + BM - 1) / BM; }
__device__ __forceinline__ uint32_t units_of(const Seq &s, uint32_t unit, uint32_t slots) {
    return slots ? max(1u, ((uint32_t)s.len + unit - 1) / unit) : 1u;
}

// Unit idx * per (JOIN: tile idx), per being the share of a workgroup; JOIN: as the
// first workgroup left it at `plan`.
template <int BM, bool JOIN>
__device__ __forceinline__ bool find_place(const AttnCache &c, uint32_t group, uint32_t slots, uint32_t unit, uint32_t idx,
                                           uint32_t *plan, uint32_t *per, Place &p) {
    const uint32_t lane = threadIdx.x & 63;
    if (!JOIN && !slots && !c.row0) {  // a row and so many tiles for each sequence: nothing to search
        const uint32_t t = (group + BM - 1) / BM, each = t * c.kv_heads;
        p.b = idx / each;
        if (p.b >= c.n) return false;
        p.s = uniform(sequence(c, p.b));
        p.tiles = t;
        p.units = 1;
        p.unit0 = 0;
        p.j = (idx - p.b * each) / c.kv_heads;
        p.h = idx - p.b * each - p.j * c.kv_heads;
        *per = 1;
        return true;
    }
    Seq s{0, 0, 0};  // of the lane's sequence; up to 64 are read once
    auto read = [&](uint32_t b0) {
        s = Seq{0, 0, 0};
        if (b0 + lane < c.n) s = sequence(c, b0 + lane);
    };
    read(0);
    *per = JOIN ? *plan : 1;
    if (!JOIN && slots) {
        uint32_t total = 0;
        for (uint32_t b0 = 0;;) {
            total += tiles_of<BM>(s, group) * units_of(s, unit, slots);
            if ((b0 += 64) >= c.n) break;
            read(b0);
        }
        *per = max(1u, (lane_of(wave_scan(total), 63) * c.kv_heads + slots - 1) / slots);
        if (blockIdx.x == 0) *plan = *per;
        if (c.n > 64) read(0);
    }
    const uint32_t want = JOIN ? idx : idx * *per;
    uint32_t base = 0, start = 0;
    for (uint32_t b0 = 0; b0 < c.n; b0 += 64) {
        if (b0) read(b0);
        const uint32_t t = tiles_of<BM>(s, group), u = units_of(s, unit, slots);
        const uint32_t all = t * c.kv_heads * u, mine = JOIN ? t * c.kv_heads : all;
        const uint32_t end = wave_scan(mine), send = JOIN ? wave_scan(all) : end;
        const uint64_t hit = __ballot(base + end > want);
        if (hit) {
            const int w = __ffsll((unsigned long long)hit) - 1;
            p.b = b0 + w;
            p.s = Seq{lane_of(s.r0, w), lane_of(s.nq, w), lane_of(s.len, w)};
            p.tiles = lane_of(t, w);
            p.units = lane_of(u, w);
            const uint32_t rel = want - (base + lane_of(end - mine, w)), tile = JOIN ? rel : rel / p.units;
            p.unit0 = JOIN ? 0 : rel - tile * p.units;
            p.j = tile / c.kv_heads;
            p.h = tile - p.j * c.kv_heads;
            p.start = start + lane_of(send - all, w) + tile * p.units;
            return true;
        }
        base += lane_of(end, 63);
        start += lane_of(send, 63);
    }
    return false;
}

// Item `idx` of a call, found by every wave for itself.  Row tiles of BM rows,
// keys in units of UNIT.  Where there are fewer tiles than workgroups on the chip (half
// of `slots`; 0: never), each sequence's tiles are cut into parts of at most C units:
// ragged lengths share the chip evenly.  Order: sequence, tile (the last first: it sees most), part, key head -
// heads innermost, so that a head's workgroups stay on the same XCDs' L2.
// JOIN: an item per tile instead of one per part.
template <int BM, int UNIT, bool JOIN>
__device__ __forceinline__ bool find_item(const AttnCache &c, uint32_t group, uint32_t slots, uint32_t idx, uint32_t *plan,
                                          Item &it) {
    const uint32_t lane = threadIdx.x & 63;
    if (!JOIN && !slots && !c.row0) {  // a row and so many tiles for each sequence: nothing to search
        const uint32_t t = (group + BM - 1) / BM, each = t * c.kv_heads;
        it.b = idx / each;
        if (it.b >= c.n) return false;
        const Seq q = uniform(sequence(c, it.b));
        const uint32_t j = (idx - it.b * each) / c.kv_heads;
        it.rt = t - 1 - j;
        it.part = 0;
        it.h = idx - it.b * each - j * c.kv_heads;
        it.parts = 1;
        it.slot = idx;
        it.r0 = q.r0;
        it.nq = q.nq;
        it.len = q.len;
        return true;
    }
    Seq s{0, 0, 0};  // of the lane's sequence; up to 64 are read once
    auto read = [&](uint32_t b0) {
        s = Seq{0, 0, 0};
        if (b0 + lane < c.n) s = sequence(c, b0 + lane);
    };
    read(0);
    uint32_t C = JOIN ? *plan : kWhole;
    if (JOIN && C == kWhole) return false;
    if (!JOIN && slots) {
        float total = 0, seen = 0;  // units if each tile had the deepest's, and about what they have
        uint32_t deepest = 0, tiles = 0;
        for (uint32_t b0 = 0;;) {
            const uint32_t t = tiles_of<BM>(s, group);
            tiles += t;
            total += (float)t * (float)((s.len + UNIT - 1) / UNIT);
            seen += (float)t * ((float)s.len - 0.5f * (float)min(s.nq, s.len)) * (1.0f / UNIT);
            deepest = max(deepest, t ? (uint32_t)(s.len + UNIT - 1) / UNIT : 0);
            if ((b0 += 64) >= c.n) break;
            read(b0);
        }
        total = lane_of(wave_scan(total), 63);
        tiles = lane_of(wave_scan(tiles), 63);
        auto largest = [](uint32_t x) {
#pragma unroll
            for (int m = 32; m; m >>= 1) x = max(x, (uint32_t)__shfl_xor((int)x, m));
            return x;
        };
        // Whole tiles, or parts for one round of the chip, or for two, by units of time: a start and an end cost
        // about two, joining ten, and beyond one round the work is spread evenly but for half a part.  196 tiles of
        // 325 units make 392 parts of 163 in one round, which leaves a quarter of the chip idle, or 980 of 65 in two
        // (398 and 361 us when the rule was made); 500 of up to 32 units are best left whole (62 us for 82).
        const float chip = (float)(slots / 2);
        seen = lane_of(wave_scan(seen), 63) * (float)c.kv_heads / chip;
        auto time = [&](uint32_t items, uint32_t longest) {
            return (float)items <= chip ? (float)(longest + 2) : seen + 2.0f * (float)items / chip + 0.5f * (float)longest;
        };
        float best = time(tiles * c.kv_heads, largest(deepest));
        for (uint32_t k = 1; k <= 2; ++k) {
            const uint32_t room = k * (slots / 2) / c.kv_heads;
            if (tiles >= room) continue;
            const uint32_t Ck = max(3u, (uint32_t)__builtin_ceilf(total / (float)(room - tiles) * 1.00001f));
            uint32_t sum = 0, longest = 0;
            for (uint32_t b0 = 0; b0 < c.n; b0 += 64) {
                if (c.n > 64) read(b0);
                const uint32_t u = (uint32_t)(s.len + UNIT - 1) / UNIT, parts = max(1u, (u + Ck - 1) / Ck);
                const uint32_t t = tiles_of<BM>(s, group);
                sum += t * parts;
                longest = max(longest, t ? (u + parts - 1) / parts : 0);
            }
            const float cost = time(lane_of(wave_scan(sum), 63) * c.kv_heads, largest(longest)) + 10.0f;
            if (cost < best) {
                best = cost;
                C = Ck;
            }
        }
        if (blockIdx.x == 0) *plan = C;
        if (c.n > 64) read(0);
    }
    if (!JOIN && C == kWhole && c.n <= 64) {
        // No parts: the tiles with the most units first, whichever sequence they are of, so that the last
        // ones to start are short.  reach(U): tiles of the lane's sequence that have at least U units, which
        // are its last ones: the largest U that idx tiles or fewer reach is that of tile idx.
        const uint32_t t = tiles_of<BM>(s, group);
        const int32_t past = s.len - s.nq;
        auto reach = [&](uint32_t U) {
            const int32_t tok = (int32_t)((U - 1) * UNIT) - past;  // a last row of this token or later
            if (U == 1 || tok <= 0) return t;                      // (a tile that sees nothing is written too)
            return tok >= s.nq ? 0u : t - ((uint32_t)tok * group + BM) / BM + 1;
        };
        auto total = [&](uint32_t U) { return lane_of(wave_scan(reach(U)), 63) * c.kv_heads; };
        if (idx >= total(1)) return false;
        uint32_t lo = 1, hi = (c.max_pages * c.page_size + UNIT - 1) / UNIT + 1;  // total(lo) > idx >= total(hi)
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (total(mid) > idx) lo = mid; else hi = mid;
        }
        const uint32_t more = reach(lo + 1), mine = reach(lo) - more;  // tiles of exactly lo units
        const uint32_t rel = idx - total(lo + 1), end = wave_scan(mine) * c.kv_heads;
        const int w = __ffsll((unsigned long long)__ballot(end > rel)) - 1;
        const uint32_t at = rel - lane_of(end - mine * c.kv_heads, w), j = at / c.kv_heads;
        it.b = w;
        it.r0 = lane_of(s.r0, w);
        it.nq = lane_of(s.nq, w);
        it.len = lane_of(s.len, w);
        it.parts = 1;
        it.rt = lane_of(t - 1 - more, w) - j;
        it.part = 0;
        it.h = at - j * c.kv_heads;
        it.slot = idx;
        return true;
    }
    uint32_t base = 0, slot0 = 0;
    for (uint32_t b0 = 0; b0 < c.n; b0 += 64) {
        if (b0) read(b0);
        uint32_t t = ((uint32_t)s.nq * group + BM - 1) / BM, parts = 1;
        if (C != kWhole) parts = max(1u, ((uint32_t)(s.len + UNIT - 1) / UNIT + C - 1) / C);
        const uint32_t all = t * parts * c.kv_heads, mine = JOIN ? t * c.kv_heads : all;
        const uint32_t end = wave_scan(mine), send = JOIN ? wave_scan(all) : 0;
        const uint64_t hit = __ballot(base + end > idx);
        if (hit) {
            const int w = __ffsll((unsigned long long)hit) - 1;
            it.b = b0 + w;
            it.r0 = __builtin_amdgcn_readlane(s.r0, w);
            it.nq = __builtin_amdgcn_readlane(s.nq, w);
            it.len = __builtin_amdgcn_readlane(s.len, w);
            it.parts = __builtin_amdgcn_readlane(parts, w);
            t = __builtin_amdgcn_readlane(t, w);
            const uint32_t rel = idx - (base + __builtin_amdgcn_readlane(end - mine, w));
            const uint32_t per = JOIN ? c.kv_heads : it.parts * c.kv_heads;
            const uint32_t j = rel / per, rem = rel - j * per;
            it.rt = t - 1 - j;
            it.part = rem / c.kv_heads;
            it.h = rem - it.part * c.kv_heads;
            // where the tile's first part's sums are
            it.slot = JOIN ? slot0 + __builtin_amdgcn_readlane(send - all, w) + j * it.parts * c.kv_heads + it.h : idx;
            return true;
        }
        base += __builtin_amdgcn_readlane(end, 63);
        if (JOIN) slot0 += __builtin_amdgcn_readlane(send, 63);
    }
    return false;
}

// Keys that the tile's last row sees, and the units of them that each part takes.
template <int BM, int UNIT>
__device__ __forceinline__ void tile_keys(const Item &it, uint32_t group, int32_t *end, uint32_t *per, uint32_t *parts) {
    const uint32_t last = min((it.rt + 1) * BM, (uint32_t)it.nq * group) - 1;
    *end = max(0, it.len - it.nq + (int32_t)(last / group) + 1);
    const uint32_t units = (uint32_t)(*end + UNIT - 1) / UNIT;
    *per = max(1u, (units + it.parts - 1) / it.parts);
    *parts = max(1u, (units + *per - 1) / *per);
}

// Runs of 16 keys of a sequence: N neighbours at a time, STEP runs from one time to
// the next; past the last key the last run again, or the one before (its loads stay in
// bounds, its keys are masked).  Page numbers come by scalar loads: fetch() asks for
// N runs' and place() takes them later, so that the look-up of a tile's pages goes on
// under the tile before it.
template <int N, int STEP = N>
struct Runs {
    const int32_t *table;
    uint32_t j, slot, next, last;  // page index and slot of the next run, its number, and the last one's
    uint32_t step_j, step_slot;    // STEP - N runs further, in pages and slots
    uint32_t page[N], at[N];       // of the runs asked for
    __device__ __forceinline__ void start(const AttnCache &c, uint32_t b, uint32_t run, int32_t keys) {
        const uint32_t n = (uint32_t)(keys + 15) / 16;
        last = n ? n - 1 : 0;
        next = min(run, last);
        table = c.table + (uint64_t)b * c.max_pages;
        j = next * 16 / c.page_size;
        slot = next * 16 - j * c.page_size;
        step_j = (STEP - N) * 16 / c.page_size;
        step_slot = (STEP - N) * 16 - step_j * c.page_size;
        fetch(c);
    }
    __device__ __forceinline__ void fetch(const AttnCache &c) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            page[i] = (uint32_t)*(const __attribute__((address_space(4))) int32_t *)(uintptr_t)(table + j);
            at[i] = slot;
            const uint32_t far = i + 1 == N ? 1 + STEP - N : 1;  // to the run after it
            if (next + far <= last) {
                next += far;
                slot += 16 + (far > 1 ? step_slot : 0);
                j += far > 1 ? step_j : 0;
                if (slot >= c.page_size) {
                    slot -= c.page_size;
                    ++j;
                }
                if (far > 1 && slot >= c.page_size) {
                    slot -= c.page_size;
                    ++j;
                }
            }
        }
    }
    // Element offset of run i's first key; a page outside the cache is noted and read as page 0.
    __device__ __forceinline__ uint64_t place(const AttnCache &c, uint64_t head, int i, bool *bad) const {
        const bool in = page[i] < c.pages;
        *bad |= !in;
        return (in ? page[i] : 0) * c.page_stride + at[i] * c.token_stride + head;
    }
};

// Running softmax of a lane's row: m the largest exponent (of 2) so far, or a bit
// below, l the sum of this lane's weights.  Sums are scaled down only where the
// largest rises by more than 2^8: every weight stays under 2^8 and nothing is
// lost in f32.
struct Row {
    float m, l;
};
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ float across32(float x) {  // the larger of lanes l and l ^ 32
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float across16(float x) {  // and of l ^ 16
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

// 4 numbers of a result row, times f; f is 0 for a row that sees nothing.
template <uint32_t R>
__device__ __forceinline__ void write4(const AttnArgs &A, uint64_t row, uint32_t head, int dim, uint32_t d, f32x4 y, float f) {
    const uint64_t at = row * A.out_stride + (uint64_t)head * dim + d;
    if constexpr (R == kF32) {
        *(f32x4 *)((float *)A.out + at) = y * f;
    } else {
        typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
        *(bf4 *)((uint16_t *)A.out + at) = bf4{(__bf16)(y[0] * f), (__bf16)(y[1] * f), (__bf16)(y[2] * f), (__bf16)(y[3] * f)};
    }
}

__device__ __forceinline__ f32x4 mfma16(bf8 a, bf8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(bf8 a, bf8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Where masks cut through a tile, its values that are not finite are staged as 0
// (a masked weight of 0 would make them a NaN in rows that do not see them) and
// added here, after the loop, to the rows that see them, a key at a time: it is
// rare.  o: a lane's numbers of O^T, of 32 x 32 products (W32) or 16 x 16.
template <uint32_t C, int D, bool W32, typename V, int NB>
__device__ __forceinline__ void add_not_finite(const AttnCache &c, const Item &it, int32_t from, int32_t to, int32_t sees,
                                               V (&o)[NB]) {
    constexpr int M = W32 ? 32 : 16;
    const uint32_t d0 = (thread_id() & 63) / M * 4;
    Runs<1> runs;
    bool bad;  // (noted before)
    runs.start(c, it.b, (uint32_t)from / 16, to);
#pragma unroll 1
    for (int32_t run = from / 16 * 16; run < to; run += 16, runs.fetch(c)) {
        const uint64_t base = runs.place(c, it.h * c.head_stride, 0, &bad) + d0;
#pragma unroll 1
        for (int32_t key = max(run, from); key < min(run + 16, to); ++key) {
            const uint64_t at = base + (uint64_t)(key - run) * c.token_stride;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < M * M / 64; ++e) {
                    const float x = load1<C>(c.v, at + i * M + e / 4 * 8 + e % 4);
                    o[i][e] += key < sees && !__builtin_isfinite(x) ? x : 0.0f;
                    if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
        }
    }
}

// ---- few rows on long caches: the keys split over waves and workgroups -----------
// A workgroup takes 16 rows of one key head at a time; its W waves take a W-th of
// the keys each, KEYS at a time, loading keys straight into matrix operand
// registers and values through their own LDS tiles.  The order of the head
// dimension in the first product is free: lane group g holds numbers N g .. of each
// 4 N, as one load brings them.  No barrier but at a tile's end: a wave's LDS tile
// is its own.
//
// Bound: HBM.  32 sequences of up to 16,001 tokens, BF16 cache of 4 heads of 128 (485
// MB): 79 us, 6.2 TB/s, the rate of a plain read here; one of 131,071 tokens 46 us
// (5.8 TB/s); 128 sequences on an E4M3 cache (594 MB) 122 us (4.9 TB/s: f32 rows'
// three terms of half the bytes, and two tile ends a workgroup).  577 tokens take 9
// us: 2.7 to find the place, 1.6 to the first loads, 3.7 to the end of the only step,
// 0.8 to the end.  With a part of each sequence a workgroup instead of equal shares 95
// us for the first; the next tile's loads after this one's end 87; three waves a SIMD
// the same time as two.
template <uint32_t R, uint32_t C, int D>
struct SplitCfg {
    static constexpr int QT = kTerms<R>, KT = kTerms<C>, BM = 16;
    static constexpr int PT = QT == 1 ? 2 : 3;  // of the weights: the matrix cores have time to spare here
    static constexpr int KEYS = C == kE4M3 && D <= 128 ? 64 : 32;  // about 8 KB of keys and of values in flight a wave
    static constexpr int W = KT == 3 && D == 256 ? 2 : 4, UNIT = W * KEYS;  // waves: as many as their tiles fit the LDS
    static constexpr int OCC = D == 256 ? 1 : KT == 3 ? (D == 64 ? 2 : 1) : D == 64 ? 3 : 2;  // waves on a SIMD
    static constexpr int TILE = KEYS * D * 2;            // bytes of one plane
    static constexpr int WAVE = TILE * KT > BM * D * 4 ? TILE * KT : BM * D * 4;
    static constexpr int SLOT = BM * (D + 2);            // floats of a part's sums
};

__device__ __forceinline__ u32x2 read_tr(const uint8_t *lds, uint32_t at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((CZ_LDS s16x4 *)(lds + at)));
}

template <uint32_t R, uint32_t C, int D>
__global__ __launch_bounds__((64 * SplitCfg<R, C, D>::W), (SplitCfg<R, C, D>::OCC)) void k_attn_split(AttnArgs A, uint32_t slots,
                                                                                                 uint32_t unit) {
    using G = SplitCfg<R, C, D>;
    constexpr int QT = G::QT, KT = G::KT, PT = G::PT, W = G::W, NS = D / 32, NB = D / 16, KEYS = G::KEYS, NR = KEYS / 16;
    constexpr int PN = Piece<C>::N, SUB = PN / 8, NK = NS / SUB, NV = KEYS * D / PN / 64;
    __shared__ __align__(16) uint8_t sh[W * G::WAVE];
    __shared__ float sh_m[W][16], sh_l[W][16];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15;
    Place pl;
    uint32_t left;
    if (!find_place<G::BM, false>(A.c, A.group, slots, unit, blockIdx.x, (uint32_t *)A.work, &left, pl)) return;

    // A tile of the share: its rows, and the wave's keys.
    struct Segment {
        Item it;
        uint32_t take;
        bool whole, opens;          // all of the tile's units; its first ones
        int32_t end, first, stop;   // keys that its last row sees; the wave's
    };
    auto segment = [&] {
        Segment sg;
        sg.it = Item{pl.b, pl.tiles - 1 - pl.j, pl.h, 0, 0, 0, pl.s.r0, pl.s.nq, pl.s.len};
        sg.take = min(left, pl.units - pl.unit0);
        sg.whole = sg.take == pl.units;
        sg.opens = pl.unit0 == 0;
        const uint32_t last = min((sg.it.rt + 1) * 16, (uint32_t)sg.it.nq * A.group) - 1;
        sg.end = max(0, sg.it.len - sg.it.nq + (int32_t)(last / A.group) + 1);
        const int32_t f = slots ? (int32_t)(pl.unit0 * unit) : 0;
        const int32_t st = slots ? min(sg.end, f + (int32_t)(sg.take * unit)) : sg.end;
        const int32_t share = (max(0, st - f) + W * KEYS - 1) / (W * KEYS) * KEYS;
        sg.first = f + (int32_t)wave * share;
        sg.stop = min(st, sg.first + share);
        return sg;
    };
    // the tile after it; the next sequence has been read ahead
    Seq ahead;
    auto advance = [&](uint32_t took) {
        left -= took;
        if (!left) return false;
        pl.unit0 = 0;
        if (++pl.h < A.c.kv_heads) return true;
        pl.h = 0;
        if (++pl.j < pl.tiles) return true;
        pl.j = 0;
        do {
            if (++pl.b == A.c.n) return false;
            pl.s = uniform(ahead);
            pl.tiles = tiles_of<G::BM>(pl.s, A.group);
            ahead = sequence(A.c, min(pl.b + 1, A.c.n - 1));
        } while (!pl.tiles);
        pl.units = units_of(pl.s, unit, slots);
        return true;
    };

    Runs<NR> runs;
    bool bad_page = false;
    Piece<C> kr[NR][NK], vr[NV];
    // addresses: a scalar base for a run of keys or a load of values, and one offset a lane for each kind
    const uint32_t ts = (uint32_t)A.c.token_stride * kSize<C>, klane = col * ts + g * PN * kSize<C>;
    const uint32_t vlane = lane / (D / PN) * ts + lane % (D / PN) * PN * kSize<C>;
    uint64_t base[NR];
    auto load_keys = [&](const Item &it) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            base[n] = runs.place(A.c, it.h * A.c.head_stride, n, &bad_page) * kSize<C>;
#pragma unroll
            for (int s = 0; s < NK; ++s) kr[n][s].load_once((const uint8_t *)A.c.k + base[n] + klane + s * 4 * PN * kSize<C>);
        }
        runs.fetch(A.c);
    };
    auto load_values = [&] {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            constexpr int KL = 64 / (D / PN);  // keys a load
            vr[i].load_once((const uint8_t *)A.c.v + base[i * KL / 16] + i * KL % 16 * ts + vlane);
        }
    };
    auto start = [&](const Segment &sg) {
        if (sg.first >= sg.stop) return;
        runs.start(A.c, sg.it.b, (uint32_t)sg.first / 16, sg.end);
        load_keys(sg.it);
        load_values();
    };
    Segment sg = segment();
    start(sg);
    ahead = sequence(A.c, min(pl.b + 1, A.c.n - 1));

    // tile after tile until the share is used up; the next one's first loads go out before this one's end
    for (;;) {
    const Item it = sg.it;
    const uint32_t r = it.rt * 16 + col, rows = (uint32_t)it.nq * A.group;
    const bool valid = r < rows;
    const uint32_t tok = valid ? r / A.group : 0, x = it.h * A.group + (valid ? r - tok * A.group : 0);
    const uint64_t row = (uint64_t)(it.r0 + (int32_t)tok);
    const int32_t sees = valid ? min(max(it.len - it.nq + (int32_t)tok + 1, 0), sg.end) : 0;
    const int32_t sees_min = __builtin_amdgcn_readfirstlane(sees);
    float c2 = A.scale * (C == kE4M3 && A.c.k_scale ? A.c.k_scale[it.h] : 1.0f) * 1.44269504088896340736f;
    const uint32_t flip = c2 < 0.0f ? 0x80000000u : 0u;
    c2 = fabsf(c2);

    bf8 q[NS][QT];
#pragma unroll
    for (int s = 0; s < NS; ++s)
        query8<R>(A.q, row * A.q_stride + (uint64_t)x * D + s / SUB * 4 * PN + g * PN + s % SUB * 8, flip, q[s]);

    f32x4 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f32x4{0, 0, 0, 0};
    Row st{-INFINITY, 0.0f};
    uint8_t *const lds = sh + wave * G::WAVE;
    const int32_t wfirst = sg.first, wstop = sg.stop;
    int32_t bad_at = -1;
    for (int32_t key0 = wfirst; key0 < wstop; key0 += KEYS) {
        f32x4 sc[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            sc[n] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                bf8 k[KT];
                kr[n][s / SUB].terms(s % SUB, k);
                sc[n] = product<KT, QT>(k, q[s], sc[n], mfma16);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (key0 + KEYS < wstop) load_keys(it);
        // values into the wave's tile; what is behind the sequence's end counts as 0
        const bool masked = key0 + KEYS > sees_min;
        if (masked) {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (key0 + (int32_t)((i * 64 + lane) / (D / PN)) >= it.len) vr[i].zero();
                bad |= vr[i].clean();
            }
            if (bad_at < 0 && __any(bad)) bad_at = key0;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t id = i * 64 + lane, key = id / (D / PN), ch = id % (D / PN);
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                bf8 v[KT];
                vr[i].terms(u, v);
#pragma unroll
                for (int t = 0; t < KT; ++t) *(bf8 *)(lds + t * G::TILE + lds_at<D>(key, ch * SUB + u)) = v[t];
            }
        }
        if (key0 + KEYS < wstop) load_values();
        __builtin_amdgcn_sched_barrier(0);

        float cc = c2;
        if (masked) {
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sc[n][i] = key0 + n * 16 + (int32_t)g * 4 + i < sees ? sc[n][i] * c2 : -INFINITY;
            cc = 1.0f;
        }
        float mx = sc[0][0];
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[n][i]);
        mx = across32(across16(mx)) * cc;
        if (__any(mx > st.m + 8.0f)) {
            const float mn = fmaxf(st.m, mx), f = exp2_hw(st.m - finite_max(mn));
            st.l *= f;
#pragma unroll
            for (int i = 0; i < NB; ++i) o[i] *= f;
            st.m = mn;
        }
        const float mu = finite_max(st.m);
        const uint32_t tk = g * 4 + (col >> 2), tc = (col & 3) >> 1, tb = (col & 1) * 8;
#pragma unroll
        for (int n = 0; n < NR; n += 2) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = exp2_hw(__builtin_fmaf(sc[n + i / 4][i % 4], cc, -mu));
                st.l += p[i];
            }
            bf8 pt[PT];
            split8<PT>(p, pt);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                bf8 v[KT];
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    const uint32_t at = t * G::TILE + lds_at<D>(tk, i * 2 + tc) + tb + n * 16 * D * 2;
                    const u32x2 a = read_tr(lds, at), b = read_tr(lds, at + 16 * D * 2);
                    v[t] = __builtin_bit_cast(bf8, u32x4{a[0], a[1], b[0], b[1]});
                }
                o[i] = product<KT, PT>(v, pt, o[i], mfma16);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (bad_at >= 0) add_not_finite<C, D, false>(A.c, it, bad_at, min(wstop, it.len), sees, o);

    const Segment done = sg;
    const bool more = advance(sg.take);
    if (more) {
        sg = segment();
        start(sg);
    }

    // the waves' sums
    const uint32_t tid = thread_id(), ecol = tid & 15, eg = tid >> 4 & 3;
    st.l += __shfl_xor(st.l, 16);
    st.l += __shfl_xor(st.l, 32);
    if (eg == 0) {
        sh_m[wave][ecol] = st.m;
        sh_l[wave][ecol] = st.l;
    }
    float *const mine = (float *)lds;
#pragma unroll
    for (int i = 0; i < NB; ++i) *(f32x4 *)(mine + ecol * D + ((i * 16 + eg * 4) ^ ((ecol & 7) << 2))) = o[i];
    __syncthreads();
    // a workgroup's share starts with at most one tile's end and ends with at most one tile's start
    float *const part = (float *)A.work + kPlanFloats + (2 * (uint64_t)blockIdx.x + done.opens) * G::SLOT;
    const float vs = C == kE4M3 && A.c.v_scale ? A.c.v_scale[it.h] : 1.0f;
#pragma unroll
    for (int e = 0; e < 16 * D / 4 / (64 * W); ++e) {
        const uint32_t id = e * 64 * W + tid, rr = id / (D / 4), d = id % (D / 4) * 4;
        const uint32_t tr = it.rt * 16 + rr;
        if (tr >= rows) continue;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, sh_m[w][rr]);
        const float mf = finite_max(m);
        f32x4 y{0, 0, 0, 0};
        float l = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = exp2_hw(sh_m[w][rr] - mf);
            const f32x4 z = *(const f32x4 *)((const float *)(sh + w * G::WAVE) + rr * D + (d ^ ((rr & 7) << 2)));
            l = __builtin_fmaf(sh_l[w][rr], f, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(z[i], f, y[i]);
        }
        if (!done.whole) {
            *(f32x4 *)(part + rr * D + d) = y;
            if (d == 0) {
                part[16 * D + rr] = m;
                part[16 * D + 16 + rr] = l;
            }
        } else {
            const uint32_t t = tr / A.group;
            write4<R>(A, (uint64_t)it.r0 + t, it.h * A.group + tr - t * A.group, D, d, y,
                      it.len - it.nq + (int32_t)t + 1 > 0 ? vs / l : 0.0f);
        }
    }
    if (!more) break;
    __syncthreads();
    }
    if (bad_page) flag(A.c.err, kAttnBadPage);
}

// Joins the parts of a tile.  LD lanes read LD * 4 numbers of a part's row; a
// workgroup takes ROWS rows of them, NG groups of lanes sharing a row's parts.
// UNIT > 0: of the prompt kernel's parts, else of shares of units of `unit` keys.
template <uint32_t R, uint32_t C, int D, int BM, int UNIT, int LD, int ROWS>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs A, uint32_t slots, uint32_t unit) {
    constexpr uint32_t NG = 256 / LD / ROWS, BLOCKS = BM / ROWS, SLOT = BM * (D + 2);
    Item it;
    const uint32_t rb = blockIdx.x % BLOCKS * ROWS, rr = rb + threadIdx.x / (LD * NG);
    uint32_t parts;
    uint64_t slot0, next;  // the first part's sums, and from the second's to the next
    if constexpr (UNIT > 0) {
        if (!find_item<BM, UNIT, true>(A.c, A.group, slots, blockIdx.x / BLOCKS, (uint32_t *)A.work, it)) return;
        int32_t end;
        uint32_t per;
        tile_keys<BM, UNIT>(it, A.group, &end, &per, &parts);
        slot0 = it.slot;
        next = A.c.kv_heads;
        // (rows that overlap, which has been flagged, can place a tile where no part is)
        if (slot0 + (parts - 1) * next >= slots) return;
    } else {
        Place p;
        uint32_t per;
        if (!find_place<BM, true>(A.c, A.group, slots, unit, blockIdx.x / BLOCKS, (uint32_t *)A.work, &per, p)) return;
        const uint32_t w = p.start / per;
        parts = (p.start + p.units - 1) / per - w + 1;
        slot0 = 2 * (uint64_t)w;
        next = 2;
        if (slot0 + 2 * (uint64_t)parts > 2 * (uint64_t)slots) return;
        it = Item{p.b, p.tiles - 1 - p.j, p.h, 0, 0, 0, p.s.r0, p.s.nq, p.s.len};
    }
    const uint32_t tr = it.rt * BM + rr;
    if (parts == 1 || it.rt * BM + rb >= (uint32_t)it.nq * A.group) return;
    const float *const first = (const float *)A.work + kPlanFloats + slot0 * SLOT;
    const uint64_t step = next * SLOT;
    const uint32_t pg = threadIdx.x / LD % NG, dl = threadIdx.x % LD, d = (blockIdx.y * LD + dl) * 4;
    // a group keeps its own running maximum; the groups are joined like the parts
    float m = -INFINITY, l = 0;
    f32x4 y{0, 0, 0, 0};
    for (uint32_t p = pg; p < parts; p += NG) {
        const float *const s = first + p * step + (UNIT == 0 && p == 0 ? SLOT : 0);
        const float pm = s[BM * D + rr], pl = s[BM * D + BM + rr];
        const f32x4 z = *(const f32x4 *)(s + rr * D + d);
        const float mn = fmaxf(m, pm), f0 = exp2_hw(m - finite_max(mn)), f1 = exp2_hw(pm - finite_max(mn));
        m = mn;
        l = __builtin_fmaf(pl, f1, l * f0);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(z[i], f1, y[i] * f0);
    }
    if constexpr (NG > 1) {
        __shared__ float sh_m[ROWS][NG], sh_l[ROWS][NG];
        __shared__ f32x4 sh_y[ROWS][NG][LD];
        const uint32_t w = threadIdx.x / (LD * NG);
        if (dl == 0) {
            sh_m[w][pg] = m;
            sh_l[w][pg] = l;
        }
        sh_y[w][pg][dl] = y;
        __syncthreads();
        if (pg) return;
        m = sh_m[w][0];
#pragma unroll
        for (uint32_t i = 1; i < NG; ++i) m = fmaxf(m, sh_m[w][i]);
        const float mf = finite_max(m);
        l = 0;
        y = f32x4{0, 0, 0, 0};
#pragma unroll
        for (uint32_t g = 0; g < NG; ++g) {
            const float f = exp2_hw(sh_m[w][g] - mf);
            l = __builtin_fmaf(sh_l[w][g], f, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(sh_y[w][g][dl][i], f, y[i]);
        }
    }
    if (tr >= (uint32_t)it.nq * A.group) return;
    const uint32_t t = tr / A.group;
    const float vs = C == kE4M3 && A.c.v_scale ? A.c.v_scale[it.h] : 1.0f;
    write4<R>(A, (uint64_t)it.r0 + t, it.h * A.group + tr - t * A.group, D, d, y,
              it.len - it.nq + (int32_t)t + 1 > 0 ? vs / l : 0.0f);
}

// ---- prompts ---------------------------------------------------------------------
// A workgroup takes BM rows of one key head, 32 per wave, and walks over tiles of BK
// keys that its four waves share in LDS as bf16 planes: an E4M3 cache is widened and
// an f32 one split once, as the tile is staged.  KS = 1: 128 rows, each wave all keys
// of a tile.  KS = 2: 64 rows, two waves share 32 rows and take half of a tile's keys
// each: for few rows, and where 128-row tiles would leave CUs idle (6 tokens on each
// of 16 caches of 8,000, BF16: 52 us, 160 with 16-row tiles).
//
// Bound: the matrix cores and, at two waves a SIMD, the vector work of the softmax
// beside them (44 and 57% of a SIMD's cycles at 8,192 BF16 tokens, 53 and 57 with f32
// rows; the clock falls under such load as it does under a large product).  8,192
// tokens, 32 heads on 4 of 128: 605-618 us, 890-910 TFLOP/s of the visible products,
// where a large bf16 product reaches 1,220; packed prompts of f32 rows 339-345 us, 345
// TFLOP/s and three times that in products; 777 tokens on 20,000 cached in E4M3 305 us,
// 850 TFLOP/s.  A short prompt (500 tokens of f32 rows, 29 us) is 4 us to find its
// tile, 8 to the end of the first 64 keys and 2 to 4 for each 64 after.
//
// 64-key tiles but where registers or LDS are short: with three terms of q a 64-key
// tile spills (444 us for 358).  A wave looks up one page a tile: four look-ups a wave
// were as many scalar instructions as vector ones, 6% of the time.  Measured and not
// kept: fixed interleaving of matrix and vector instructions (750 for 700 us), raised
// priority of the waves in the first product (within 2%), values loaded only after the
// keys are staged (spills), eight waves to a 64-row tile (500 tokens of f32 rows 27.4 for 27.6 us,
// BF16 16.6 for 15.8), a term of the weights at a time over four blocks of the head
// (30.7 for 27.6: spills), q's third term in the LDS for heads of 128 too (the same).
template <uint32_t R, uint32_t C, int D, int KS>
struct TileCfg {
    static constexpr int QT = kTerms<R>, KT = kTerms<C>, BM = 128 / KS;
    static constexpr int BK = KS == 1 && (KT == 3 || D == 256 || (QT == 3 && D == 128)) ? 32 : 64;
    static constexpr int PLANE = BK * D * 2, HALF = PLANE * KT;       // bytes of a tile's K, and of its V
    static constexpr int BUF = 4 * HALF <= 128 * 1024 ? 2 : 1;
    // Three terms of a q of 256 do not fit the registers: the third waits in the LDS, in the order its
    // reads take it.
    static constexpr bool QLDS = QT == 3 && D == 256;
    static constexpr int QBYTES = QLDS ? BM * D * 2 : 0, LDS = BUF * 2 * HALF + QBYTES;
    static constexpr int OCC = LDS > 80 * 1024 || D == 256 ? 1 : 2;  // waves on a SIMD
    static constexpr int SLOT = BM * (D + 2);
    static constexpr bool FITS = LDS <= 160 * 1024;
};

template <uint32_t R, uint32_t C, int D, int KS>
__global__ __launch_bounds__(256, (TileCfg<R, C, D, KS>::OCC)) void k_attn_tile(AttnArgs A, uint32_t slots) {
    using G = TileCfg<R, C, D, KS>;
    constexpr int QT = G::QT, KT = G::KT, BK = G::BK, WK = BK / KS, NS = D / 16, NB = D / 32, NN = WK / 32;
    constexpr int PN = Piece<C>::N, SUB = PN / 8, NL = BK * D / PN / 256;
    __shared__ __align__(16) uint8_t sh[G::LDS];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 5, col = lane & 31, wrow = (KS == 1 ? wave : wave & 1) * 32, kq = KS == 1 ? 0 : wave >> 1;
    Item it;
    if (!find_item<G::BM, BK, false>(A.c, A.group, slots, blockIdx.x, (uint32_t *)A.work, it)) return;
    int32_t end;
    uint32_t per, parts;
    tile_keys<G::BM, BK>(it, A.group, &end, &per, &parts);
    if (it.part >= parts) return;
    const int32_t first = (int32_t)(it.part * per * BK), stop = min(end, first + (int32_t)(per * BK));

    const uint32_t rows = (uint32_t)it.nq * A.group, r = it.rt * G::BM + wrow + col;
    const bool valid = r < rows;
    const uint32_t tok = valid ? r / A.group : 0, x = it.h * A.group + (valid ? r - tok * A.group : 0);
    const uint64_t row = (uint64_t)(it.r0 + (int32_t)tok);
    const int32_t sees = valid ? min(max(it.len - it.nq + (int32_t)tok + 1, 0), end) : 0;
    const int32_t sees_min = __builtin_amdgcn_readfirstlane(sees);
    // the wave's last row; a wave without rows sees nothing
    const uint32_t w0 = it.rt * G::BM + wrow, wl = min(w0 + 32, rows);
    const int32_t sees_max = w0 < rows ? min(max(it.len - it.nq + (int32_t)((wl - 1) / A.group) + 1, 0), end) : 0;
    float c2 = A.scale * (C == kE4M3 && A.c.k_scale ? A.c.k_scale[it.h] : 1.0f) * 1.44269504088896340736f;
    const uint32_t flip = c2 < 0.0f ? 0x80000000u : 0u;
    c2 = fabsf(c2);

    constexpr int QR = G::QLDS ? 2 : QT;  // terms of q in registers
    bf8 q[NS][QR];
    const uint32_t qlds = G::BUF * 2 * G::HALF + (wrow / 32 * NS * 64 + lane) * 16;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        bf8 all[QT];
        query8<R>(A.q, row * A.q_stride + (uint64_t)x * D + s * 16 + g * 8, flip, all);
#pragma unroll
        for (int n = 0; n < QR; ++n) q[s][n] = all[n];
        if constexpr (G::QLDS) *(bf8 *)(sh + qlds + s * 1024) = all[2];  // (waves of the same rows write the same)
    }
    f32x16 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    Row st{-INFINITY, 0.0f};

    const uint64_t head = it.h * A.c.head_stride;
    // A wave stages a quarter of the tile's keys, all of one run.
    constexpr int KW = BK / 4, KL = 64 / (D / PN);  // keys a wave, and a load
    Runs<1, BK / 16> runs;
    bool bad_page = false;
    if (first < stop) runs.start(A.c, it.b, (uint32_t)first / 16 + wave * KW / 16, end);
    Piece<C> kr[NL], vr[NL];
    const uint32_t ch = lane % (D / PN), tkey = wave * KW + lane / (D / PN), ts = (uint32_t)A.c.token_stride * kSize<C>;
    const uint32_t voff = (tkey & 15) * ts + ch * PN * kSize<C>;
    uint64_t at_run;
    auto load_keys = [&] {
        at_run = runs.place(A.c, head, 0, &bad_page) * kSize<C>;
        runs.fetch(A.c);
#pragma unroll
        for (int i = 0; i < NL; ++i) kr[i].load((const uint8_t *)A.c.k + at_run + i * KL * ts + voff);
    };
    auto load_values = [&] {
#pragma unroll
        for (int i = 0; i < NL; ++i) vr[i].load((const uint8_t *)A.c.v + at_run + i * KL * ts + voff);
    };
    // masks cut through the workgroup's tiles from here on
    const int32_t cut = min(max(it.len - it.nq + (int32_t)(it.rt * G::BM / A.group) + 1, 0), end);
    bool bad = false;
    auto put = [&](const Piece<C> &piece, int i, uint8_t *to) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            bf8 x[KT];
            piece.terms(u, x);
#pragma unroll
            for (int t = 0; t < KT; ++t) *(bf8 *)(to + t * G::PLANE + lds_at<D>(i * KL + tkey, ch * SUB + u)) = x[t];
        }
    };
    auto store_keys = [&](uint8_t *to) {
#pragma unroll
        for (int i = 0; i < NL; ++i) put(kr[i], i, to);
    };
    auto store_values = [&](int32_t key0, uint8_t *to) {
        if (key0 + BK > cut) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                if (key0 + (int32_t)(i * KL + tkey) >= it.len) vr[i].zero();
                bad |= vr[i].clean();
            }
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) put(vr[i], i, to + G::HALF);
    };
    const uint32_t klds0 = lds_at<D>(col, g);
    const uint32_t vlds0 = lds_at<D>(g * 4 + ((lane & 15) >> 2), ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) + (lane & 1) * 8;
    uint32_t buf = 0;
    if (first < stop) {
        load_keys();
        load_values();
        store_keys(sh);
        store_values(first, sh);
    }
    __syncthreads();
    for (int32_t key0 = first; key0 < stop; key0 += BK) {
        const bool more = key0 + BK < stop;
        uint8_t *const next = sh + (G::BUF == 2 ? (buf ^ 1) : 0) * 2 * G::HALF;
        if (more) {
            load_keys();
            load_values();
        }
        const int32_t kw = key0 + (int32_t)kq * WK;  // the wave's keys
        // where piece 0 of the lane's K and V reads is: piece n is at that ^ 16 n, worked out as it is needed
        uint32_t klds = klds0, vlds = vlds0;
        asm volatile("" : "+v"(klds), "+v"(vlds));
        const uint8_t *const ks = sh + buf * 2 * G::HALF + kq * WK * D * 2, *const vs = ks + G::HALF;
        const bool masked = kw + WK > sees_min;
        const float cc = masked ? 1.0f : c2;
        f32x16 sc[NN];
        bf8 pt[WK / 16][QT];
        float mu;
        // scores of 32 keys
        auto scores = [&](int n) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[n][e] = 0.0f;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                bf8 k[KT];
#pragma unroll
                for (int t = 0; t < KT; ++t) k[t] = *(const bf8 *)(ks + t * G::PLANE + n * 32 * D * 2 + (klds ^ s << 5));
                bf8 all[QT];
#pragma unroll
                for (int w = 0; w < QR; ++w) all[w] = q[s][w];
                if constexpr (G::QLDS) all[2] = *(const bf8 *)(sh + qlds + s * 1024);
                sc[n] = product<KT, QT>(k, all, sc[n], mfma32);
            }
        };
        // their mask and maximum; what was summed so far is scaled down where that rises
        auto largest = [&](int n) {
            if (masked)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    sc[n][e] = kw + n * 32 + (e / 4) * 8 + (int32_t)g * 4 + e % 4 < sees ? sc[n][e] * c2 : -INFINITY;
            float m[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) m[e] = fmaxf(fmaxf(sc[n][e], sc[n][e + 4]), fmaxf(sc[n][e + 8], sc[n][e + 12]));
            const float mx = across32(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]))) * cc;
            if (__any(mx > st.m + 8.0f)) {
                const float mn = fmaxf(st.m, mx), f = exp2_hw(st.m - finite_max(mn));
                st.l *= f;
#pragma unroll
                for (int i = 0; i < NB; ++i) o[i] *= f;
                st.m = mn;
            }
            mu = finite_max(st.m);
        };
        // weights of 16 keys
        auto weights = [&](int n) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = exp2_hw(__builtin_fmaf(sc[n / 2][(n % 2) * 8 + i], cc, -mu));
            st.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            split8<QT>(p, pt[n]);
        };
        // their products with the values
        auto values = [&](int n) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                bf8 v[KT];
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    const uint32_t at = t * G::PLANE + n * 16 * D * 2 + (vlds ^ i << 6);
                    const u32x2 a = read_tr(vs, at), b = read_tr(vs, at + 8 * D * 2);
                    v[t] = __builtin_bit_cast(bf8, u32x4{a[0], a[1], b[0], b[1]});
                }
                o[i] = product<KT, QT>(v, pt[n], o[i], mfma32);
            }
        };
        if (kw < sees_max) {
            if constexpr (QT == 3) {
                // the registers are full of q's terms: one thing after the other
#pragma unroll
                for (int n = 0; n < NN; ++n) {
                    scores(n);
                    __builtin_amdgcn_sched_barrier(0);
                    largest(n);
#pragma unroll
                    for (int h = 2 * n; h < 2 * n + 2; ++h) {
                        weights(h);
                        __builtin_amdgcn_sched_barrier(0);
                        values(h);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            } else {
                // the second half's scores (matrix) beside the first half's weights (vector)
                scores(0);
                largest(0);
                if constexpr (NN == 2) scores(1);
                weights(0);
                weights(1);
                values(0);
                values(1);
                if constexpr (NN == 2) {
                    largest(1);  // (what it scales down has to hold the first half)
                    weights(2);
                    weights(3);
                    values(2);
                    values(3);
                }
            }
        }
        if (G::BUF == 1) __syncthreads();
        if (more) {
            store_keys(next);
            store_values(key0 + BK, next);
        }
        if (G::BUF == 2) buf ^= 1;
        __syncthreads();
    }

    if (bad_page) flag(A.c.err, kAttnBadPage);
    // whether any thread staged a value that is not finite (the tiles' place is free)
    if (lane == 0) ((uint32_t *)sh)[wave] = 0;
    if (bad) ((uint32_t *)sh)[wave] = 1;
    __syncthreads();
    const u32x4 bads = *(const u32x4 *)sh;
    const bool any_bad = bads[0] | bads[1] | bads[2] | bads[3];
    if constexpr (KS == 2) __syncthreads();
    const uint32_t etid = thread_id(), ecol = etid & 31, eg = etid >> 5 & 1, elane = etid & 63;
    st.l += __shfl_xor(st.l, 32);
    if constexpr (KS == 2) {
        static_assert(2 * (32 * D + 64) * 4 <= G::LDS, "the sums fit the tiles' place");
        // the second two waves' sums to the first two
        float *const to = (float *)sh + wrow / 32 * (32 * D + 64);
        if (kq) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *(f32x4 *)(to + (i * 4 + e / 4) * 256 + elane * 4) = f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
            if (eg == 0) {
                to[32 * D + ecol] = st.m;
                to[32 * D + 32 + ecol] = st.l;
            }
        }
        __syncthreads();
        if (kq) return;
        const float om = to[32 * D + ecol], m = fmaxf(st.m, om), f0 = exp2_hw(st.m - finite_max(m)), f1 = exp2_hw(om - finite_max(m));
        st.l = __builtin_fmaf(to[32 * D + 32 + ecol], f1, st.l * f0);
        st.m = m;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const f32x4 z = *(const f32x4 *)(to + (i * 4 + e / 4) * 256 + elane * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][e + j] = __builtin_fmaf(z[j], f1, o[i][e + j] * f0);
            }
    }
    if (any_bad) add_not_finite<C, D, true>(A.c, it, max(first, cut / BK * BK), min(stop, it.len), sees, o);
    const uint32_t rr = wrow + ecol, er = it.rt * G::BM + rr;
    if (er >= rows) return;
    const uint32_t etok = er / A.group, ex = it.h * A.group + er - etok * A.group;
    const uint64_t erow = (uint64_t)(it.r0 + (int32_t)etok);
    const float vsc = C == kE4M3 && A.c.v_scale ? A.c.v_scale[it.h] : 1.0f;
    if (parts > 1) {
        float *const part = (float *)A.work + kPlanFloats + (uint64_t)it.slot * G::SLOT;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *(f32x4 *)(part + rr * D + i * 32 + e * 2 + eg * 4) = f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
        if (eg == 0) {
            part[G::BM * D + rr] = st.m;
            part[G::BM * D + G::BM + rr] = st.l;
        }
        return;
    }
    const float f = it.len - it.nq + (int32_t)etok + 1 > 0 ? vsc / st.l : 0.0f;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            write4<R>(A, erow, ex, D, i * 32 + e * 2 + eg * 4, f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]}, f);
}

// The instance for a row type, cache type and head dimension.
template <typename F>
void pick(uint32_t row_t, uint32_t cache_t, uint32_t dim, F &&f) {
    auto by_dim = [&](auto r, auto c) {
        if (dim == 64) f(r, c, std::integral_constant<int, 64>{});
        else if (dim == 128) f(r, c, std::integral_constant<int, 128>{});
        else f(r, c, std::integral_constant<int, 256>{});
    };
    using F32 = std::integral_constant<uint32_t, kF32>;
    using BF16 = std::integral_constant<uint32_t, kBF16>;
    using E4M3 = std::integral_constant<uint32_t, kE4M3>;
    if (row_t == kF32 && cache_t == kF32) by_dim(F32{}, F32{});
    else if (row_t == kF32 && cache_t == kBF16) by_dim(F32{}, BF16{});
    else if (row_t == kF32) by_dim(F32{}, E4M3{});
    else if (cache_t == kBF16) by_dim(BF16{}, BF16{});
    else by_dim(BF16{}, E4M3{});
}

}  // namespace

// Rows from which a workgroup takes four.
constexpr uint32_t kAppendBlockRows = 2048;

void launch_append(const AppendArgs &A, uint32_t row_t, uint32_t dim, hipStream_t st) {
    pick(row_t, A.c.dtype, dim, [&](auto r, auto c, auto d) {
        constexpr uint32_t groups = 256 / (d() / 8);
        if (A.c.rows >= kAppendBlockRows)
            k_append<r(), c(), d(), 4><<<(A.c.rows + 3) / 4, 256, 0, st>>>(A);
        else
            k_append<r(), c(), d(), 1><<<dim3(A.c.rows, (A.q_heads + 2 * A.c.kv_heads + groups - 1) / groups), 256, 0, st>>>(A);
    });
}

namespace {

enum Kernel { kSplit, kTile64, kTile128 };

struct Plan {
    Kernel kernel;
    uint32_t tiles, slots;  // row tiles x key heads at most; workgroups or parts that share them (0: one for each tile)
    uint32_t unit;          // kSplit: keys that go to a workgroup together
};

Plan plan(const AttnArgs &A, uint32_t dim) {
    Plan p;
    const uint64_t rows = (uint64_t)A.c.rows * A.group, longest = (uint64_t)A.c.max_pages * A.c.page_size;
    const bool f32 = A.c.dtype == kF32;
    // a sequence's last tile may be in part empty
    auto tiles = [&](uint32_t bm) { return (uint32_t)std::min<uint64_t>(rows / bm + A.c.n, rows) * A.c.kv_heads; };
    // Up to 16 rows a sequence the keys are read once by the kernel that streams them; 64-row tiles to 64 rows a
    // sequence, and on short contexts while 128-row ones would not fill the CUs (no such instance for an f32 cache
    // of 256: its tile does not fit the LDS).
    const bool t64 = !(f32 && dim == 256);
    p.kernel = rows <= 16ull * A.c.n ? kSplit
               : t64 && (rows <= 64ull * A.c.n || (tiles(128) < 256 && longest <= 2048)) ? kTile64 : kTile128;
    if (p.kernel != kSplit) {
        // one or two workgroups on a CU (TileCfg::OCC), in up to two rounds; a few units are not worth joining
        const uint32_t chip = dim == 256 || (f32 && (dim == 128 || p.kernel == kTile64)) ? 256 : 512;
        p.tiles = tiles(p.kernel == kTile64 ? 64 : 128);
        p.slots = p.tiles < chip && longest > 512 ? 2 * chip : 0;
        p.unit = 0;
        return p;
    }
    // as many workgroups as are on the chip at once, or tiles where those are more: shorter shares, which
    // the chip takes in turn; many tiles need no sharing
    const uint32_t chip = dim == 256 || (f32 && dim == 128) ? 256 : 512;
    p.tiles = tiles(16);
    p.unit = f32 && dim == 256 ? 64 : A.c.dtype == kE4M3 && dim <= 128 ? 256 : 128;  // SplitCfg::UNIT
    p.slots = p.tiles < 2048 && longest > p.unit ? std::max(chip, p.tiles) : 0;
    // (all units are counted in 32 bits)
    while (p.slots && (uint64_t)p.tiles * (longest / p.unit + 2) > 0x7fffffffull) p.unit *= 2;
    return p;
}

}  // namespace

uint64_t attn_work_bytes(const AttnArgs &A, uint32_t dim) {
    const Plan p = plan(A, dim);
    const uint64_t rows = p.kernel == kSplit ? 2 * 16 : p.kernel == kTile64 ? 64 : 128;
    return (kPlanFloats + p.slots * rows * (dim + 2)) * 4;
}

void launch_attn(const AttnArgs &A, uint32_t row_t, uint32_t dim, hipStream_t st) {
    const Plan p = plan(A, dim);
    auto join = [&](auto r, auto c, auto d, auto bm, auto unit) {
        // with many parts a tile, a workgroup joins 32 numbers of a row or two rows, else as many rows as its lanes hold
        constexpr int all = 1024 / d() < bm() ? 1024 / d() : bm();
        if (!p.slots) return;
        if (p.slots <= 16 * p.tiles)
            k_attn_join<r(), c(), d(), bm(), unit(), d() / 4, all><<<p.tiles * (bm() / all), 256, 0, st>>>(A, p.slots, p.unit);
        else if constexpr (bm() == 16)
            k_attn_join<r(), c(), d(), bm(), unit(), 8, 1><<<dim3(p.tiles * bm(), d() / 32), 256, 0, st>>>(A, p.slots, p.unit);
        else
            k_attn_join<r(), c(), d(), bm(), unit(), d() / 4, 2><<<p.tiles * (bm() / 2), 256, 0, st>>>(A, p.slots, p.unit);
    };
    pick(row_t, A.c.dtype, dim, [&](auto r, auto c, auto d) {
        auto tile = [&](auto ks) {
            using G = TileCfg<r(), c(), d(), ks()>;
            if constexpr (G::FITS) {
                k_attn_tile<r(), c(), d(), ks()><<<std::max(p.tiles, p.slots), 256, 0, st>>>(A, p.slots);
                join(r, c, d, std::integral_constant<int, G::BM>{}, std::integral_constant<int, G::BK>{});
            }
        };
        if (p.kernel == kTile128) {
            tile(std::integral_constant<int, 1>{});
        } else if (p.kernel == kTile64) {
            tile(std::integral_constant<int, 2>{});
        } else {
            using G = SplitCfg<r(), c(), d()>;
            k_attn_split<r(), c(), d()><<<p.slots ? p.slots : p.tiles, 64 * G::W, 0, st>>>(A, p.slots, p.unit);
            join(r, c, d, std::integral_constant<int, 16>{}, std::integral_constant<int, 0>{});
        }
    });
}

}  // namespace cz
