// cz_attn.hip - attention over a paged key-value cache: new keys and values into
// the cache, one new token per sequence, and prompts.
//
// A sequence's new tokens are the last of its len tokens: row i of new rows sits
// at position len - new + i and sees the positions up to its own.
#include "cz_attn.h"

#include "cz_device.h"

#include <algorithm>
#include <type_traits>

namespace cz {
namespace {

__device__ __forceinline__ void flag(uint32_t *err, AttnError what) {
    __hip_atomic_store(err + what, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

__device__ __forceinline__ uint16_t bf16_rne(float x) {
    const __bf16 b = (__bf16)x;
    uint16_t u;
    __builtin_memcpy(&u, &b, 2);
    return u;
}
__device__ __forceinline__ float bf16_f32(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// Nearest E4M3 byte (ties to even), saturating at 448; a NaN stays one.
__device__ __forceinline__ uint8_t e4m3_rne(float x) {
    const float c = x != x ? x : fminf(fmaxf(x, -448.0f), 448.0f);
    return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false) & 255);
}

template <uint32_t T>
__device__ __forceinline__ float load1(const void *p, uint64_t i) {
    if constexpr (T == kF32) return ((const float *)p)[i];
    if constexpr (T == kBF16) return bf16_f32(((const uint16_t *)p)[i]);
    if constexpr (T == kE4M3) return __builtin_amdgcn_cvt_f32_fp8(((const uint8_t *)p)[i], 0);
}
template <uint32_t T>
__device__ __forceinline__ void store1(void *p, uint64_t i, float x) {
    if constexpr (T == kF32) ((float *)p)[i] = x;
    if constexpr (T == kBF16) ((uint16_t *)p)[i] = bf16_rne(x);
    if constexpr (T == kE4M3) ((uint8_t *)p)[i] = e4m3_rne(x);
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

// The sequence of a row, or n where the row belongs to none.
__device__ __forceinline__ uint32_t sequence_of(const AttnCache &c, uint32_t row) {
    if (!c.row0) return row;
    uint32_t lo = 0, hi = c.n;  // first b with row0[b + 1] > row
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (c.row0[mid + 1] > (int32_t)row) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// A page number of the table; one outside the cache is flagged and read as 0.
__device__ __forceinline__ uint32_t page_at(const AttnCache &c, uint32_t b, uint32_t i) {
    // uniform: a scalar load
    const uint32_t p = (uint32_t)*(const __attribute__((address_space(4))) int32_t *)(uintptr_t)(c.table + (uint64_t)b * c.max_pages + i);
    if (p < c.pages) return p;
    flag(c.err, kAttnBadPage);
    return 0;
}

// ---- append -------------------------------------------------------------------
// A wave per head vector: head x of row t, of the query (rotated into q_out),
// then the keys, then the values.  A pair of the rotation sits in one lane.
template <uint32_t R, uint32_t C, int D>
__global__ __launch_bounds__(256) void k_append(AppendArgs A) {
    constexpr int N = D / 64;
    const uint32_t lane = threadIdx.x & 63, heads = A.q_heads + 2 * A.c.kv_heads;
    const uint64_t item = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
    const uint32_t t = (uint32_t)(item / heads), x = (uint32_t)(item % heads);
    if (t >= A.c.rows) return;
    const uint32_t b = sequence_of(A.c, t);
    if (b >= A.c.n) return;
    const Seq s = sequence(A.c, b);
    const int32_t pos = s.len - s.nq + ((int32_t)t - s.r0);
    if (pos < 0) return;
    const uint32_t kind = x < A.q_heads ? 0 : x < A.q_heads + A.c.kv_heads ? 1 : 2;
    const uint32_t h = kind == 0 ? x : kind == 1 ? x - A.q_heads : x - A.q_heads - A.c.kv_heads;
    const void *src = kind == 0 ? A.q : kind == 1 ? A.k : A.v;
    const uint64_t at = (uint64_t)t * (kind == 0 ? A.q_stride : kind == 1 ? A.k_stride : A.v_stride) + (uint64_t)h * D;
    if (kind != 2 && A.rope && (uint32_t)pos >= A.positions) {
        flag(A.c.err, kAttnBadPosition);
        return;
    }
    float y[N];
    const float *w = kind == 0 ? A.q_norm : kind == 1 ? A.k_norm : nullptr;
    float ss = 0;
    for (int i = 0; i < N; ++i) {
        y[i] = load1<R>(src, at + i * 64 + lane);
        ss = __builtin_fmaf(y[i], y[i], ss);
    }
    if (w) {
        for (int m = 32; m; m >>= 1) ss += __shfl_xor(ss, m);
        const float r = 1.0f / __builtin_sqrtf(ss / D + A.eps);
        for (int i = 0; i < N; ++i) y[i] = y[i] * r * w[i * 64 + lane];
    }
    __shared__ float sh[4][D];
    float *mine = sh[threadIdx.x / 64];
    if (kind != 2 && A.rope) {
        for (int i = 0; i < N; ++i) mine[i * 64 + lane] = y[i];
        __builtin_amdgcn_wave_barrier();
        const float *cs = A.rope + (uint64_t)pos * A.dims;
        const uint32_t half = A.dims / 2;
        for (int i = 0; i < N; ++i) {
            const uint32_t d = i * 64 + lane;
            if (d < half) y[i] = mine[d] * cs[d] - mine[d + half] * cs[half + d];
            else if (d < A.dims) y[i] = mine[d] * cs[d - half] + mine[d - half] * cs[d];
        }
    }
    if (kind == 0) {
        for (int i = 0; i < N; ++i) store1<R>(A.q_out, (uint64_t)t * A.q_out_stride + (uint64_t)h * D + i * 64 + lane, y[i]);
        return;
    }
    const uint32_t page = (uint32_t)A.c.table[(uint64_t)b * A.c.max_pages + pos / A.c.page_size];
    if (page >= A.c.pages) {
        flag(A.c.err, kAttnBadPage);
        return;
    }
    const uint64_t to = page * A.c.page_stride + h * A.c.head_stride + (pos % A.c.page_size) * A.c.token_stride;
    const float *sc = kind == 1 ? A.c.k_scale : A.c.v_scale;
    for (int i = 0; i < N; ++i) {
        const float z = C == kE4M3 && sc ? y[i] / sc[h] : y[i];
        store1<C>(kind == 1 ? A.c.k : A.c.v, to + i * 64 + lane, z);
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

// x in N terms: one rounds to nearest.  Infinities have no lower terms (inf - inf);
// a NaN stays one in some term.
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf8 (&t)[N]) {
    if constexpr (N == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[0][i] = (__bf16)x[i];
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
    __device__ __forceinline__ void zero() { a = b = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void terms(bf8 (&t)[3]) const {
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = __uint_as_float(a[i]);
            x[4 + i] = __uint_as_float(b[i]);
        }
        split8<3>(x, t);
    }
};
template <>
struct Eight<kBF16> {
    u32x4 a;
    __device__ __forceinline__ void load(const uint8_t *p) { a = *(const u32x4 *)p; }
    __device__ __forceinline__ void zero() { a = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void terms(bf8 (&t)[1]) const { t[0] = __builtin_bit_cast(bf8, a); }
};
template <>
struct Eight<kE4M3> {
    u32x2 a;
    __device__ __forceinline__ void load(const uint8_t *p) { a = *(const u32x2 *)p; }
    __device__ __forceinline__ void zero() { a = u32x2{0, 0}; }
    __device__ __forceinline__ void terms(bf8 (&t)[1]) const { t[0] = e4m3x8(a[0], a[1]); }
};

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
// row: the pieces of a row are permuted by the key so that 8 lanes' pieces of K (8
// keys), and the 4 keys x 32 bytes that 16 lanes read of V, fall on different
// banks.  Keys 8 apart are permuted alike: one address serves both.
template <int D>
__device__ __forceinline__ uint32_t lds_at(uint32_t key, uint32_t chunk) {
    const uint32_t f = ((key & 7) << 1) & (D / 8 - 1);
    return key * (D * 2) + ((chunk ^ f) << 4);
}

// Halves (bf16) of w that are not finite, as a mask.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}
// Values that are not finite become 0, in all their terms; whether there were any.
template <int N>
__device__ __forceinline__ bool clean(bf8 (&v)[N]) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t bad = 0;
#pragma unroll
        for (int t = 0; t < N; ++t) bad |= not_finite(__builtin_bit_cast(u32x4, v[t])[i]);
#pragma unroll
        for (int t = 0; t < N; ++t) {
            u32x4 w = __builtin_bit_cast(u32x4, v[t]);
            w[i] &= ~bad;
            v[t] = __builtin_bit_cast(bf8, w);
        }
        any |= bad;
    }
    return any != 0;
}

// One part of the work: keys of a row tile of a key head.
struct Item {
    uint32_t b, rt, h, part, parts, slot;
    int32_t r0, nq, len;
};

// Item `idx` of a call, found by every wave for itself.  Row tiles of BM rows,
// keys in units of UNIT.  Where there are fewer tiles than `slots` workgroups
// (0: never), each sequence's tiles are cut into parts of at most C units, C the
// smallest that keeps the parts within `slots`: ragged lengths share the chip
// evenly.  Order: sequence, tile (the last first: it sees most), part, key head -
// heads innermost, so that a head's workgroups stay on the same XCDs' L2.
// JOIN: an item per tile instead of one per part.
template <int BM, int UNIT, bool JOIN>
__device__ __forceinline__ bool find_item(const AttnCache &c, uint32_t group, uint32_t slots, uint32_t idx, Item &it) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t C = 0xffffffffu;
    if (slots) {
        float total = 0;
        uint32_t tiles = 0;
        for (uint32_t b0 = 0; b0 < c.n; b0 += 64) {
            if (b0 + lane < c.n) {
                const Seq s = sequence(c, b0 + lane);
                const uint32_t t = ((uint32_t)s.nq * group + BM - 1) / BM;
                tiles += t;
                total += (float)t * (float)((s.len + UNIT - 1) / UNIT);
            }
        }
#pragma unroll
        for (int m = 32; m; m >>= 1) {
            total += __shfl_xor(total, m);
            tiles += __shfl_xor(tiles, m);
        }
        const uint32_t room = slots / c.kv_heads;
        if (tiles < room) C = max(1u, (uint32_t)__builtin_ceilf(total / (float)(room - tiles) * 1.00001f));
    }
    uint32_t base = 0, slot0 = 0;
    for (uint32_t b0 = 0; b0 < c.n; b0 += 64) {
        Seq s{0, 0, 0};
        uint32_t t = 0, parts = 1;
        if (b0 + lane < c.n) {
            s = sequence(c, b0 + lane);
            t = ((uint32_t)s.nq * group + BM - 1) / BM;
            const uint32_t u = (uint32_t)(s.len + UNIT - 1) / UNIT;
            if (C != 0xffffffffu) parts = max(1u, (u + C - 1) / C);
        }
        const uint32_t all = t * parts * c.kv_heads, mine = JOIN ? t * c.kv_heads : all;
        uint32_t end = mine, send = all;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t x = __shfl_up(end, m), y = JOIN ? __shfl_up(send, m) : 0;
            if ((int)lane >= m) {
                end += x;
                send += y;
            }
        }
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

// Element offsets of a sequence's runs of 16 keys, one after the other; past the
// last key the last run again (its loads stay in bounds, its keys are masked).
struct Runs {
    uint32_t j, slot, last;  // next run's page index and slot; runs left
    __device__ __forceinline__ void start(const AttnCache &c, uint32_t run, int32_t keys) {
        const uint32_t n = (uint32_t)(keys + 15) / 16, at = min(run, n ? n - 1 : 0);
        j = at * 16 / c.page_size;
        slot = at * 16 - j * c.page_size;
        last = n ? n - 1 - at : 0;
    }
    __device__ __forceinline__ uint64_t next(const AttnCache &c, const Item &it, uint64_t head) {
        const uint64_t at = page_at(c, it.b, j) * c.page_stride + slot * c.token_stride + head;
        if (last) {
            --last;
            slot += 16;
            if (slot >= c.page_size) {
                slot = 0;
                ++j;
            }
        }
        return at;
    }
    __device__ __forceinline__ void skip(const AttnCache &c, uint32_t runs) {
        for (uint32_t i = 0; i < runs && last; ++i) {
            --last;
            slot += 16;
            if (slot >= c.page_size) {
                slot = 0;
                ++j;
            }
        }
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
// added here, after the loop, to the rows that see them: products of indicators
// count the +inf and the -inf (a NaN is both) of each number in keys from .. to.
// Rare, so its reads are plain.  W32: results of 32 x 32 (a lane's numbers as in
// O^T), else 16 x 16; keys in the order of the weights.
template <uint32_t C, int D, bool W32, typename V, int NB>
__device__ __forceinline__ void add_not_finite(const AttnCache &c, const Item &it, int32_t from, int32_t to, int32_t sees,
                                               V (&o)[NB]) {
    constexpr int RUN = W32 ? 16 : 32, M = W32 ? 32 : 16;
    const uint32_t lane = threadIdx.x & 63, g = lane / M, col = lane % M;
#pragma unroll 1
    for (int32_t key0 = from; key0 < to; key0 += RUN) {
        int32_t key[8];
        bf8 vis;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            key[j] = key0 + (j / 4) * (RUN / 2) + (int32_t)g * 4 + j % 4;
            vis[j] = (__bf16)(key[j] < sees ? 1.0f : 0.0f);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            bf8 up, down;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t k = (uint32_t)min(key[j], to - 1);
                const uint32_t pg = (uint32_t)c.table[(uint64_t)it.b * c.max_pages + k / c.page_size];
                const float x = load1<C>(c.v, (pg < c.pages ? pg : 0) * c.page_stride + it.h * c.head_stride +
                                                  k % c.page_size * c.token_stride + i * M + col);
                const bool in = key[j] < to;
                up[j] = (__bf16)(in && (x != x || x == INFINITY) ? 1.0f : 0.0f);
                down[j] = (__bf16)(in && (x != x || x == -INFINITY) ? 1.0f : 0.0f);
            }
            V z;
#pragma unroll
            for (int e = 0; e < M * M / 64; ++e) z[e] = 0.0f;
            V n;
            if constexpr (W32) n = mfma32(up, vis, z); else n = mfma16(up, vis, z);
#pragma unroll
            for (int e = 0; e < M * M / 64; ++e)
                if (n[e] > 0.0f) o[i][e] += INFINITY;
            if constexpr (W32) n = mfma32(down, vis, z); else n = mfma16(down, vis, z);
#pragma unroll
            for (int e = 0; e < M * M / 64; ++e)
                if (n[e] > 0.0f) o[i][e] -= INFINITY;
        }
    }
}

// ---- few rows on long caches: the keys split over waves and workgroups -----------
// A workgroup takes 16 rows of one key head; its W waves take every W-th run
// of 32 keys, each loading its keys straight into matrix operand registers and its
// values through its own LDS tile.
template <uint32_t R, uint32_t C, int D>
struct SplitCfg {
    static constexpr int QT = kTerms<R>, KT = kTerms<C>, BM = 16, KEYS = 32;
    static constexpr int W = KT == 3 && D == 256 ? 2 : 4, UNIT = W * KEYS;  // waves: as many as their tiles fit the LDS
    static constexpr int TILE = KEYS * D * 2;            // bytes of one plane
    static constexpr int WAVE = TILE * KT > BM * D * 4 ? TILE * KT : BM * D * 4;
    static constexpr int SLOT = BM * (D + 2);            // floats of a part's sums
};

__device__ __forceinline__ u32x2 read_tr(const uint8_t *lds, uint32_t at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((CZ_LDS s16x4 *)(lds + at)));
}

template <uint32_t R, uint32_t C, int D>
__global__ __launch_bounds__((64 * SplitCfg<R, C, D>::W)) void k_attn_split(AttnArgs A, uint32_t slots) {
    using G = SplitCfg<R, C, D>;
    constexpr int QT = G::QT, KT = G::KT, W = G::W, NS = D / 32, NB = D / 16, NV = 32 * D / 8 / 64;
    __shared__ __align__(16) uint8_t sh[W * G::WAVE];
    __shared__ float sh_m[W][16], sh_l[W][16];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 4, col = lane & 15;
    Item it;
    if (!find_item<G::BM, G::UNIT, false>(A.c, A.group, slots, blockIdx.x, it)) return;
    int32_t end;
    uint32_t per, parts;
    tile_keys<G::BM, G::UNIT>(it, A.group, &end, &per, &parts);
    if (it.part >= parts) return;
    const int32_t first = (int32_t)(it.part * per * G::UNIT), stop = min(end, first + (int32_t)(per * G::UNIT));

    const uint32_t r = it.rt * 16 + col, rows = (uint32_t)it.nq * A.group;
    const bool valid = r < rows;
    const uint32_t tok = valid ? r / A.group : 0, x = it.h * A.group + (valid ? r - tok * A.group : 0);
    const uint64_t row = (uint64_t)(it.r0 + (int32_t)tok);
    const int32_t sees = valid ? min(max(it.len - it.nq + (int32_t)tok + 1, 0), end) : 0;
    const int32_t sees_min = __builtin_amdgcn_readfirstlane(sees);
    float c2 = A.scale * (C == kE4M3 && A.c.k_scale ? A.c.k_scale[it.h] : 1.0f) * 1.44269504088896340736f;
    const uint32_t flip = c2 < 0.0f ? 0x80000000u : 0u;
    c2 = fabsf(c2);

    bf8 q[NS][QT];
#pragma unroll
    for (int s = 0; s < NS; ++s) query8<R>(A.q, row * A.q_stride + (uint64_t)x * D + s * 32 + g * 8, flip, q[s]);

    f32x4 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) o[i] = f32x4{0, 0, 0, 0};
    Row st{-INFINITY, 0.0f};
    uint8_t *const lds = sh + wave * G::WAVE;

    const uint64_t head = it.h * A.c.head_stride;
    Runs runs;
    runs.start(A.c, (uint32_t)(first / 16) + wave * 2, end);
    Eight<C> kr[2][NS], vr[NV];
    const uint32_t ts = (uint32_t)A.c.token_stride, klane = (col * ts + g * 8) * kSize<C>;
    auto load = [&] {
        const uint8_t *kb[2], *vb[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint64_t at = runs.next(A.c, it, head) * kSize<C>;
            kb[n] = (const uint8_t *)A.c.k + at;
            vb[n] = (const uint8_t *)A.c.v + at;
        }
        runs.skip(A.c, 2 * (W - 1));
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int s = 0; s < NS; ++s)
                kr[n][s].load(kb[n] + (klane + s * 32 * kSize<C>));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t id = i * 64 + lane, key = id / (D / 8), ch = id % (D / 8);
            vr[i].load(vb[i * 64 / (D / 8) / 16] + ((key & 15) * ts + ch * 8) * kSize<C>);
        }
    };
    int32_t key0 = first + (int32_t)wave * 32, bad_at = -1;
    if (key0 < stop) load();
    for (; key0 < stop; key0 += G::UNIT) {
        f32x4 sc[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            sc[n] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                bf8 k[KT];
                kr[n][s].terms(k);
                sc[n] = product<KT, QT>(k, q[s], sc[n], mfma16);
            }
        }
        // values into the wave's tile; what is behind the sequence's end counts as 0
        const bool tail = key0 + 32 > it.len, masked = key0 + 32 > sees_min;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t id = i * 64 + lane, key = id / (D / 8), ch = id % (D / 8);
            if (tail && key0 + (int32_t)key >= it.len) vr[i].zero();
            bf8 v[KT];
            vr[i].terms(v);
            if (masked) bad |= clean(v);
#pragma unroll
            for (int t = 0; t < KT; ++t) *(bf8 *)(lds + t * G::TILE + lds_at<D>(key, ch)) = v[t];
        }
        if (bad_at < 0 && __any(bad)) bad_at = key0;
        if (key0 + G::UNIT < stop) load();

        float cc = c2;
        if (masked) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sc[n][i] = key0 + n * 16 + (int32_t)g * 4 + i < sees ? sc[n][i] * c2 : -INFINITY;
            cc = 1.0f;
        }
        float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                         fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
        mx = across32(across16(mx)) * cc;
        if (__any(mx > st.m + 8.0f)) {
            const float mn = fmaxf(st.m, mx), f = exp2_hw(st.m - finite_max(mn));
            st.l *= f;
#pragma unroll
            for (int i = 0; i < NB; ++i) o[i] *= f;
            st.m = mn;
        }
        const float mu = finite_max(st.m);
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = exp2_hw(__builtin_fmaf(sc[i / 4][i % 4], cc, -mu));
            st.l += p[i];
        }
        bf8 pt[QT];
        split8<QT>(p, pt);

        const uint32_t tk = g * 4 + (col >> 2), tc = (col & 3) >> 1, tb = (col & 1) * 8;
        auto values = [&](int i, bf8 (&v)[KT]) {
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const uint32_t at = t * G::TILE + lds_at<D>(tk, i * 2 + tc) + tb;
                const u32x2 a = read_tr(lds, at), b = read_tr(lds, at + 16 * D * 2);
                v[t] = __builtin_bit_cast(bf8, u32x4{a[0], a[1], b[0], b[1]});
            }
        };
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            bf8 v[KT];
            values(i, v);
            o[i] = product<KT, QT>(v, pt, o[i], mfma16);
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (bad_at >= 0)
        for (int32_t k = bad_at; k < stop; k += G::UNIT)
            add_not_finite<C, D, false>(A.c, it, k, min(k + 32, min(stop, it.len)), sees, o);

    // the waves' sums
    st.l += __shfl_xor(st.l, 16);
    st.l += __shfl_xor(st.l, 32);
    if (lane < 16) {
        sh_m[wave][col] = st.m;
        sh_l[wave][col] = st.l;
    }
    float *const mine = (float *)lds;
#pragma unroll
    for (int i = 0; i < NB; ++i) *(f32x4 *)(mine + col * D + ((i * 16 + g * 4) ^ ((col & 7) << 2))) = o[i];
    __syncthreads();
    float *const part = (float *)A.work + (uint64_t)it.slot * G::SLOT;
    const float vs = C == kE4M3 && A.c.v_scale ? A.c.v_scale[it.h] : 1.0f;
#pragma unroll
    for (int e = 0; e < 16 * D / 4 / (64 * W); ++e) {
        const uint32_t id = e * 64 * W + threadIdx.x, rr = id / (D / 4), d = id % (D / 4) * 4;
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
        if (parts > 1) {
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
}

// Joins the parts of a tile of BM rows: a workgroup per 16 rows.
template <uint32_t R, uint32_t C, int D, int BM, int UNIT>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs A, uint32_t slots) {
    Item it;
    const uint32_t sub = blockIdx.x % (BM / 16);
    if (!find_item<BM, UNIT, true>(A.c, A.group, slots, blockIdx.x / (BM / 16), it)) return;
    int32_t end;
    uint32_t per, parts;
    tile_keys<BM, UNIT>(it, A.group, &end, &per, &parts);
    if (parts == 1) return;
    const float vs = C == kE4M3 && A.c.v_scale ? A.c.v_scale[it.h] : 1.0f;
    const float *const first = (const float *)A.work + (uint64_t)it.slot * (BM * (D + 2));
    const uint64_t step = (uint64_t)A.c.kv_heads * (BM * (D + 2));
    const uint32_t rows = (uint32_t)it.nq * A.group;
#pragma unroll
    for (int e = 0; e < 16 * D / 4 / 256; ++e) {
        const uint32_t id = e * 256 + threadIdx.x, rr = sub * 16 + id / (D / 4), d = id % (D / 4) * 4;
        const uint32_t tr = it.rt * BM + rr;
        if (tr >= rows) continue;
        float m = -INFINITY, l = 0;
        for (uint32_t p = 0; p < parts; ++p) m = fmaxf(m, first[p * step + BM * D + rr]);
        const float mf = finite_max(m);
        f32x4 y{0, 0, 0, 0};
        for (uint32_t p = 0; p < parts; ++p) {
            const float *const s = first + p * step;
            const float f = exp2_hw(s[BM * D + rr] - mf);
            const f32x4 z = *(const f32x4 *)(s + rr * D + d);
            l = __builtin_fmaf(s[BM * D + BM + rr], f, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(z[i], f, y[i]);
        }
        const uint32_t t = tr / A.group;
        write4<R>(A, (uint64_t)it.r0 + t, it.h * A.group + tr - t * A.group, D, d, y,
                  it.len - it.nq + (int32_t)t + 1 > 0 ? vs / l : 0.0f);
    }
}

// ---- prompts ---------------------------------------------------------------------
// A workgroup takes 128 rows of one key head, 32 per wave, and walks over tiles of
// BK keys that its four waves share in LDS as bf16 planes: an E4M3 cache is widened
// and an f32 one split once, as the tile is staged.
template <uint32_t R, uint32_t C, int D>
struct TileCfg {
    static constexpr int QT = kTerms<R>, KT = kTerms<C>, BM = 128;
    static constexpr int BK = KT == 3 || D == 256 ? 32 : 64;
    static constexpr int PLANE = BK * D * 2, HALF = PLANE * KT;       // bytes of a tile's K, and of its V
    static constexpr int BUF = 4 * HALF <= 128 * 1024 ? 2 : 1;
    static constexpr int SLOT = BM * (D + 2);
};

template <uint32_t R, uint32_t C, int D>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void k_attn_tile(AttnArgs A, uint32_t slots) {
    using G = TileCfg<R, C, D>;
    constexpr int QT = G::QT, KT = G::KT, BK = G::BK, NS = D / 16, NB = D / 32, NN = BK / 32, NL = BK * D / 8 / 256;
    __shared__ __align__(16) uint8_t sh[G::BUF * 2 * G::HALF];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t g = lane >> 5, col = lane & 31;
    Item it;
    if (!find_item<G::BM, BK, false>(A.c, A.group, slots, blockIdx.x, it)) return;
    int32_t end;
    uint32_t per, parts;
    tile_keys<G::BM, BK>(it, A.group, &end, &per, &parts);
    if (it.part >= parts) return;
    const int32_t first = (int32_t)(it.part * per * BK), stop = min(end, first + (int32_t)(per * BK));

    const uint32_t rows = (uint32_t)it.nq * A.group, r = it.rt * G::BM + wave * 32 + col;
    const bool valid = r < rows;
    const uint32_t tok = valid ? r / A.group : 0, x = it.h * A.group + (valid ? r - tok * A.group : 0);
    const uint64_t row = (uint64_t)(it.r0 + (int32_t)tok);
    const int32_t sees = valid ? min(max(it.len - it.nq + (int32_t)tok + 1, 0), end) : 0;
    const int32_t sees_min = __builtin_amdgcn_readfirstlane(sees);
    // the wave's last row; a wave without rows sees nothing
    const uint32_t w0 = it.rt * G::BM + wave * 32, wl = min(w0 + 32, rows);
    const int32_t sees_max = w0 < rows ? min(max(it.len - it.nq + (int32_t)((wl - 1) / A.group) + 1, 0), end) : 0;
    float c2 = A.scale * (C == kE4M3 && A.c.k_scale ? A.c.k_scale[it.h] : 1.0f) * 1.44269504088896340736f;
    const uint32_t flip = c2 < 0.0f ? 0x80000000u : 0u;
    c2 = fabsf(c2);

    bf8 q[NS][QT];
#pragma unroll
    for (int s = 0; s < NS; ++s) query8<R>(A.q, row * A.q_stride + (uint64_t)x * D + s * 16 + g * 8, flip, q[s]);
    f32x16 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    Row st{-INFINITY, 0.0f};

    const uint64_t head = it.h * A.c.head_stride;
    Runs runs;
    runs.start(A.c, (uint32_t)(first / 16), end);
    Eight<C> kr[NL], vr[NL];
    // a thread's pieces: 8 numbers of key id / (D / 8), so a wave's are of one run
    const uint32_t ch = threadIdx.x % (D / 8), tkey = threadIdx.x / (D / 8);
    const uint32_t voff = ((tkey & 15) * (uint32_t)A.c.token_stride + ch * 8) * kSize<C>;
    constexpr int STEP = 256 / (D / 8);  // keys from one piece of a thread to its next
    const uint32_t vnext = STEP < 16 ? STEP * (uint32_t)A.c.token_stride * kSize<C> : 0;
    auto load = [&] {
        uint64_t base[BK / 16];
#pragma unroll
        for (int i = 0; i < BK / 16; ++i) base[i] = runs.next(A.c, it, head) * kSize<C>;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            // with 16 keys or more from piece to piece, waves are of different runs
            constexpr int PER = STEP >= 16 ? STEP / 16 : 1;
            uint64_t at = base[STEP >= 16 ? i * PER : i * STEP / 16];
            if constexpr (PER > 1) {
                const uint32_t run = wave * 64 / (D / 8) / 16;
#pragma unroll
                for (int n = 1; n < PER; ++n) at = run == n ? base[i * PER + n] : at;
            }
            const uint32_t off = voff + (STEP < 16 && i * STEP % 16 ? vnext : 0);
            kr[i].load((const uint8_t *)A.c.k + at + off);
            vr[i].load((const uint8_t *)A.c.v + at + off);
        }
    };
    // masks cut through the workgroup's tiles from here on
    const int32_t cut = min(max(it.len - it.nq + (int32_t)(it.rt * G::BM / A.group) + 1, 0), end);
    bool bad = false;
    auto store = [&](int32_t key0, uint8_t *to) {
        const bool tail = key0 + BK > it.len, masked = key0 + BK > cut;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const uint32_t key = i * STEP + tkey;
            if (tail && key0 + (int32_t)key >= it.len) vr[i].zero();
            bf8 k[KT], v[KT];
            kr[i].terms(k);
            vr[i].terms(v);
            if (masked) bad |= clean(v);
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                *(bf8 *)(to + t * G::PLANE + lds_at<D>(tkey, ch) + i * STEP * D * 2) = k[t];
                *(bf8 *)(to + G::HALF + t * G::PLANE + lds_at<D>(tkey, ch) + i * STEP * D * 2) = v[t];
            }
        }
    };
    uint32_t buf = 0;
    if (first < stop) {
        load();
        store(first, sh);
    }
    __syncthreads();
    for (int32_t key0 = first; key0 < stop; key0 += BK) {
        const bool more = key0 + BK < stop;
        if (more) load();
        const uint8_t *const ks = sh + buf * 2 * G::HALF, *const vs = ks + G::HALF;
        if (key0 < sees_max) {
            f32x16 sc[NN];
#pragma unroll
            for (int n = 0; n < NN; ++n) {
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[n][e] = 0.0f;
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    bf8 k[KT];
#pragma unroll
                    for (int t = 0; t < KT; ++t) k[t] = *(const bf8 *)(ks + t * G::PLANE + lds_at<D>(n * 32 + col, s * 2 + g));
                    sc[n] = product<KT, QT>(k, q[s], sc[n], mfma32);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            float cc = c2;
            const bool masked = key0 + BK > sees_min;
            if (masked) {
#pragma unroll
                for (int n = 0; n < NN; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        sc[n][e] = key0 + n * 32 + (e / 4) * 8 + (int32_t)g * 4 + e % 4 < sees ? sc[n][e] * c2 : -INFINITY;
                cc = 1.0f;
            }
            float mx = sc[0][0];
#pragma unroll
            for (int n = 0; n < NN; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[n][e]);
            mx = across32(mx) * cc;
            if (__any(mx > st.m + 8.0f)) {
                const float mn = fmaxf(st.m, mx), f = exp2_hw(st.m - finite_max(mn));
                st.l *= f;
#pragma unroll
                for (int i = 0; i < NB; ++i) o[i] *= f;
                st.m = mn;
            }
            const float mu = finite_max(st.m);
            // 16 keys at a time: weights, then their products
            const uint32_t tk = g * 4 + ((lane & 15) >> 2), tc = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), tb = (lane & 1) * 8;
#pragma unroll
            for (int n = 0; n < BK / 16; ++n) {
                float p[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    p[i] = exp2_hw(__builtin_fmaf(sc[n / 2][(n % 2) * 8 + i], cc, -mu));
                    st.l += p[i];
                }
                bf8 pt[QT];
                split8<QT>(p, pt);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    bf8 v[KT];
#pragma unroll
                    for (int t = 0; t < KT; ++t) {
                        const uint32_t at = t * G::PLANE + lds_at<D>(tk, i * 4 + tc) + tb + n * 16 * D * 2;
                        const u32x2 a = read_tr(vs, at), b = read_tr(vs, at + 8 * D * 2);
                        v[t] = __builtin_bit_cast(bf8, u32x4{a[0], a[1], b[0], b[1]});
                    }
                    o[i] = product<KT, QT>(v, pt, o[i], mfma32);
                }
            }
        }
        if (G::BUF == 1) __syncthreads();
        if (more) store(key0 + BK, sh + (G::BUF == 2 ? (buf ^ 1) : 0) * 2 * G::HALF);
        if (G::BUF == 2) buf ^= 1;
        __syncthreads();
    }

    if (__syncthreads_or(bad))
        add_not_finite<C, D, true>(A.c, it, max(first, cut / BK * BK), min(stop, it.len), sees, o);
    st.l += __shfl_xor(st.l, 32);
    if (!valid) return;
    const uint32_t rr = wave * 32 + col;
    const float vsc = C == kE4M3 && A.c.v_scale ? A.c.v_scale[it.h] : 1.0f;
    if (parts > 1) {
        float *const part = (float *)A.work + (uint64_t)it.slot * G::SLOT;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *(f32x4 *)(part + rr * D + i * 32 + e * 2 + g * 4) = f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
        if (g == 0) {
            part[G::BM * D + rr] = st.m;
            part[G::BM * D + G::BM + rr] = st.l;
        }
        return;
    }
    const float f = it.len - it.nq + (int32_t)tok + 1 > 0 ? vsc / st.l : 0.0f;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            write4<R>(A, row, x, D, i * 32 + e * 2 + g * 4, f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]}, f);
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

void launch_append(const AppendArgs &A, uint32_t row_t, uint32_t dim, hipStream_t st) {
    const uint64_t items = (uint64_t)A.c.rows * (A.q_heads + 2 * A.c.kv_heads);
    pick(row_t, A.c.dtype, dim, [&](auto r, auto c, auto d) {
        k_append<r(), c(), d()><<<(uint32_t)((items + 3) / 4), 256, 0, st>>>(A);
    });
}

namespace {

// Workgroups that share a call's work when its row tiles are fewer: two on a CU.
constexpr uint32_t kSplitSlots = 512, kTileSlots = 512;

struct Plan {
    bool tile;              // the prompt kernel
    uint32_t tiles, slots;  // row tiles x key heads at most; workgroups that share them (0: one for each tile)
};

Plan plan(const AttnArgs &A) {
    Plan p;
    const uint64_t rows = (uint64_t)A.c.rows * A.group;
    p.tile = A.c.row0 && rows > 64ull * A.c.n;
    const uint32_t bm = p.tile ? 128 : 16, want = p.tile ? kTileSlots : kSplitSlots;
    // a sequence's last tile may be in part empty
    p.tiles = (uint32_t)std::min<uint64_t>(rows / bm + A.c.n, rows) * A.c.kv_heads;
    p.slots = p.tiles < want ? want : 0;
    return p;
}

}  // namespace

uint64_t attn_work_bytes(const AttnArgs &A, uint32_t dim) {
    const Plan p = plan(A);
    return std::max<uint64_t>(16, (uint64_t)p.slots * (p.tile ? 128 : 16) * (dim + 2) * 4);
}

void launch_attn(const AttnArgs &A, uint32_t row_t, uint32_t dim, hipStream_t st) {
    const Plan p = plan(A);
    const uint32_t grid = std::max(p.tiles, p.slots);
    pick(row_t, A.c.dtype, dim, [&](auto r, auto c, auto d) {
        if (p.tile) {
            using G = TileCfg<r(), c(), d()>;
            k_attn_tile<r(), c(), d()><<<grid, 256, 0, st>>>(A, p.slots);
            if (p.slots) k_attn_join<r(), c(), d(), G::BM, G::BK><<<p.tiles * (G::BM / 16), 256, 0, st>>>(A, p.slots);
        } else {
            using G = SplitCfg<r(), c(), d()>;
            k_attn_split<r(), c(), d()><<<grid, 64 * G::W, 0, st>>>(A, p.slots);
            if (p.slots) k_attn_join<r(), c(), d(), G::BM, G::UNIT><<<p.tiles, 256, 0, st>>>(A, p.slots);
        }
    });
}

}  // namespace cz
