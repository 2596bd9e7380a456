// cz_attn.hip - attention over a paged key-value cache: new keys and values into
// the cache, one new token per sequence, and prompts.
//
// A sequence's new tokens are the last of its len tokens: row i of new rows sits
// at position len - new + i and sees the positions up to its own.
#include "cz_attn.h"

#include "cz_device.h"

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
    const uint32_t p = (uint32_t)c.table[(uint64_t)b * c.max_pages + i];
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
// A workgroup per row and query head; its four waves take every fourth key and
// are joined at the end.
template <uint32_t R, uint32_t C, int D>
__global__ __launch_bounds__(256) void k_attn(AttnArgs A) {
    constexpr int N = D / 64;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64, heads = A.group * A.c.kv_heads;
    const uint32_t t = blockIdx.x / heads, x = blockIdx.x % heads, h = x / A.group;
    const uint32_t b = sequence_of(A.c, t);
    if (b >= A.c.n) return;
    const Seq s = sequence(A.c, b);
    if ((int32_t)t < s.r0 || (int32_t)t >= s.r0 + s.nq) return;
    const int32_t sees = s.len - s.nq + ((int32_t)t - s.r0) + 1;
    const float c = A.scale * (C == kE4M3 && A.c.k_scale ? A.c.k_scale[h] : 1.0f);
    float q[N], o[N], m = -INFINITY, l = 0;
    for (int i = 0; i < N; ++i) {
        q[i] = load1<R>(A.q, (uint64_t)t * A.q_stride + (uint64_t)x * D + i * 64 + lane);
        o[i] = 0;
    }
    for (int32_t j = wave; j < sees; j += 4) {
        const uint64_t at = page_at(A.c, b, j / A.c.page_size) * A.c.page_stride + h * A.c.head_stride +
                            (j % A.c.page_size) * A.c.token_stride + lane;
        float p = 0;
        for (int i = 0; i < N; ++i) p = __builtin_fmaf(q[i], load1<C>(A.c.k, at + i * 64), p);
        for (int w = 32; w; w >>= 1) p += __shfl_xor(p, w);
        p *= c;
        const float mn = fmaxf(m, p), f = m == mn ? 1.0f : cz_expf(m - mn);
        const float e = p == -INFINITY ? 0.0f : cz_expf(p - mn);
        m = mn;
        l = l * f + e;
        for (int i = 0; i < N; ++i) o[i] = __builtin_fmaf(e, load1<C>(A.c.v, at + i * 64), o[i] * f);
    }
    __shared__ float so[4][D], sm[4], sl[4];
    for (int i = 0; i < N; ++i) so[wave][i * 64 + lane] = o[i];
    sm[wave] = m;
    sl[wave] = l;
    __syncthreads();
    if (wave) return;
    const float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float lt = 0, f[4];
    for (int w = 0; w < 4; ++w) {
        f[w] = sm[w] == mx ? 1.0f : cz_expf(sm[w] - mx);
        lt += sl[w] * f[w];
    }
    const float vs = C == kE4M3 && A.c.v_scale ? A.c.v_scale[h] : 1.0f;
    for (int i = 0; i < N; ++i) {
        float y = 0;
        for (int w = 0; w < 4; ++w) y = __builtin_fmaf(so[w][i * 64 + lane], f[w], y);
        y = sees > 0 ? y / lt * vs : 0.0f;
        store1<R>(A.out, (uint64_t)t * A.out_stride + (uint64_t)x * D + i * 64 + lane, y);
    }
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

uint64_t attn_work_bytes(const AttnArgs &, uint32_t) { return 16; }

void launch_attn(const AttnArgs &A, uint32_t row_t, uint32_t dim, hipStream_t st) {
    pick(row_t, A.c.dtype, dim, [&](auto r, auto c, auto d) {
        k_attn<r(), c(), d()><<<A.c.rows * A.group * A.c.kv_heads, 256, 0, st>>>(A);
    });
}

}  // namespace cz
