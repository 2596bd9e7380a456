// cz_attn.h - attention over a paged key-value cache: what the entry points
// (colizig_hip.hip) hand to the kernels (cz_attn.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cz {

enum AttnType : uint32_t { kF32 = 0, kBF16 = 1, kE4M3 = 2 };

// Words that the kernels set to 1 (host-coherent memory, read by
// colizig_hip_sync).
enum AttnError : uint32_t { kAttnBadPage = 0, kAttnBadLength = 1, kAttnBadPosition = 2, kAttnErrors = 3 };

// A paged cache and the sequences of one call.  Strides are in elements.
struct AttnCache {
    void *k, *v;
    const float *k_scale, *v_scale;  // [kv_heads] or null: all 1
    uint64_t page_stride, head_stride, token_stride;
    uint32_t pages, page_size, kv_heads, dtype;
    const int32_t *row0;   // [n + 1], or null: sequence b is row b
    const int32_t *len;    // [n]
    const int32_t *table;  // [n][max_pages]
    uint32_t n, rows, max_pages;
    uint32_t *err;         // [kAttnErrors]
};

struct AppendArgs {
    AttnCache c;
    const void *q, *k, *v;
    void *q_out;
    uint64_t q_stride, k_stride, v_stride, q_out_stride;
    uint32_t q_heads;
    const float *rope;  // [positions][dims]: dims / 2 cosines, dims / 2 sines; null: no rotation
    uint32_t positions, dims;
    const float *q_norm, *k_norm;  // [head_dim] or null
    float eps;
};

struct AttnArgs {
    AttnCache c;
    const void *q;
    void *out;
    uint64_t q_stride, out_stride;
    uint32_t group;  // query heads per key head
    float scale;
    void *work;
};

// The kernels of one call on `st`; the arguments have been checked.  row_t: the
// type of the rows (kF32 or kBF16).
void launch_append(const AppendArgs &A, uint32_t row_t, uint32_t dim, hipStream_t st);
void launch_attn(const AttnArgs &A, uint32_t row_t, uint32_t dim, hipStream_t st);
// Bytes of AttnArgs::work that launch_attn uses.
uint64_t attn_work_bytes(const AttnArgs &A, uint32_t dim);

}  // namespace cz
