// The paged cache's kernels: their arguments and the device helpers they
// share.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/qwhip.h"
#include "device.h"
#include "paged_plan.h"

namespace qwh {

constexpr uint32_t kNoRow = 0xffffffffu;

struct PagedAppendArgs {
    qwh_paged_cache cache;  // (planes of one layer)
    qwh_paged_batch batch;
    const float *qkv;
    uint32_t qkv_stride, heads;
    const float *q_norm, *k_norm, *rope_cos, *rope_sin;
    float eps;
    uint64_t positions;     // positions from here on are left out
    float *query;
    uint32_t query_stride;
    uint32_t units;         // wavefronts a row (set by the launch)
};

struct PagedAttentionArgs {
    qwh_paged_cache cache;  // (planes of one layer)
    qwh_paged_batch batch;
    float *out;
    const float *query;
    uint32_t query_stride, heads;
};

struct PagedCopyArgs {
    qwh_paged_cache cache;
    uint64_t code_page, scale_page;  // bytes of a page's rows
    uint32_t code_pieces, scale_pieces;  // of a page's keys or values in a layer
};

hipError_t launch_paged_append(hipStream_t s, const PagedAppendArgs &args);
hipError_t launch_paged_copy(hipStream_t s, const qwh_paged_cache &cache, const paged::CopyLaunch &launch, bool is_short);
size_t paged_attention_scratch_bytes(int cus, const PagedAttentionArgs &a);
hipError_t launch_paged_attention(hipStream_t s, int cus, const PagedAttentionArgs &a, void *scratch, size_t scratch_bytes);

// The planes of one layer of a pool.
inline qwh_paged_cache paged_layer(const qwh_paged_cache &c, uint32_t layer) {
    qwh_paged_cache one = c;
    const uint64_t rows = (uint64_t)c.pages * c.page_size * layer, width = (uint64_t)c.kv_heads * c.head_dim;
    one.k_codes += rows * width;
    one.v_codes += rows * width;
    one.k_scales += rows * (width / 64) * 2;
    one.v_scales += rows * (width / 64) * 2;
    return one;
}

#ifdef __HIPCC__
namespace {

// LDS stores of this wavefront before its later loads of other lanes' data.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The sequence of row `row` (< batch.rows) and its place among the sequence's
// new tokens, by a whole wavefront; false for a row of no sequence. Starts
// that never fall put as many of them at or below the row as there are
// sequences up to its own, so counting them needs one round of loads per 64
// sequences.
__device__ __forceinline__ bool paged_row(const qwh_paged_batch &batch, uint32_t row, int lane, uint32_t &b, uint32_t &t) {
    if (!batch.row_starts) {
        b = row;
        t = 0;
        return row < batch.batch;
    }
    uint32_t below = 0;
    for (uint32_t i = 0; i <= batch.batch; i += 64) {
        const bool le = i + lane <= batch.batch && batch.row_starts[i + lane] <= row;
        const uint32_t n = (uint32_t)__popcll(__ballot(le));
        below += n;
        if (n < 64) break;
    }
    if (below == 0 || below > batch.batch) return false;
    b = below - 1;
    t = row - batch.row_starts[b];
    return true;
}

// The pool row of position pos < table_pages * page_size, or kNoRow.
__device__ __forceinline__ uint32_t paged_pool_row(const qwh_paged_cache &c, const uint32_t *table, uint32_t pos) {
    const uint32_t at = pos / c.page_size;
    const uint32_t page = table[at];
    return page < c.pages ? page * c.page_size + (pos - at * c.page_size) : kNoRow;
}

__device__ __forceinline__ float quad_max(const float (&v)[4]) {
    return fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
}

// The largest of 8 or 16 aligned lanes.
template <int LANES>
__device__ __forceinline__ float group_max(float m) {
    m = fmaxf(m, dev::xor_lane<1>(m));
    m = fmaxf(m, dev::xor_lane<2>(m));
    m = fmaxf(m, dev::xor_lane<4>(m));
    if constexpr (LANES == 16) m = fmaxf(m, dev::xor_lane<8>(m));
    return m;
}

// Four values of a 64-value group whose largest magnitude is m as q8
// (quant.zig:209-288): their codes, and the group's scale by the lane that
// has a place for it.
__device__ __forceinline__ void store_q8x4_of(float m, const float (&v)[4], uint8_t *codes, uint16_t *scale) {
    const uint16_t bits = dev::f32_to_f16_bits(__fmul_rn(m, 0.0078125f));  // (m / 128: the same rounding)
    const float stored = dev::f16_bits_to_f32(bits);
    // The quotients as products with one reciprocal in f64, to 2^-50 of it.
    // Rounded to f32 they are the f32 quotients: a value of 24 bits by a scale
    // of 11 is 2^-37 or more of itself away from any middle of two f32.
    double inverse = __builtin_amdgcn_rcp((double)stored);
    inverse = fma(fma(-(double)stored, inverse, 1.0), inverse, inverse);
    inverse = fma(fma(-(double)stored, inverse, 1.0), inverse, inverse);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float scaled = stored == 0.0f ? 0.0f : (float)((double)v[i] * inverse);
        word |= (uint32_t)(dev::round_code(scaled, -128, 127) + 128) << (8 * i);
    }
    *reinterpret_cast<uint32_t *>(codes) = word;
    if (scale) *scale = bits;
}

// The same of a group that LANES aligned lanes hold.
template <int LANES>
__device__ __forceinline__ void store_q8x4(const float (&v)[4], uint8_t *codes, uint16_t *scale) {
    store_q8x4_of(group_max<LANES>(quad_max(v)), v, codes, scale);
}

}  // namespace
#endif

}  // namespace qwh
