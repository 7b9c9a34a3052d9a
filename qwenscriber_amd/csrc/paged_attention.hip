// Attention of new tokens over a paged q8 cache (kernels.zig:697-767
// decodeAttentionStepQ8 for every new token, over its sequence's pages).
#include <cfloat>

#include "common.h"
#include "paged.h"

namespace qwh {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// One wavefront per row and query head: 64 positions a round, a lane scoring
// one of them over the whole head row, then every lane adding up its
// dimensions of the weighted values.
template <int D>
__global__ __launch_bounds__(64) void paged_attention_simple_kernel(const PagedAttentionArgs a, float scaling) {
    const int lane = threadIdx.x;
    const uint32_t h = blockIdx.x, row = blockIdx.y * 65535u + blockIdx.z;
    __shared__ float q[D];
    __shared__ float w[64];
    __shared__ uint32_t rows[64];
    uint32_t b, t;
    if (row >= a.batch.rows || !paged_row(a.batch, row, lane, b, t)) return;
    const uint32_t kvh = h / (a.heads / a.cache.kv_heads);
    const uint32_t kv_width = a.cache.kv_heads * D, gpr = kv_width / 64;
    for (int d = lane; d < D; d += 64) q[d] = a.query[(size_t)row * a.query_stride + h * D + d];
    __syncthreads();
    const uint64_t held = (uint64_t)a.batch.table_pages * a.cache.page_size;
    uint64_t end = (uint64_t)a.batch.first[b] + t + 1;
    if (end > held) end = held;
    const uint32_t *table = a.batch.tables + (size_t)b * a.batch.table_pages;
    const uint16_t *k_scales = reinterpret_cast<const uint16_t *>(a.cache.k_scales);
    const uint16_t *v_scales = reinterpret_cast<const uint16_t *>(a.cache.v_scales);
    float m = -INFINITY, l = 0.0f, acc[D / 64];
    for (int i = 0; i < D / 64; ++i) acc[i] = 0.0f;
    for (uint64_t base = 0; base < end; base += 64) {
        const uint32_t r = base + lane < end ? paged_pool_row(a.cache, table, (uint32_t)(base + lane)) : kNoRow;
        float s = -INFINITY;
        if (r != kNoRow) {
            const uint8_t *k = a.cache.k_codes + (size_t)r * kv_width + kvh * D;
            float dot = 0.0f;
            for (int g = 0; g < D / 64; ++g) {
                float part = 0.0f;
                for (int d = 0; d < 64; ++d) part = fmaf(q[64 * g + d], (float)((int)k[64 * g + d] - 128), part);
                dot = fmaf(dev::f16_bits_to_f32(k_scales[(size_t)r * gpr + kvh * (D / 64) + g]), part, dot);
            }
            s = dot * scaling;
        }
        const float m_new = fmaxf(m, dev::wave_max(s));
        if (m_new == -INFINITY) continue;
        const float alpha = exp2f(m - m_new);
        const float e = r != kNoRow ? exp2f(s - m_new) : 0.0f;
        l = l * alpha + dev::wave_sum(e);
        m = m_new;
        w[lane] = e;
        rows[lane] = r;
        __syncthreads();
        for (int i = 0; i < D / 64; ++i) {
            float sum = 0.0f;
            for (int p = 0; p < 64; ++p) {
                if (rows[p] == kNoRow) continue;
                const size_t vr = rows[p];
                sum = fmaf(w[p] * dev::f16_bits_to_f32(v_scales[vr * gpr + kvh * (D / 64) + i]),
                           (float)((int)a.cache.v_codes[vr * kv_width + kvh * D + 64 * i + lane] - 128), sum);
            }
            acc[i] = acc[i] * alpha + sum;
        }
        __syncthreads();
    }
    for (int i = 0; i < D / 64; ++i)
        a.out[((size_t)row * a.heads + h) * D + 64 * i + lane] = l == 0.0f ? 0.0f : acc[i] / l;
}

}  // namespace

size_t paged_attention_scratch_bytes(int, const PagedAttentionArgs &) { return 256; }

hipError_t launch_paged_attention(hipStream_t s, int, const PagedAttentionArgs &a, void *, size_t) {
    const uint32_t rows = a.batch.row_starts ? a.batch.rows : a.batch.batch;
    const float scaling = kLog2e / sqrtf((float)a.cache.head_dim);
    const dim3 grid(a.heads, (rows + 65534) / 65535, rows < 65535 ? rows : 65535);
    switch (a.cache.head_dim) {
    case 64: paged_attention_simple_kernel<64><<<grid, 64, 0, s>>>(a, scaling); break;
    case 128: paged_attention_simple_kernel<128><<<grid, 64, 0, s>>>(a, scaling); break;
    case 192: paged_attention_simple_kernel<192><<<grid, 64, 0, s>>>(a, scaling); break;
    case 256: paged_attention_simple_kernel<256><<<grid, 64, 0, s>>>(a, scaling); break;
    default: return hipErrorNotSupported;
    }
    return hipGetLastError();
}

}  // namespace qwh
