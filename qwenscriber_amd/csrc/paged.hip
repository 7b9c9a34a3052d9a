// A q8 key/value cache in pages (the pool of qwh_paged_cache): the append of
// new tokens with their head norms and rotation, and copies of pages. The
// attention over the pages is in paged_attention.hip.
#include "common.h"
#include "device.h"
#include "paged.h"

namespace qwh {
namespace {

// ---- append ----
//
// decoder.zig:180-216 for every new token: y = x / sqrt(mean(x^2) + eps) * w
// per query and key head, the rotation of its position, the query row out,
// and key and value rows quantized into their page (quant.quantizeRow(.q8)).
//
// One wavefront a head row (a query head, a key head) or 256 values of the
// value row: no wavefront waits for another, and a step's few rows still
// spread over the device. The pair that the rotation mixes, dimensions d and
// d + D/2, is one lane's, so norm and rotation need one reduction and no
// exchange. Norm and rotation are in f64 (the square of an f32 is exact
// there): a key's code is a rounding of its value, and 32-bit sums put about
// one code in 10^5 on the other side of a border, by the order of the sum.
template <int D>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendArgs a) {
    constexpr int H = D / 2;
    constexpr int NP = (H + 63) / 64;  // pairs per lane
    __shared__ float lds_k[4][D];
    const uint32_t wave = threadIdx.x >> 6;
    const int lane = threadIdx.x & 63;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + wave;
    const uint32_t row = (uint32_t)(unit / a.units);
    const uint32_t u = (uint32_t)(unit % a.units);
    if (row >= a.batch.rows) return;
    uint32_t b, t;
    if (!paged_row(a.batch, row, lane, b, t)) return;
    const uint64_t position = (uint64_t)a.batch.first[b] + t;
    if (position >= a.positions) return;
    const uint32_t pos = (uint32_t)position;
    const uint32_t pool_row = paged_pool_row(a.cache, a.batch.tables + (size_t)b * a.batch.table_pages, pos);
    const float *src = a.qkv + (size_t)row * a.qkv_stride;
    const uint32_t kv_width = a.cache.kv_heads * D;
    const uint32_t gpr = kv_width / 64;
    if (u < a.heads + a.cache.kv_heads) {
        const bool is_key = u >= a.heads;
        if (is_key && pool_row == kNoRow) return;
        const float *x = src + (size_t)u * D;
        const float *w = is_key ? a.k_norm : a.q_norm;
        float lo[NP], hi[NP], wl[NP], wh[NP], c[NP], s[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int j = lane + 64 * i;
            const int jc = j < H ? j : 0;
            lo[i] = x[jc];
            hi[i] = x[jc + H];
            wl[i] = w[jc];
            wh[i] = w[jc + H];
            c[i] = a.rope_cos[(size_t)pos * H + jc];
            s[i] = a.rope_sin[(size_t)pos * H + jc];
        }
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (lane + 64 * i < H) ss += (double)lo[i] * lo[i] + (double)hi[i] * hi[i];
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 64);
        const double inv = 1.0 / sqrt(ss / D + (double)a.eps);
        float *q_out = a.query + (size_t)row * a.query_stride + (size_t)u * D;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int j = lane + 64 * i;
            if (j >= H) continue;
            const double yl = (double)lo[i] * inv * wl[i], yh = (double)hi[i] * inv * wh[i];
            const float rl = (float)(yl * c[i] - yh * s[i]), rh = (float)(yh * c[i] + yl * s[i]);
            float *out = is_key ? &lds_k[wave][0] : q_out;
            out[j] = rl;
            out[j + H] = rh;
        }
        if (!is_key) return;
        wave_fence();
        const uint32_t col = (u - a.heads) * D;
        if (lane * 4 < D) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = lds_k[wave][4 * lane + i];
            store_q8x4(v, lane, a.cache.k_codes + (size_t)pool_row * kv_width + col,
                       reinterpret_cast<uint16_t *>(a.cache.k_scales) + (size_t)pool_row * gpr + col / 64);
        }
        return;
    }
    if (pool_row == kNoRow) return;
    const uint32_t col = (u - a.heads - a.cache.kv_heads) * 256;
    const uint32_t left = kv_width - col;  // values from here on, a multiple of 64
    if ((uint32_t)lane * 4 < left) {
        const float4 f = *reinterpret_cast<const float4 *>(src + (size_t)(a.heads + a.cache.kv_heads) * D + col + 4 * lane);
        const float v[4] = {f.x, f.y, f.z, f.w};
        store_q8x4(v, lane, a.cache.v_codes + (size_t)pool_row * kv_width + col,
                   reinterpret_cast<uint16_t *>(a.cache.v_scales) + (size_t)pool_row * gpr + col / 64);
    }
}

// ---- copies of pages ----
//
// A page is, in every layer, key codes, value codes, key scales and value
// scales; all layers' 16-byte pieces of these (2-byte ones of scales whose
// page is no multiple of 16 bytes) stand in one line, and a workgroup takes an
// equal stretch of it: no workgroup has a small plane to itself. A thread
// holds its kPieces pieces through a whole chain of steps (paged_plan.h): what
// one step reads, an earlier or later step of the same thread writes, so
// chains need no barrier, and a source that goes to several pages is read
// once.
constexpr int kPieces = 4;

template <bool kNarrowScales>
__global__ __launch_bounds__(256) void paged_copy_kernel(const PagedCopyArgs a, const paged::CopySteps steps) {
    const uint32_t begin = steps.chain[blockIdx.y], end = steps.chain[blockIdx.y + 1];
    const uint32_t per_layer = 2 * (a.code_pieces + a.scale_pieces);
    const uint64_t start = (uint64_t)blockIdx.x * (256 * kPieces);
    const uint32_t first_layer = (uint32_t)(start / per_layer), offset = (uint32_t)(start - (uint64_t)first_layer * per_layer);
    uint8_t *at[kPieces];  // the piece in page 0
    bool in_codes[kPieces], there[kPieces];
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
        uint32_t i = offset + 256 * k + threadIdx.x;
        const uint32_t more = i / per_layer;
        uint32_t layer = first_layer + more;
        i -= more * per_layer;
        there[k] = layer < a.cache.layers;
        layer = min(layer, a.cache.layers - 1);  // (read, not written)
        const bool codes = i < 2 * a.code_pieces;
        if (!codes) i -= 2 * a.code_pieces;
        const uint32_t plane = codes ? a.code_pieces : a.scale_pieces;
        const bool values = i >= plane;
        if (values) i -= plane;
        const uint32_t bytes = kNarrowScales && !codes ? 2 : 16;
        uint8_t *base = codes ? (values ? a.cache.v_codes : a.cache.k_codes) : (values ? a.cache.v_scales : a.cache.k_scales);
        in_codes[k] = codes;
        at[k] = base + (uint64_t)layer * a.cache.pages * (codes ? a.code_page : a.scale_page) + (uint64_t)i * bytes;
    }
    typedef uint32_t Piece __attribute__((ext_vector_type(4)));
    const auto load = [&](Piece(&v)[kPieces], uint32_t src) {
        const uint64_t in_code = src * a.code_page, in_scale = src * a.scale_page;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const uint8_t *from = at[k] + (in_codes[k] ? in_code : in_scale);
            if (!kNarrowScales || in_codes[k]) v[k] = *reinterpret_cast<const Piece *>(from);
            else v[k].x = *reinterpret_cast<const uint16_t *>(from);
        }
    };
    const auto store = [&](const Piece(&v)[kPieces], uint32_t dst) {
        const uint64_t in_code = dst * a.code_page, in_scale = dst * a.scale_page;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            if (!there[k]) continue;
            uint8_t *to = at[k] + (in_codes[k] ? in_code : in_scale);
            if (!kNarrowScales || in_codes[k]) *reinterpret_cast<Piece *>(to) = v[k];
            else *reinterpret_cast<uint16_t *>(to) = (uint16_t)v[k].x;
        }
    };
    Piece v[kPieces] = {}, saved[kPieces] = {};
    uint32_t held = paged::kSaved;  // the page in v
    for (uint32_t i = begin; i < end; ++i) {
        const uint32_t src = steps.src[i], dst = steps.dst[i];
        if (dst == paged::kSaved) load(saved, src);
        else if (src == paged::kSaved) store(saved, dst);
        else {
            if (src != held) load(v, src);
            held = src;
            store(v, dst);
        }
    }
}

}  // namespace

hipError_t launch_paged_append(hipStream_t s, const PagedAppendArgs &args) {
    PagedAppendArgs a = args;
    const uint32_t D = a.cache.head_dim;
    a.units = a.heads + a.cache.kv_heads + (a.cache.kv_heads * D + 255) / 256;
    const uint64_t blocks = ((uint64_t)a.batch.rows * a.units + 3) / 4;
    if (blocks > 0xffffffu) return hipErrorInvalidValue;  // (x 256 threads: the grid's 32 bits)
    switch (D) {
    case 64: paged_append_kernel<64><<<(uint32_t)blocks, 256, 0, s>>>(a); break;
    case 128: paged_append_kernel<128><<<(uint32_t)blocks, 256, 0, s>>>(a); break;
    case 192: paged_append_kernel<192><<<(uint32_t)blocks, 256, 0, s>>>(a); break;
    case 256: paged_append_kernel<256><<<(uint32_t)blocks, 256, 0, s>>>(a); break;
    default: return hipErrorNotSupported;
    }
    return hipGetLastError();
}

hipError_t launch_paged_copy(hipStream_t s, const qwh_paged_cache &cache, const paged::CopySteps &steps) {
    PagedCopyArgs a{};
    a.cache = cache;
    const uint64_t width = (uint64_t)cache.kv_heads * cache.head_dim;
    a.code_page = cache.page_size * width;
    a.scale_page = cache.page_size * (width / 64) * 2;
    // 16-byte pieces of the scales where every page starts and ends on them.
    const bool narrow = a.scale_page % 16 != 0 || !paged::aligned(cache.k_scales, 16) || !paged::aligned(cache.v_scales, 16);
    a.code_pieces = (uint32_t)(a.code_page / 16);
    a.scale_pieces = (uint32_t)(a.scale_page / (narrow ? 2 : 16));
    const uint64_t pieces = 2 * ((uint64_t)a.code_pieces + a.scale_pieces) * cache.layers;
    const uint64_t blocks = (pieces + 256 * kPieces - 1) / (256 * kPieces);
    if (blocks > 0xffffffu) return hipErrorInvalidValue;
    const dim3 grid((uint32_t)blocks, steps.chains);
    if (narrow) paged_copy_kernel<true><<<grid, 256, 0, s>>>(a, steps);
    else paged_copy_kernel<false><<<grid, 256, 0, s>>>(a, steps);
    return hipGetLastError();
}

}  // namespace qwh
