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
// A wavefront takes 8, 4, 2 or 2 (head_dim 64, 128, 192, 256) neighbouring
// query or key heads of a row, a group of lanes each, or 512 values of the
// value row: no wavefront waits for another, and a step's few rows still
// spread over the device. The values are asked for first; the way to the page
// (the row's sequence, its position, its table) is a chain of loads of its own
// meanwhile. A lane has four dimensions and the four that the rotation mixes
// with them (D/2 further), so norm and rotation need one reduction over the
// group, no exchange, and mostly neither do the 64 values of a scale. Norm and
// rotation are in f64 (the square of an f32 is exact there): a key's code is a
// rounding of its value, and 32-bit sums put about one code in 10^5 on the
// other side of a border, by the order of the sum. Bound by instructions and
// the stream of bytes about alike: 1608 tokens of 16 + 8 heads of 128 take 12.8
// us (3.3 TB/s; a whole wavefront a head, 21), a step of up to 256 tokens the
// 5 us of a launch.
template <int MASK>
__device__ __forceinline__ double xor_lane64(double v) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_bit_cast(uint32_t, dev::xor_lane<MASK>(__builtin_bit_cast(float, (uint32_t)x)));
    const uint32_t hi = __builtin_bit_cast(uint32_t, dev::xor_lane<MASK>(__builtin_bit_cast(float, (uint32_t)(x >> 32))));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// 1 / sqrt(x): the hardware's, about 2^-26 off, and two of Newton's steps.
__device__ __forceinline__ double inverse_root(double x) {
    const double r0 = __builtin_amdgcn_rsq(x);
    double r = r0;
    r = fma(r * 0.5, fma(-x * r, r, 1.0), r);
    r = fma(r * 0.5, fma(-x * r, r, 1.0), r);
    return r0 == 0.0 ? 0.0 : r;  // (of infinity)
}

typedef float Quad __attribute__((ext_vector_type(4), aligned(4)));

// Lanes of a head, and heads and value quads of a wavefront.
constexpr int head_lanes(int D) { return D == 64 ? 8 : D == 128 ? 16 : 32; }
constexpr uint32_t kValues = 512;

template <int D>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendArgs a) {
    constexpr int H = D / 2, kLanes = head_lanes(D), kHeads = 64 / kLanes;
    __shared__ float lds_k[D == 192 ? 4 : 1][D == 192 ? kHeads * D : 1];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const uint32_t unit = blockIdx.x * 4 + wave;
    const uint32_t row = unit / a.units, u = unit % a.units;
    if (row >= a.batch.rows) return;
    const uint32_t kv_width = a.cache.kv_heads * D, normed = a.heads + a.cache.kv_heads;
    const uint32_t head_units = (normed + kHeads - 1) / kHeads;
    const float *src = a.qkv + (size_t)row * a.qkv_stride;
    const bool is_value = u >= head_units;
    const uint32_t first_head = u * kHeads, head = first_head + lane / kLanes, value = (u - head_units) * kValues + 4 * lane;
    const int at = 4 * (lane % kLanes);  // of the head's dimensions
    const bool there = head < normed && at < H;
    float lo[4] = {}, hi[4] = {};
    const auto take = [](float(&to)[4], const float *from) {
        const Quad v = *reinterpret_cast<const Quad *>(from);
        to[0] = v.x;
        to[1] = v.y;
        to[2] = v.z;
        to[3] = v.w;
    };
    if (is_value) {
        if (value < kv_width) take(lo, src + (size_t)normed * D + value);
        if (value + 256 < kv_width) take(hi, src + (size_t)normed * D + value + 256);
    } else if (there) {
        take(lo, src + (size_t)head * D + at);
        take(hi, src + (size_t)head * D + at + H);
    }
    uint32_t b, t;
    if (!paged_row(a.batch, row, lane, b, t)) return;
    const uint64_t position = (uint64_t)a.batch.first[b] + t;
    if (position >= a.positions) return;
    const uint32_t pos = (uint32_t)position;
    const uint32_t pool_row = paged_pool_row(a.cache, a.batch.tables + (size_t)b * a.batch.table_pages, pos);
    const uint32_t gpr = kv_width / 64;
    if (is_value) {
        if (pool_row == kNoRow) return;
        uint8_t *codes = a.cache.v_codes + (size_t)pool_row * kv_width + value;
        uint16_t *scales = reinterpret_cast<uint16_t *>(a.cache.v_scales) + (size_t)pool_row * gpr + value / 64;
        if (value < kv_width) store_q8x4<16>(lo, codes, lane % 16 == 0 ? scales : nullptr);  // (a multiple of 64)
        if (value + 256 < kv_width) store_q8x4<16>(hi, codes + 256, lane % 16 == 0 ? scales + 4 : nullptr);
        return;
    }
    // (first_head + kHeads - 1 may be a key where first_head is a query.)
    if (pool_row == kNoRow && first_head >= a.heads) return;
    const bool is_query = head < a.heads;
    const float *w = (is_query ? a.q_norm : a.k_norm) + at;
    float wl[4] = {}, wh[4] = {}, c[4] = {}, s[4] = {};
    if (there) {
        take(wl, w);
        take(wh, w + H);
        take(c, a.rope_cos + (size_t)pos * H + at);
        take(s, a.rope_sin + (size_t)pos * H + at);
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) ss += (double)lo[i] * lo[i] + (double)hi[i] * hi[i];
    if constexpr (kLanes >= 32) ss += xor_lane64<16>(ss);
    if constexpr (kLanes >= 16) ss += xor_lane64<8>(ss);
    ss += xor_lane64<4>(ss);
    ss += xor_lane64<2>(ss);
    ss += xor_lane64<1>(ss);
    const double inv = inverse_root(ss * (1.0 / D) + (double)a.eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const double yl = (double)lo[i] * inv * wl[i], yh = (double)hi[i] * inv * wh[i];
        lo[i] = (float)(yl * c[i] - yh * s[i]);
        hi[i] = (float)(yh * c[i] + yl * s[i]);
    }
    if (there && is_query) {
        float *out = a.query + (size_t)row * a.query_stride + (size_t)head * D + at;
        *reinterpret_cast<float4 *>(out) = float4{lo[0], lo[1], lo[2], lo[3]};
        *reinterpret_cast<float4 *>(out + H) = float4{hi[0], hi[1], hi[2], hi[3]};
    }
    if (pool_row == kNoRow || first_head + kHeads <= a.heads) return;
    const bool is_key = there && !is_query;
    uint8_t *codes = a.cache.k_codes + (size_t)pool_row * kv_width;
    uint16_t *scales = reinterpret_cast<uint16_t *>(a.cache.k_scales) + (size_t)pool_row * gpr;
    if constexpr (D == 192) {
        // Scales' groups of 64 and halves of 96 do not fit: over LDS, 48
        // lanes a head.
        if (there) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lds_k[wave][lane / kLanes * D + at + i] = lo[i];
                lds_k[wave][lane / kLanes * D + at + H + i] = hi[i];
            }
        }
        wave_fence();
#pragma unroll
        for (int k = 0; k < kHeads; ++k) {
            const uint32_t h = first_head + k;
            if (h < a.heads || h >= normed || lane >= D / 4) continue;
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = lds_k[wave][k * D + 4 * lane + i];
            const uint32_t col = (h - a.heads) * D + 4 * lane;
            store_q8x4<16>(v, codes + col, lane % 16 == 0 ? scales + col / 64 : nullptr);
        }
    } else if (is_key) {
        const uint32_t col = (head - a.heads) * D + at;
        if constexpr (D == 64) {
            const float m = group_max<8>(fmaxf(quad_max(lo), quad_max(hi)));
            store_q8x4_of(m, lo, codes + col, at == 0 ? scales + col / 64 : nullptr);
            store_q8x4_of(m, hi, codes + col + H, nullptr);
        } else {
            store_q8x4<16>(lo, codes + col, lane % 16 == 0 ? scales + col / 64 : nullptr);
            store_q8x4<16>(hi, codes + col + H, lane % 16 == 0 ? scales + (col + H) / 64 : nullptr);
        }
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
// once. Bound by HBM where chains are short: 300 pages of 16 positions in 28
// layers, 284 MB read and as much written, 117 us (4.9 TB/s; 8 pieces a thread,
// 157). A long chain is bound by its round trips, a load and the store of it
// a step: the same 300 pages each to the page before it, 394 us.
constexpr int kPieces = 4;

template <bool kNarrowScales, typename Steps>
__global__ __launch_bounds__(256) void paged_copy_kernel(const PagedCopyArgs a, const Steps steps) {
    static_assert(sizeof(a) + sizeof(steps) <= 4096, "a kernel's arguments");
    const uint32_t begin = steps.begin(blockIdx.y), end = steps.end(blockIdx.y);
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
        const uint32_t src = steps.source(i), dst = steps.target(i);
        if (dst == paged::kSaved) load(saved, src);
        else if (src == paged::kSaved) {
            store(saved, dst);
            held = paged::kSaved;  // (dst may be the page in v)
        } else {
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
    const uint32_t heads = 64 / head_lanes((int)D);
    a.units = (a.heads + a.cache.kv_heads + heads - 1) / heads + (a.cache.kv_heads * D + kValues - 1) / kValues;
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

hipError_t launch_paged_copy(hipStream_t s, const qwh_paged_cache &cache, const paged::CopyLaunch &launch, bool is_short) {
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
    const dim3 grid((uint32_t)blocks, launch.chains());
    const auto run = [&](const auto &steps) {
        if (narrow) paged_copy_kernel<true><<<grid, 256, 0, s>>>(a, steps);
        else paged_copy_kernel<false><<<grid, 256, 0, s>>>(a, steps);
    };
    if (is_short) run(paged::pack_short(launch));
    else run(paged::pack(launch));
    return hipGetLastError();
}

}  // namespace qwh
