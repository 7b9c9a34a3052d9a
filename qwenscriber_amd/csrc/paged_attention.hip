// Attention of new tokens over a paged q8 cache (kernels.zig:697-767
// decodeAttentionStepQ8 for every new token, over its sequence's pages).
//
// A sequence's n new tokens and the R query heads of a key/value head are
// n * R query rows that share the stored rows: scores and weighted values are
// matrix products on the f16 matrix cores, queries against positions. A
// stored code u - 128 is exact in f16; its group's scale multiplies the
// group's products (keys) or the weight (values). Queries and weights are f32
// and go in as two f16 terms, x = hi + lo to 2^-22 (one term, 2^-11, would
// cost the f32 activations their precision), so every product runs twice.
// Sums are f32; the softmax keeps a running maximum and sum per query row, in
// base 2.
//
// The positions of a sequence are split over workgroups, by as many units of
// kUnit positions as give the device about `target` workgroups for the whole
// batch whatever the lengths are: lengths are device values, so every
// workgroup works out the same split from them (paged_work). A split that is
// not alone leaves a record (maximum, sum, weighted values) per query row,
// and a second launch joins the records in order.
#include <cfloat>

#include "common.h"
#include "paged.h"

namespace qwh {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint32_t kUnit = 128;     // positions: one round of a workgroup
constexpr uint32_t kTileRows = 16;  // query rows of a workgroup

struct KernelArgs {
    PagedAttentionArgs p;
    uint32_t held;          // positions a page table holds
    uint32_t ratio;         // query heads per key/value head
    uint32_t target;        // workgroups wanted
    float scaling;          // log2(e) / sqrt(head_dim)
    float *values, *sums;   // records: [record][row][D] and [record][row][2]
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// New tokens of sequence b (0 past the batch) and positions they see.
__device__ __forceinline__ uint32_t new_tokens(const qwh_paged_batch &batch, uint32_t b) {
    if (b >= batch.batch) return 0;
    if (!batch.row_starts) return 1;
    const uint32_t begin = min(batch.row_starts[b], batch.rows), end = min(batch.row_starts[b + 1], batch.rows);
    return end > begin ? end - begin : 0;
}

__device__ __forceinline__ uint32_t seen_positions(const KernelArgs &a, uint32_t b, uint32_t n) {
    if (n == 0) return 0;
    const uint64_t end = (uint64_t)a.p.batch.first[b] + n;
    return end < a.held ? (uint32_t)end : a.held;
}

// The whole batch's split: units of a workgroup, from the sum over the
// sequences of row tiles times units. By a whole wavefront.
__device__ __forceinline__ uint32_t split_units(const KernelArgs &a, int lane) {
    uint64_t total = 0;
    for (uint32_t base = 0; base < a.p.batch.batch; base += 64) {
        const uint32_t b = base + lane, n = new_tokens(a.p.batch, b);
        const uint64_t tiles = ((uint64_t)n * a.ratio + kTileRows - 1) / kTileRows;
        total += tiles * ((seen_positions(a, b, n) + kUnit - 1) / kUnit);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) total += __shfl_xor((unsigned long long)total, m, 64);
    const uint64_t units = (total * a.p.cache.kv_heads + a.target - 1) / a.target;
    return units > 1 ? (uint32_t)units : 1;
}

// A workgroup's part: query rows [tile * kTileRows, ...) of sequence b over
// split `split` of `splits`; `record` counts the parts of the sequences with
// more than one split.
struct Work {
    uint32_t b, n, tile, split, splits, record;
};

// Part number `item` (tiles of a sequence fastest, then its splits), or false
// past the last. Every wavefront of the workgroup gets the same.
__device__ __forceinline__ bool paged_work(const KernelArgs &a, uint32_t item, uint32_t units, int lane, Work &w) {
    // (64 bits: starts that fall, against the interface, can name more rows
    // than there are, and must not wrap into a part that is none.)
    uint64_t before = 0;
    uint32_t records = 0;
    for (uint32_t base = 0; base < a.p.batch.batch; base += 64) {
        const uint32_t b = base + lane, n = new_tokens(a.p.batch, b);
        const uint32_t tiles = (uint32_t)(((uint64_t)n * a.ratio + kTileRows - 1) / kTileRows);
        const uint32_t splits = ((seen_positions(a, b, n) + kUnit - 1) / kUnit + units - 1) / units;
        const uint32_t items = tiles * splits, recorded = splits > 1 ? items : 0;
        uint64_t sum = items;
        uint32_t rec = recorded;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint64_t s2 = __shfl_up((unsigned long long)sum, d, 64);
            const uint32_t r2 = __shfl_up(rec, d, 64);
            if (lane >= d) {
                sum += s2;
                rec += r2;
            }
        }
        const uint64_t past = __ballot(before + sum > item);
        if (past) {
            const int at = __builtin_ctzll(past);
            const uint32_t rest = __shfl((uint32_t)(item - before - (sum - items)), at, 64);
            const uint32_t t = __shfl(tiles, at, 64);
            w.b = base + at;
            w.n = __shfl(n, at, 64);
            w.splits = __shfl(splits, at, 64);
            w.split = rest / t;
            w.tile = rest - w.split * t;
            w.record = records + __shfl(rec - recorded, at, 64) + rest;
            return true;
        }
        before += __shfl((unsigned long long)sum, 63, 64);
        records += __shfl(rec, 63, 64);
    }
    return false;
}

// Eight codes (two words) as f16 (u - 128) * 2^-9: a byte in a 16-bit half is
// u * 2^-24, a subnormal that the multiply-add takes as it is.
constexpr float kCodeScale = 512.0f;  // what brings such products back

__device__ __forceinline__ h2 code_pair(uint32_t halves) {
    const h2 x = __builtin_bit_cast(h2, halves);
    const h2 up = {(_Float16)32768.0f, (_Float16)32768.0f}, bias = {(_Float16)-0.25f, (_Float16)-0.25f};
    return __builtin_elementwise_fma(x, up, bias);
}

__device__ __forceinline__ h8 codes8(uint32_t low, uint32_t high) {
    const h2 a = code_pair(__builtin_amdgcn_perm(0u, low, 0x0c010c00u));
    const h2 b = code_pair(__builtin_amdgcn_perm(0u, low, 0x0c030c02u));
    const h2 c = code_pair(__builtin_amdgcn_perm(0u, high, 0x0c010c00u));
    const h2 d = code_pair(__builtin_amdgcn_perm(0u, high, 0x0c030c02u));
    return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Byte T of each of eight words, in order.
template <int T>
__device__ __forceinline__ h8 codes_across(const uint32_t (&w)[8]) {
    constexpr uint32_t sel = 0x0c000c00u | (uint32_t)T | (uint32_t)(T + 4) << 16;
    const h2 a = code_pair(__builtin_amdgcn_perm(w[1], w[0], sel));
    const h2 b = code_pair(__builtin_amdgcn_perm(w[3], w[2], sel));
    const h2 c = code_pair(__builtin_amdgcn_perm(w[5], w[4], sel));
    const h2 d = code_pair(__builtin_amdgcn_perm(w[7], w[6], sel));
    return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// x as hi + lo, both f16 (rounded to nearest, together 2^-22 of x).
__device__ __forceinline__ void two_terms(const float (&x)[8], h8 &hi, h8 &lo) {
#pragma unroll
    for (int i = 0; i < 8; ++i) hi[i] = (_Float16)x[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = (_Float16)(x[i] - (float)hi[i]);
}

__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The largest of a value over the four lanes that share lane % 16.
__device__ __forceinline__ float quarters_max(float v) {
    v = fmaxf(v, dev::xor_lane<16>(v));
    return fmaxf(v, dev::xor_lane<32>(v));
}

__device__ __forceinline__ float quarters_sum(float v) {
    v += dev::xor_lane<16>(v);
    return v + dev::xor_lane<32>(v);
}

// Sixteen query rows (columns of the products) over a range of positions.
// Each of the four wavefronts takes every fourth 32 positions by itself, two
// blocks of 16:
//   scores  [position][row] = K [16 x 32 values] Q^T, lane l: row l % 16,
//           positions 4 * (l / 16) .. + 3 of each block;
//   values  [dimension][row] += V^T [16 x 32 positions] P^T: the weights a
//           lane holds are the operand P^T of its own row, if the 32
//           positions are counted in the order (quarter, block, four), so
//           weights never leave their lane. V^T takes lane l % 16's four
//           dimensions of a group (one word a position), a product for each.
// Loads go straight to registers, the next tile's before this one's products.
template <int D>
__global__ __launch_bounds__(256, 2) void paged_few_kernel(const KernelArgs a) {
    constexpr int G = D / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = lane & 15, quarter = lane >> 4;
    const qwh_paged_cache &c = a.p.cache;
    const uint32_t kvh = blockIdx.x % c.kv_heads;
    Work work;
    const uint32_t units = split_units(a, lane);
    if (!paged_work(a, blockIdx.x / c.kv_heads, units, lane, work)) return;
    const uint32_t first = a.p.batch.first[work.b];
    const uint32_t start = a.p.batch.row_starts ? a.p.batch.row_starts[work.b] : work.b;
    // This lane's query row: token t, head kvh * ratio + r; it sees positions
    // up to `limit`.
    const uint32_t f = work.tile * kTileRows + n;
    const uint32_t t = f / a.ratio, r = f - t * a.ratio;
    const bool active = t < work.n;
    const uint32_t last_t = min((work.tile * kTileRows + kTileRows - 1) / a.ratio, work.n - 1);
    const uint32_t first_t = work.tile * kTileRows / a.ratio;
    const auto place = [&](uint32_t token) {  // its position, at most the tables' last
        const uint64_t p = (uint64_t)first + token;
        return p < a.held ? (uint32_t)p : a.held - 1;
    };
    const uint32_t limit = place(t), common = place(first_t);
    const uint32_t begin = work.split * units * kUnit;
    uint32_t end = place(last_t) + 1;
    if (begin >= end) return;  // (no row of the tile sees this split)
    if (end - begin > units * kUnit) end = begin + units * kUnit;

    __shared__ uint32_t lds_rows[4][32];
    __shared__ float lds_scale[4][2][G][32];
    __shared__ float lds_acc[2][kTileRows][D + 4];
    __shared__ float lds_state[2][2][kTileRows];

    // The query row in two terms, scaled by a power of two to below 2^8.
    const size_t row = (size_t)start + t;
    h8 qh[G][2], ql[G][2];
    float qs;
    {
        float q[G][16];
        float top = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const f4 *src = reinterpret_cast<const f4 *>(a.p.query + (active ? row * a.p.query_stride + (kvh * a.ratio + r) * D + 64 * g + 16 * quarter : 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f4 v = src[i];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    q[g][4 * i + k] = active ? v[k] : 0.0f;
                    top = fmaxf(top, fabsf(q[g][4 * i + k]));
                }
            }
        }
        top = quarters_max(top);
        int e = 0;
        if (top > 0.0f && top < INFINITY) (void)__builtin_frexpf(top, &e);
        e = e < -100 ? -100 : e;
        const float up = __builtin_ldexpf(1.0f, 8 - e);
        qs = a.scaling * __builtin_ldexpf(kCodeScale, e - 8);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = q[g][8 * k + i] * up;
                two_terms(x, qh[g][k], ql[g][k]);
            }
    }

    const uint32_t kv_width = c.kv_heads * D, gpr = kv_width / 64;
    const uint32_t *table = a.p.batch.tables + (size_t)work.b * a.p.batch.table_pages;
    const uint8_t *k_base = c.k_codes + kvh * D + 16 * quarter;
    const uint8_t *v_base = c.v_codes + kvh * D + 4 * n;
    // Lanes 0..31 load the key scales of position lane, 32..63 the value scales.
    const uint16_t *scale_base = reinterpret_cast<const uint16_t *>(lane < 32 ? c.k_scales : c.v_scales) + kvh * G;

    struct Tile {
        uint4 k[2][G];
        uint32_t v[G][8];
        uint16_t scale[G];
        uint32_t there;  // of the 32 positions, those with a row
    };
    // The pool row of this lane's position (lane % 32) of the tile at `base`.
    const auto lookup = [&](uint32_t base) {
        const uint32_t p = base + (lane & 31);
        return p < end ? paged_pool_row(c, table, p) : kNoRow;
    };
    const auto load = [&](Tile &tile, uint32_t pool_row) {
        tile.there = (uint32_t)__ballot(pool_row != kNoRow);
        const uint32_t safe = pool_row != kNoRow ? pool_row : 0;
        if (lane < 32) lds_rows[wave][lane] = safe;
        wave_fence();
        const uint32_t k0 = lds_rows[wave][n], k1 = lds_rows[wave][16 + n];
        const u4 v0 = *reinterpret_cast<const u4 *>(&lds_rows[wave][4 * quarter]);
        const u4 v1 = *reinterpret_cast<const u4 *>(&lds_rows[wave][16 + 4 * quarter]);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            tile.k[0][g] = *reinterpret_cast<const uint4 *>(k_base + (size_t)k0 * kv_width + 64 * g);
            tile.k[1][g] = *reinterpret_cast<const uint4 *>(k_base + (size_t)k1 * kv_width + 64 * g);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) tile.scale[g] = scale_base[(size_t)safe * gpr + g];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int g = 0; g < G; ++g) {
                tile.v[g][i] = *reinterpret_cast<const uint32_t *>(v_base + (size_t)v0[i] * kv_width + 64 * g);
                tile.v[g][4 + i] = *reinterpret_cast<const uint32_t *>(v_base + (size_t)v1[i] * kv_width + 64 * g);
            }
        wave_fence();
    };

    float m = -INFINITY, l = 0.0f;
    float e_w = -100.0f;  // acc is in units of 2^e_w
    f4 acc[G][4];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};

    const auto use = [&](const Tile &tile, uint32_t base) {
#pragma unroll
        for (int g = 0; g < G; ++g) lds_scale[wave][lane >> 5][g][lane & 31] = dev::f16_bits_to_f32(tile.scale[g]);
        wave_fence();
        f4 s[2];
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            s[blk] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint4 w = tile.k[blk][g];
                const h8 ka = codes8(w.x, w.y), kb = codes8(w.z, w.w);
                f4 x = mma(ka, ql[g][0], f4{0.0f, 0.0f, 0.0f, 0.0f});
                x = mma(kb, ql[g][1], x);
                x = mma(ka, qh[g][0], x);
                x = mma(kb, qh[g][1], x);
                const f4 ks = *reinterpret_cast<const f4 *>(&lds_scale[wave][0][g][16 * blk + 4 * quarter]);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[blk][i] = fmaf(ks[i], x[i], s[blk][i]);
            }
        }
        const bool whole = tile.there == 0xffffffffu && base + 31 <= common;
        if (!whole) {
#pragma unroll
            for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t at = 16 * blk + 4 * quarter + i;
                    if (!(tile.there >> at & 1u) || base + at > limit) s[blk][i] = -INFINITY;
                }
        }
        float mx = m;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[blk][i]);
        mx = quarters_max(mx);
        // A row that has seen nothing yet: weights of 0 against any maximum.
        const float low = (mx == -INFINITY ? 0.0f : mx) * qs;
        const float turn = fmaf(m, qs, -low);  // log2 of what earlier weights lose
        m = mx;
        float p[8];
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[4 * blk + i] = exp2_fast(fmaf(s[blk][i], qs, -low));
        // The weights with their value scales, and the power of two that
        // brings the row's largest (of earlier ones too) near f16's top.
        float w[G][8], largest = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const f4 s0 = *reinterpret_cast<const f4 *>(&lds_scale[wave][1][g][4 * quarter]);
            const f4 s1 = *reinterpret_cast<const f4 *>(&lds_scale[wave][1][g][16 + 4 * quarter]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[g][i] = p[i] * s0[i];
                w[g][4 + i] = p[4 + i] * s1[i];
            }
            if (!whole) {  // (a scale that is no number must not reach rows that do not see it)
#pragma unroll
                for (int i = 0; i < 8; ++i) w[g][i] = s[i / 4][i & 3] == -INFINITY ? 0.0f : w[g][i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) largest = fmaxf(largest, w[g][i]);
        }
        largest = quarters_max(largest);
        const float e_now = fmaxf(fmaxf(e_w + ceilf(turn), (float)((int)(__float_as_uint(largest) >> 23) - 126)), -100.0f);
        if (__ballot(turn != 0.0f || e_now != e_w)) {
            l *= exp2_fast(turn);
            const float both = exp2_fast(turn + (e_w - e_now));
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[g][i] *= both;
            e_w = e_now;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) l += p[i];
        const float up = exp2_fast(12.0f - e_w);
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[g][i] *= up;
            h8 ph, pl;
            two_terms(w[g], ph, pl);
            const h8 v0 = codes_across<0>(tile.v[g]), v1 = codes_across<1>(tile.v[g]);
            const h8 v2 = codes_across<2>(tile.v[g]), v3 = codes_across<3>(tile.v[g]);
            acc[g][0] = mma(v0, ph, mma(v0, pl, acc[g][0]));
            acc[g][1] = mma(v1, ph, mma(v1, pl, acc[g][1]));
            acc[g][2] = mma(v2, ph, mma(v2, pl, acc[g][2]));
            acc[g][3] = mma(v3, ph, mma(v3, pl, acc[g][3]));
        }
        wave_fence();
    };

    uint32_t base = begin + 32 * wave;
    if (base < end) {
        Tile even, odd;
        load(even, lookup(base));
        uint32_t ahead = lookup(base + kUnit < end ? base + kUnit : base);
        for (;;) {
            const uint32_t second = base + kUnit;
            if (second < end) {
                load(odd, ahead);
                ahead = lookup(second + kUnit < end ? second + kUnit : second);
            }
            use(even, base);
            if (second >= end) break;
            base = second + kUnit;
            if (base < end) {
                load(even, ahead);
                ahead = lookup(base + kUnit < end ? base + kUnit : base);
            }
            use(odd, second);
            if (base >= end) break;
        }
    }

    // The four wavefronts' states into the first's: 2 and 3 hand theirs to 0
    // and 1, then 1 to 0. Maxima in base 2, values without their powers of two.
    l = quarters_sum(l);
    float M = m == -INFINITY ? -INFINITY : m * qs;
    const float back = exp2_fast(e_w - 12.0f) * kCodeScale;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][i] *= back;
#pragma unroll
    for (int half = 2; half >= 1; half /= 2) {
        if (wave >= half && wave < 2 * half) {
            const int slot = wave - half;
            if (quarter == 0) {
                lds_state[slot][0][n] = M;
                lds_state[slot][1][n] = l;
            }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f4 *>(&lds_acc[slot][n][64 * g + 16 * quarter + 4 * i]) =
                        f4{acc[g][0][i], acc[g][1][i], acc[g][2][i], acc[g][3][i]};
        }
        __syncthreads();
        if (wave < half) {
            const float m2 = lds_state[wave][0][n], l2 = lds_state[wave][1][n];
            const float top = fmaxf(M, m2), low = top == -INFINITY ? 0.0f : top;
            const float f1 = exp2_fast(M - low), f2 = exp2_fast(m2 - low);
            M = top;
            l = l * f1 + l2 * f2;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f4 other = *reinterpret_cast<const f4 *>(&lds_acc[wave][n][64 * g + 16 * quarter + 4 * i]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[g][k][i] = acc[g][k][i] * f1 + other[k] * f2;
                }
        }
        __syncthreads();
    }
    if (wave != 0 || !active) return;
    if (work.splits > 1) {
        const size_t rec = ((size_t)work.record * c.kv_heads + kvh) * kTileRows + n;
        if (quarter == 0) {
            a.sums[2 * rec] = M;
            a.sums[2 * rec + 1] = l;
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f4 *>(a.values + rec * D + 64 * g + 16 * quarter + 4 * i) =
                    f4{acc[g][0][i], acc[g][1][i], acc[g][2][i], acc[g][3][i]};
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float *out = a.p.out + (row * a.p.heads + kvh * a.ratio + r) * D + 16 * quarter;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f4 *>(out + 64 * g + 4 * i) =
                f4{acc[g][0][i] * inv, acc[g][1][i] * inv, acc[g][2][i] * inv, acc[g][3][i] * inv};
}

// Joins the records of a query row (one wavefront) in the order of its
// splits. Rows of sequences with one split were written by their workgroup.
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const KernelArgs a, uint32_t rows) {
    constexpr int G = D / 64;
    const int lane = threadIdx.x & 63;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t row = (uint32_t)(unit / a.p.heads), h = (uint32_t)(unit % a.p.heads);
    if (row >= rows) return;
    uint32_t b, t;
    if (!paged_row(a.p.batch, row, lane, b, t)) return;
    const uint32_t units = split_units(a, lane);
    // The sequence's first record.
    uint32_t records = 0, splits = 0, tiles = 0;
    for (uint32_t base = 0; base <= b; base += 64) {
        const uint32_t s = base + lane, n = new_tokens(a.p.batch, s);
        const uint32_t s_tiles = (uint32_t)(((uint64_t)n * a.ratio + kTileRows - 1) / kTileRows);
        const uint32_t s_splits = ((seen_positions(a, s, n) + kUnit - 1) / kUnit + units - 1) / units;
        uint32_t mine = s < b && s_splits > 1 ? s_tiles * s_splits : 0;
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) mine += __shfl_xor(mine, m, 64);
        records += mine;
        if (b - base < 64) {
            splits = (uint32_t)__builtin_amdgcn_readlane((int)s_splits, (int)(b - base));
            tiles = (uint32_t)__builtin_amdgcn_readlane((int)s_tiles, (int)(b - base));
        }
    }
    if (splits <= 1) return;
    const uint32_t kvh = h / a.ratio, f = t * a.ratio + (h - kvh * a.ratio);
    const uint32_t tile = f / kTileRows, n = f - tile * kTileRows;
    const uint64_t seen = (uint64_t)a.p.batch.first[b] + t + 1;
    const uint32_t span = units * kUnit;
    const uint32_t used = ((seen < a.held ? (uint32_t)seen : a.held) + span - 1) / span;
    float M = -INFINITY, L = 0.0f, acc[G];
#pragma unroll
    for (int g = 0; g < G; ++g) acc[g] = 0.0f;
    for (uint32_t s0 = 0; s0 < used; s0 += 4) {
        float m[4], l[4], v[4][G];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t s = min(s0 + k, used - 1);
            const size_t rec = ((size_t)(records + s * tiles + tile) * a.p.cache.kv_heads + kvh) * kTileRows + n;
            m[k] = a.sums[2 * rec];
            l[k] = a.sums[2 * rec + 1];
#pragma unroll
            for (int g = 0; g < G; ++g) v[k][g] = a.values[rec * D + 64 * g + lane];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (s0 + k >= used) break;
            const float top = fmaxf(M, m[k]), low = top == -INFINITY ? 0.0f : top;
            const float f1 = exp2_fast(M - low), f2 = exp2_fast(m[k] - low);
            M = top;
            L = L * f1 + l[k] * f2;
#pragma unroll
            for (int g = 0; g < G; ++g) acc[g] = acc[g] * f1 + v[k][g] * f2;
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int g = 0; g < G; ++g) a.p.out[((size_t)row * a.p.heads + h) * D + 64 * g + lane] = acc[g] * inv;
}

// Workgroups wanted: three on a CU at once.
uint32_t target_groups(int cus) { return 3u * (uint32_t)(cus > 0 ? cus : 256); }

// Records: parts of sequences of two splits and more. Each has at most twice
// its units' share of the target.
uint64_t max_records(int cus, const PagedAttentionArgs &a) {
    return (2ull * target_groups(cus) + a.cache.kv_heads - 1) / a.cache.kv_heads * a.cache.kv_heads;
}

template <int D>
hipError_t launch_attention(hipStream_t s, int cus, const KernelArgs &k) {
    const qwh_paged_batch &b = k.p.batch;
    // Row tiles at most: whole ones of all rows, and one more a sequence.
    const uint64_t tiles = b.row_starts ? (uint64_t)b.rows * k.ratio / kTileRows + (b.batch < b.rows ? b.batch : b.rows)
                                        : (uint64_t)b.batch * ((k.ratio + kTileRows - 1) / kTileRows);
    const uint64_t blocks = (k.target / k.p.cache.kv_heads + tiles) * k.p.cache.kv_heads;
    const uint32_t rows = b.row_starts ? b.rows : b.batch;
    const uint64_t join = ((uint64_t)rows * k.p.heads + 3) / 4;
    if (blocks > 0xffffffu || join > 0xffffffu) return hipErrorInvalidValue;
    paged_few_kernel<D><<<(uint32_t)blocks, 256, 0, s>>>(k);
    // (One unit in all: nothing to join.)
    if (k.held > kUnit) paged_join_kernel<D><<<(uint32_t)join, 256, 0, s>>>(k, rows);
    return hipGetLastError();
}

}  // namespace

size_t paged_attention_scratch_bytes(int cus, const PagedAttentionArgs &a) {
    return max_records(cus, a) * kTileRows * (a.cache.head_dim + 2) * sizeof(float) + 256;
}

hipError_t launch_paged_attention(hipStream_t s, int cus, const PagedAttentionArgs &a, void *scratch, size_t scratch_bytes) {
    if (paged_attention_scratch_bytes(cus, a) > scratch_bytes) return hipErrorInvalidValue;
    KernelArgs k{};
    k.p = a;
    const uint64_t held = (uint64_t)a.batch.table_pages * a.cache.page_size;
    k.held = held < 0xfffffff0ull ? (uint32_t)held : 0xfffffff0u;
    k.ratio = a.heads / a.cache.kv_heads;
    k.target = target_groups(cus);
    k.scaling = kLog2e / sqrtf((float)a.cache.head_dim);
    k.values = static_cast<float *>(scratch);
    k.sums = k.values + max_records(cus, a) * kTileRows * a.cache.head_dim;
    switch (a.cache.head_dim) {
    case 64: return launch_attention<64>(s, cus, k);
    case 128: return launch_attention<128>(s, cus, k);
    case 192: return launch_attention<192>(s, cus, k);
    case 256: return launch_attention<256>(s, cus, k);
    default: return hipErrorNotSupported;
    }
}

}  // namespace qwh
