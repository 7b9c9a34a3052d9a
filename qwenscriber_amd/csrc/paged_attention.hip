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
// The work is one line of units (kTileRows query rows by kUnit positions), a
// sequence's row tiles one after another, and each workgroup takes an equal
// stretch of it, whatever the lengths are. Lengths are device values, so every
// workgroup works out the line from them (WorkLine). A stretch that begins or
// ends inside a tile's positions leaves a record (maximum, sum, weighted
// values) per query row, and a second launch joins the records in order.
#include <cmath>

#include "common.h"
#include "paged.h"

namespace qwh {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint32_t kUnit = 128;     // positions: one round of a workgroup
constexpr uint32_t kTileRows = 8;   // query rows of a workgroup
constexpr uint32_t kDies = 8;

struct KernelArgs {
    PagedAttentionArgs p;
    uint32_t held;          // positions a page table holds
    uint32_t ratio;         // query heads per key/value head
    uint32_t ratio_magic;   // floor(2^32 / ratio) + 1 (0: ratio 1)
    uint32_t page_shift;    // log2 of page_size (32: not a power of two)
    uint32_t stretches_most;  // stretches that the records are for
    float inverse_stretches;
    float scaling;          // log2(e) / sqrt(head_dim)
    float *values, *sums;   // records: [record][row][D] and [record][row][2]
    uint32_t few_rows;      // query rows a kv head up to which a sequence takes paged_few_kernel (paged::few_rows)
    uint32_t stretches_most_many;
    float inverse_stretches_many;
    float *values_many, *sums_many;
    u4 *plan;               // per sequence: units of a stretch, its first unit, units of a tile (many: whole_units), 1: many
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// New tokens of sequence b (0 past the batch) and positions they see.
__device__ __forceinline__ uint32_t new_tokens(const qwh_paged_batch &batch, uint32_t b) {
    if (b >= batch.batch) return 0;
    if (!batch.row_starts) return 1;
    const uint32_t begin = min(batch.row_starts[b], batch.rows), end = min(batch.row_starts[b + 1], batch.rows);
    return end > begin ? end - begin : 0;
}

__device__ __forceinline__ uint32_t row_tiles(const KernelArgs &a, uint32_t n, uint32_t rows = kTileRows) {
    return (n * a.ratio + rows - 1) / rows;
}

__device__ __forceinline__ uint32_t whole_units(const KernelArgs &a, uint32_t first);
__device__ __forceinline__ uint32_t tiles_units(const KernelArgs &a, uint32_t whole, uint32_t j);

// f / ratio for f up to 2^23 + kTileRows (ratio at most 256).
__device__ __forceinline__ uint32_t by_ratio(const KernelArgs &a, uint32_t f) {
    return a.ratio_magic ? __umulhi(f, a.ratio_magic) : f;
}

// The line's length is below this for starts that never fall (the host holds
// rows and positions to it); sums stop here, so that others cannot wrap.
constexpr uint32_t kMostUnits = 0x7fffffffu;

__device__ __forceinline__ uint32_t add_units(uint32_t a, uint32_t b) { return min(a + b, kMostUnits); }

// Inclusive sums over the wavefront, in lane order.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = add_units(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true));   // row_shr:1
    v = add_units(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true));   // row_shr:2
    v = add_units(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true));   // row_shr:4
    v = add_units(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true));   // row_shr:8
    v = add_units(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));  // row_bcast:15
    v = add_units(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false));  // row_bcast:31
    return v;
}

__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }

// The line of units, 64 sequences of it at a time (a lane each). By a whole
// wavefront; what is found is uniform.
struct WorkLine {
    uint32_t base = 0;            // the first of the 64 sequences
    uint32_t before = 0;          // units before them
    uint32_t n, first, units, upto;  // this lane's sequence: new tokens, its first position, units of a row tile, units up to its end

    // `rows`: of a tile, which also says whose sequences these are.
    __device__ void load(const KernelArgs &a, int lane, uint32_t rows) {
        const qwh_paged_batch &batch = a.p.batch;
        const uint32_t b = base + lane;
        n = new_tokens(batch, b);
        if (paged::takes_many(n * a.ratio, a.few_rows) != (rows != kTileRows)) n = 0;
        first = b < batch.batch ? batch.first[b] : 0;
        const uint32_t tiles = row_tiles(a, n, rows);
        if (rows == kTileRows) {
            const uint64_t end = (uint64_t)first + n;
            const uint32_t seen = n == 0 ? 0 : end < a.held ? (uint32_t)end : a.held;
            units = (seen + kUnit - 1) / kUnit;
            upto = wave_scan(tiles * units);
        } else {
            upto = wave_scan(tiles_units(a, whole_units(a, first), tiles));
        }
    }
    // Units of the whole line (leaves its first 64 sequences loaded).
    __device__ uint32_t length(const KernelArgs &a, int lane, uint32_t rows = kTileRows) {
        load(a, lane, rows);
        uint32_t all = lane_of(upto, 63);
        if (a.p.batch.batch > 64) {
            for (base = 64; base < a.p.batch.batch; base += 64) {
                load(a, lane, rows);
                all = add_units(all, lane_of(upto, 63));
            }
            base = 0;
            load(a, lane, rows);
        }
        return all;
    }
    // The lane of the sequence that unit `at` lies in, moving on to its 64
    // (never back); false past the line.
    __device__ bool find(const KernelArgs &a, uint32_t at, int lane, int &owner, uint32_t rows = kTileRows) {
        for (;;) {
            const uint64_t past = __ballot(add_units(before, upto) > at);
            if (past) {
                owner = __builtin_ctzll(past);
                return true;
            }
            before = add_units(before, lane_of(upto, 63));
            base += 64;
            if (base >= a.p.batch.batch) return false;
            load(a, lane, rows);
        }
    }
};

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

// x as an f32 that is rounded here. A product that is converted to f16 may be
// folded into the conversion and rounded once, or twice elsewhere: hi and what
// it leaves would be of two numbers, half a step of hi apart.
__device__ __forceinline__ float settled(float x) {
    asm("" : "+v"(x));
    return x;
}

// What a half leaves of x, as a half: one mixed multiply-add each.
__device__ __forceinline__ _Float16 rest(float x, _Float16 hi) { return (_Float16)__builtin_fmaf((float)hi, -1.0f, x); }

// x as hi + lo, both f16 (rounded to nearest, together 2^-22 of x).
__device__ __forceinline__ void two_terms(const float (&x)[4], u2 &hi, u2 &lo) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = settled(x[i]);
    h4 h, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = (_Float16)y[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) l[i] = rest(y[i], h[i]);
    hi = __builtin_bit_cast(u2, h);
    lo = __builtin_bit_cast(u2, l);
}

__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Over the eight lanes of a query row: those that share lane % 8.
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, dev::xor_lane<8>(v));
    v = fmaxf(v, dev::xor_lane<16>(v));
    return fmaxf(v, dev::xor_lane<32>(v));
}

__device__ __forceinline__ float row_sum(float v) {
    v += dev::xor_lane<8>(v);
    v += dev::xor_lane<16>(v);
    return v + dev::xor_lane<32>(v);
}

// `keep` in lanes whose bit 3 is HIGH's opposite, in the others `from` of
// lane ^ 8 (a row rotation by 8 into half of the lanes).
template <bool HIGH>
__device__ __forceinline__ uint32_t take_other(uint32_t keep, uint32_t from) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)keep, (int)from, 0x128, 0xF, HIGH ? 0xC : 0x3, false);
}

// Eight query rows over a range of positions. A product's sixteen columns are
// the rows' first and second terms (lane l: column l % 16, row l % 8, term
// l / 8 % 2), so one product takes both. Each of the four wavefronts takes
// every fourth 32 positions by itself, two blocks of 16:
//   scores  [position][column] = K [16 x 32 values] Q^T, lane l: positions
//           4 * (l / 16) .. + 3 of each block. The two terms' columns are
//           added; the first term's lane goes on with block 0, the second's
//           with block 1;
//   values  [dimension][column] += V^T [16 x 32 positions] P^T, in whose 32
//           positions the order is (l / 16, block, four): a lane's weights
//           are half of its own column's operand and half of the other
//           term's, and change lanes only with that one. V^T takes lane
//           l % 16's four dimensions of a group (one word a position), a
//           product for each. The terms' sums are added at the end.
// Two tiles of registers: one in flight while the other is used.
//
// Bound by HBM with a start and an end: 16 sequences at 4096 positions (138
// MB, 28 us at the rate of a large copy) take 33 us here, 6 of them the chain
// from the batch's arrays over a table to the first tile, and 4.7 in the join;
// 61 of 1 to 5003 (325 MB, 66 us) 82 and 4.9. Loads alone take 36 in all, the
// products alone 27.
template <int D>
__global__ __launch_bounds__(256, 2) void paged_few_kernel(const KernelArgs a) {
    constexpr int G = D / 64;
    constexpr uint32_t kPieces = D / 16;  // 16-byte pieces of a head row
    const int lane = threadIdx.x & 63, wave = (int)uniform(threadIdx.x >> 6);
    const int n = lane & 15, quarter = lane >> 4, term = lane >> 3 & 1;
    const qwh_paged_cache &c = a.p.cache;
    // A stretch's heads one after another on a die.
    const uint32_t kvh = blockIdx.x / kDies % c.kv_heads;
    const uint32_t stretch = blockIdx.x / kDies / c.kv_heads * kDies + blockIdx.x % kDies;
    WorkLine line;
    const uint32_t length = line.length(a, lane);
    // (Rounded up but for the last bits of the product: at most two stretches
    // more than wanted.)
    const float share = ceilf((float)length * a.inverse_stretches * 0.999999f);
    const uint32_t per = uniform(share > 1.0f ? (uint32_t)share : 1);
    if ((uint64_t)stretch * per >= length) return;
    const uint32_t stretch_begin = stretch * per, stretch_end = min(stretch_begin + per, length);

    __shared__ uint32_t lds_rows[4][32];
    __shared__ float lds_scale[4][2][G][32];
    // A tile's value codes, a row every D + 16 bytes: the four rows that the
    // lane quarters read at once then lie on different banks.
    __shared__ __attribute__((aligned(16))) uint8_t lds_values[4][32 * (D + 16)];
    __shared__ float lds_acc[2][kTileRows][D + 4];
    __shared__ float lds_state[2][2][kTileRows];

    const uint32_t kv_width = c.kv_heads * D, gpr = kv_width / 64;
    for (uint32_t at = stretch_begin; at < stretch_end;) {
    int owner;
    if (!line.find(a, at, lane, owner)) return;
    const uint32_t b = line.base + owner, tokens = lane_of(line.n, owner), first = lane_of(line.first, owner);
    const uint32_t units = lane_of(line.units, owner), tiles = row_tiles(a, tokens);
    // The sequence's first unit, and this part of one of its row tiles.
    const uint32_t seq_begin = add_units(line.before, lane_of(line.upto, owner)) - tiles * units;
    const uint32_t tile = uniform((at - seq_begin) / units), from = (at - seq_begin) - tile * units;
    if (tile >= tiles) return;  // (starts that fall)
    const uint32_t count = min(units - from, stretch_end - at);
    const bool alone = count == units;
    const uint32_t record = 2 * stretch + (at == stretch_begin ? 0 : 1);
    if (at == seq_begin && kvh == 0 && threadIdx.x == 0) a.plan[b] = u4{per, seq_begin, units, 0};  // for the join
    at += count;
    const uint32_t start = a.p.batch.row_starts ? a.p.batch.row_starts[b] : b;
    // This lane's query row: token t, head kvh * ratio + r; it sees positions
    // up to `limit`.
    const uint32_t f = tile * kTileRows + (n & 7);
    const uint32_t t = by_ratio(a, f), r = f - t * a.ratio;
    const bool active = t < tokens;
    const uint32_t last_t = min(by_ratio(a, tile * kTileRows + kTileRows - 1), tokens - 1);
    const uint32_t first_t = by_ratio(a, tile * kTileRows);
    const auto place = [&](uint32_t token) {  // its position, at most the tables' last
        const uint64_t p = (uint64_t)first + token;
        return p < a.held ? (uint32_t)p : a.held - 1;
    };
    const uint32_t limit = place(t), common = uniform(place(first_t));
    const uint32_t begin = from * kUnit;
    uint32_t end = uniform(place(last_t)) + 1;
    if (begin >= end) continue;  // (no row of the tile sees this part)
    if (end - begin > count * kUnit) end = begin + count * kUnit;

    const uint32_t *table = a.p.batch.tables + (size_t)b * a.p.batch.table_pages;
    const uint8_t *k_base = c.k_codes + kvh * D + 16 * quarter;
    const uint8_t *v_base = c.v_codes + kvh * D;
    // Lanes 0..31 load the key scales of position lane, 32..63 the value scales.
    const uint16_t *scale_base = reinterpret_cast<const uint16_t *>(lane < 32 ? c.k_scales : c.v_scales) + kvh * G;

    // The page of this lane's position (lane % 32) of the tile at `base`. Loads
    // complete in order: a tile's pages are asked for a tile ahead of its
    // rows, so that they do not wait for the loads between.
    struct Place {
        uint32_t page, within;
    };
    const auto lookup = [&](uint32_t base) {
        const uint32_t p = min(base + (lane & 31), end - 1);
        const uint32_t at = a.page_shift < 32 ? p >> a.page_shift : p / c.page_size;
        return Place{table[at], p - at * c.page_size};
    };
    struct Tile {
        uint4 k[2][G];
        uint4 v[2 * G];  // 16-byte piece lane + 64 j of the tile's rows
        uint16_t scale[G];
        uint32_t there;  // of the 32 positions, those with a row
    };
    const auto load = [&](Tile &tile, const Place &at, uint32_t base) {
        const bool has_row = (at.page < c.pages) & (base + (lane & 31) < end);
        tile.there = (uint32_t)__ballot(has_row);
        const uint32_t safe = has_row ? at.page * c.page_size + at.within : 0;
        // (In 16-byte pieces: a layer's code plane is below 64 GiB.)
        if (lane < 32) lds_rows[wave][lane] = safe * (kv_width / 16);
#pragma unroll
        for (int g = 0; g < G; ++g) tile.scale[g] = scale_base[(size_t)safe * gpr + g];
        wave_fence();
        const uint32_t k0 = lds_rows[wave][n], k1 = lds_rows[wave][16 + n];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            tile.k[0][g] = *reinterpret_cast<const uint4 *>(k_base + ((size_t)k0 << 4) + 64 * g);
            tile.k[1][g] = *reinterpret_cast<const uint4 *>(k_base + ((size_t)k1 << 4) + 64 * g);
        }
#pragma unroll
        for (int j = 0; j < 2 * G; ++j) {
            const uint32_t at = lane + 64 * j, r = lds_rows[wave][at / kPieces];
            tile.v[j] = *reinterpret_cast<const uint4 *>(v_base + ((size_t)r << 4) + 16 * (at % kPieces));
        }
        // Every load of a tile is asked for before the tile in hand is used.
        __builtin_amdgcn_sched_barrier(0);
    };

    uint32_t base = begin + 32 * wave;
    Place ahead = lookup(base), after = lookup(base + kUnit);

    // This lane's term of the query row, scaled by a power of two to below 2^8.
    const size_t row = (size_t)start + t;
    h8 q[G][2];
    float qs;
    {
        f4 x[G][4];
        float top = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const f4 *src = reinterpret_cast<const f4 *>(a.p.query + (active ? row * a.p.query_stride + (kvh * a.ratio + r) * D + 64 * g + 16 * quarter : 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[g][i] = active ? src[i] : f4{0.0f, 0.0f, 0.0f, 0.0f};
                top = fmaxf(top, fmaxf(fmaxf(fabsf(x[g][i].x), fabsf(x[g][i].y)), fmaxf(fabsf(x[g][i].z), fabsf(x[g][i].w))));
            }
        }
        top = row_max(top);
        int e = 0;
        if (top > 0.0f && top < INFINITY) (void)__builtin_frexpf(top, &e);
        e = e < -100 ? -100 : e > 126 ? 126 : e;  // (what undoes it is finite)
        const float up = __builtin_ldexpf(1.0f, 8 - e);
        qs = a.scaling * __builtin_ldexpf(kCodeScale, e - 8);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float y[4] = {x[g][i].x * up, x[g][i].y * up, x[g][i].z * up, x[g][i].w * up};
                u2 hi, lo;
                two_terms(y, hi, lo);
                const h4 mine = __builtin_bit_cast(h4, term ? lo : hi);
#pragma unroll
                for (int j = 0; j < 4; ++j) q[g][i / 2][4 * (i & 1) + j] = mine[j];
            }
    }

    float m = -INFINITY, l = 0.0f;
    float e_w = -100.0f;  // acc is in units of 2^e_w
    f4 acc[G][4];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};

    const auto use = [&](const Tile &tile, uint32_t base) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            // (No finite number: NaN. An infinite key scale would else make
            // scores of one sign, and weights of 0 where that is below.)
            const float scale = dev::f16_bits_to_f32(tile.scale[g]);
            lds_scale[wave][lane >> 5][g][lane & 31] = fmaf(scale, 0.0f, scale);
        }
        wave_fence();
        f4 both[2];
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            both[blk] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint4 w = tile.k[blk][g];
                f4 x = mma(codes8(w.x, w.y), q[g][0], f4{0.0f, 0.0f, 0.0f, 0.0f});
                x = mma(codes8(w.z, w.w), q[g][1], x);
                const f4 ks = *reinterpret_cast<const f4 *>(&lds_scale[wave][0][g][16 * blk + 4 * quarter]);
#pragma unroll
                for (int i = 0; i < 4; ++i) both[blk][i] = fmaf(ks[i], x[i], both[blk][i]);
            }
        }
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float s0 = both[0][i] + dev::xor_lane<8>(both[0][i]), s1 = both[1][i] + dev::xor_lane<8>(both[1][i]);
            // (Rounded here, in base 2: a multiply-add of the products against
            // the scaled maximum would leave the maximum's own rounding error,
            // which is no small number where scores are large.)
            s[i] = settled((term ? s1 : s0) * qs);
        }
        const bool whole = tile.there == 0xffffffffu && base + 31 <= common;
        const int mine = 16 * term + 4 * quarter;  // this lane's first position of the tile
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!(tile.there >> (mine + i) & 1u) || base + mine + i > limit) s[i] = -INFINITY;
        }
        const float mx = row_max(fmaxf(fmaxf(m, fmaxf(s[0], s[1])), fmaxf(s[2], s[3])));
        // A row that has seen nothing yet: weights of 0 against any maximum.
        const float low = mx == -INFINITY ? 0.0f : mx;
        const float turn = m - low;  // log2 of what earlier weights lose
        m = mx;
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = exp2_fast(s[i] - low);
        // The weights with their value scales, and the power of two that
        // brings the row's largest (of earlier ones too) near f16's top.
        float w[G][4], largest = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const f4 vs = *reinterpret_cast<const f4 *>(&lds_scale[wave][1][g][mine]);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[g][i] = p[i] * vs[i];
            if (!whole) {  // (a scale that is no number must not reach rows that do not see it)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[g][i] = s[i] == -INFINITY ? 0.0f : w[g][i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) largest = fmaxf(largest, fabsf(w[g][i]));
        }
        // (Of numbers: a scale that is none is its 64 dimensions' alone.)
        largest = row_max(largest);
        const float e_now = fmaxf(fmaxf(e_w + ceilf(turn), (float)((int)(__float_as_uint(largest) >> 23) - 126)), -100.0f);
        if (__ballot(turn != 0.0f || e_now != e_w)) {
            l *= exp2_fast(turn);
            const float less = exp2_fast(turn + (e_w - e_now));
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[g][i] *= less;
            e_w = e_now;
        }
        l += (p[0] + p[1]) + (p[2] + p[3]);
        const float up = exp2_fast(12.0f - e_w);
#pragma unroll
        for (int j = 0; j < 2 * G; ++j) {
            const uint32_t at = lane + 64 * j;
            *reinterpret_cast<uint4 *>(&lds_values[wave][at / kPieces * (D + 16) + at % kPieces * 16]) = tile.v[j];
        }
        wave_fence();
#pragma unroll
        for (int g = 0; g < G; ++g) {
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = *reinterpret_cast<const uint32_t *>(
                    &lds_values[wave][(16 * (i / 4) + 4 * quarter + (i & 3)) * (D + 16) + 64 * g + 4 * n]);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[g][i] *= up;
            u2 hi, lo;
            two_terms(w[g], hi, lo);
            // Block 0's four positions, then block 1's: this column's own
            // term of its own block and of the other lane's.
            const u4 mixed = {take_other<true>(hi.x, lo.x), take_other<true>(hi.y, lo.y),
                              take_other<false>(lo.x, hi.x), take_other<false>(lo.y, hi.y)};
            const h8 weights = __builtin_bit_cast(h8, mixed);
            acc[g][0] = mma(codes_across<0>(v), weights, acc[g][0]);
            acc[g][1] = mma(codes_across<1>(v), weights, acc[g][1]);
            acc[g][2] = mma(codes_across<2>(v), weights, acc[g][2]);
            acc[g][3] = mma(codes_across<3>(v), weights, acc[g][3]);
        }
    };

    if (base < end) {
        // (The loads behind the range are of pool row 0; waits count on them.)
        Tile even, odd;
        load(even, ahead, base);
        for (; base + kUnit < end; base += 2 * kUnit) {
            ahead = lookup(base + 2 * kUnit);
            load(odd, after, base + kUnit);
            use(even, base);
            after = lookup(base + 3 * kUnit);
            load(even, ahead, base + 2 * kUnit);
            use(odd, base + kUnit);
        }
        if (base < end) use(even, base);
    }

    // The terms' sums, and the lanes' of l.
    l = row_sum(l);
    const float back = exp2_fast(e_w - 12.0f) * kCodeScale;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[g][i][j] = (acc[g][i][j] + dev::xor_lane<8>(acc[g][i][j])) * back;
    float M = m;
    const int slot_row = n & 7;
    const bool writes = term == 0;
    // The four wavefronts' states into the first's: 2 and 3 hand theirs to 0
    // and 1, then 1 to 0.
#pragma unroll
    for (int half = 2; half >= 1; half /= 2) {
        if (wave >= half && wave < 2 * half && writes) {
            const int slot = wave - half;
            if (quarter == 0) {
                lds_state[slot][0][slot_row] = M;
                lds_state[slot][1][slot_row] = l;
            }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f4 *>(&lds_acc[slot][slot_row][64 * g + 16 * quarter + 4 * i]) =
                        f4{acc[g][0][i], acc[g][1][i], acc[g][2][i], acc[g][3][i]};
        }
        __syncthreads();
        if (wave < half) {
            const float m2 = lds_state[wave][0][slot_row], l2 = lds_state[wave][1][slot_row];
            const float top = fmaxf(M, m2), low = top == -INFINITY ? 0.0f : top;
            const float f1 = exp2_fast(M - low), f2 = exp2_fast(m2 - low);
            M = top;
            l = l * f1 + l2 * f2;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f4 other = *reinterpret_cast<const f4 *>(&lds_acc[wave][slot_row][64 * g + 16 * quarter + 4 * i]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[g][k][i] = acc[g][k][i] * f1 + other[k] * f2;
                }
        }
        __syncthreads();
    }
    if (wave != 0 || !active || !writes) continue;
    if (!alone) {
        const size_t rec = ((size_t)record * c.kv_heads + kvh) * kTileRows + slot_row;
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
        continue;
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
}

// ---- many query rows ----
//
// 128 query rows of a workgroup, 32 a wavefront, over 64 positions at a time
// that the four wavefronts share: codes are turned into f16 once, on their way
// to LDS (keys by position, values by dimension), and read from there as
// operands of 32 x 32 x 16 products, each by both terms of the queries or
// weights:
//   scores  [position][row] = K Q^T, two blocks of 32 positions. Lane l holds
//           row l % 32, positions 8 i + 4 (l / 32) + 0..3 of a block;
//   values  [dimension][row] += V^T P^T, 16 positions at a time, counted in
//           that order, so that weights stay in their lane.
// Value scales: with vm the largest of a position's, the softmax runs over
// score + log2(vm), so its weights P = p vm are at most 1 (2^3: what they are
// taken against moves only when it is passed by more) and so are P vs / vm =
// p vs. Both terms of 2^12 p vs then keep 2^-22 of the row's largest; the sum
// is of 2^12 p = 2^12 P / vm. (vs / vm and 1 / vm are worked out once a tile:
// 133 -> 131 us in a long run of the chunk below.) Score and log2(vm) are one
// f32: its rounding is as large as the score's own, half a step.
// What weights are taken against is held as `low`, 12 below the largest score
// of the time: scores less `low` stay below 16, f16's range, and `low` itself,
// not the maximum, is what sums and records are relative to. From 2^26 on,
// where f32 cannot hold the maximum less 12, it is the maximum.
// Two LDS buffers and a barrier a tile: tile i + 1 is converted and tile i + 2
// asked for at the start of tile i. Units of 128 positions and at least one a
// workgroup: a start costs 5 us, so units of 64 (402 rows x 2 from position 0
// on: 27.4 us) or two a workgroup (33.6) lose to it (26.6).
//
// Bound by issue: 512 tokens of 16 heads over 8 x 128 at 7680 take 104 us and
// the join 11 (33 GFLOP, 290 TFLOP/s; the two terms are twice that), in which
// the vector unit is busy 60 % and the matrix cores 28 % of the cycles, with
// two wavefronts a SIMD (256 registers) that overlap little. A tile of a
// wavefront takes 8600 cycles: 2 x 1200 scores, 2 x 250 maximum, 2 x 1400
// weights and values, 2800 for the next tile (rows, conversion, loads).
// Converting between the products instead takes the same (it spills).
constexpr int kManyRows = 128;
constexpr int kManyPositions = 64;

typedef float f16v __attribute__((ext_vector_type(16)));

template <int D>
struct ManyLayout {
    static constexpr int G = D / 64;
    static constexpr int kKeys = 0;                                  // [64][D] f16
    static constexpr int kValues = kManyPositions * D * 2;           // [D][64] f16
    static constexpr int kScales = kValues + D * kManyPositions * 2;  // [64 / 4][G][4] f16: key scales
    static constexpr int kRatios = kScales + 2 * G * kManyPositions;  // [64 / 4][G][4] f32: value scales over vm
    static constexpr int kWeights = kRatios + 4 * G * kManyPositions;  // [2][64] f32: log2(vm), 1 / vm
    static constexpr int kBad = kWeights + 2 * kManyPositions * 4;   // [G] u64: positions whose value scale is no number
    static constexpr int kBuffer = (kBad + 8 * G + 511) / 512 * 512;  // (row addresses are put together bit by bit)
    static constexpr int kRows = 2 * kBuffer;                        // [4][64] pool rows in 16-byte pieces
    static constexpr int kPoolRows = kRows + 4 * kManyPositions * 4;  // [4][64] pool rows
    static constexpr int kThere = kPoolRows + 4 * kManyPositions * 4;  // [4] u64
    static constexpr int kBytes = kThere + 4 * 8;
    // A key row's 16-byte chunk c lies at c ^ key_turn(row), a value row's
    // (dimension's) at c ^ value_turn(d): the 16 lanes that read at once then
    // fall on all banks.
    static __device__ __forceinline__ int key_turn(int row) { return D % 128 == 0 ? row & 15 : row >> 1 & 7; }
    static __device__ __forceinline__ int value_turn(int d) { return (d >> 1 ^ d >> 4) & 7; }
};

// A value that the compiler must take to be new here: what is worked out from
// it stays inside a loop, where it costs an instruction, instead of a register
// all through it.
__device__ __forceinline__ int anew(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

__device__ __forceinline__ f16v mma32(h8 a, h8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// The units (kManyRows rows by kUnit positions) of a sequence's row tiles:
// tile j ends by position first + (j / ratio + 1) * kUnit, so it has
// whole + j / ratio units, whole = ceil(first / kUnit) + 1 (+ 1: a token's
// heads over more than one tile). tiles_units(j): those of the tiles below j.
__device__ __forceinline__ uint32_t whole_units(const KernelArgs &a, uint32_t first) {
    return (min(first, a.held) + kUnit - 1) / kUnit + 1 + (a.ratio > (uint32_t)kManyRows ? 1 : 0);
}

__device__ __forceinline__ uint32_t tiles_units(const KernelArgs &a, uint32_t whole, uint32_t j) {
    const uint32_t q = by_ratio(a, j);
    return j * whole + a.ratio * (q * (q - 1) / 2) + q * (j - q * a.ratio);
}

template <int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : D == 128 ? 2 : 1) void paged_many_kernel(const KernelArgs a) {
    using Lay = ManyLayout<D>;
    constexpr int G = D / 64;
    constexpr uint32_t kPieces = D / 16;                   // 16-byte pieces of a head row's codes
    constexpr int kValueItems = (2 * D + 255) / 256;       // (eight positions, four dimensions) a thread
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = (int)uniform(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const qwh_paged_cache &c = a.p.cache;
    const uint32_t kvh = blockIdx.x % c.kv_heads, stretch = blockIdx.x / c.kv_heads;
    WorkLine line;
    const uint32_t length = line.length(a, lane, kManyRows);
    const float share = ceilf((float)length * a.inverse_stretches_many * 0.999999f);
    const uint32_t per = uniform(share > 1.0f ? (uint32_t)share : 1);
    if ((uint64_t)stretch * per >= length) return;
    const uint32_t stretch_begin = stretch * per, stretch_end = min(stretch_begin + per, length);
    const uint32_t kv_width = c.kv_heads * D, gpr = kv_width / 64;

    for (uint32_t at = stretch_begin; at < stretch_end;) {
        int owner;
        if (!line.find(a, at, lane, owner, kManyRows)) return;
        const uint32_t b = line.base + owner, tokens = lane_of(line.n, owner), first = lane_of(line.first, owner);
        const uint32_t whole = whole_units(a, first), tiles = row_tiles(a, tokens, kManyRows);
        const uint32_t seq_begin = add_units(line.before, lane_of(line.upto, owner)) - tiles_units(a, whole, tiles);
        // The tile that unit `at` lies in: the last that begins at or below it.
        uint32_t tile = 0, step = 1;
        while (step * 64 < tiles) step *= 64;
        for (; step >= 1; step /= 64) {
            const uint32_t j = tile + lane * step;
            const uint64_t below = __ballot(j < tiles && tiles_units(a, whole, j) <= at - seq_begin);
            if (!below) return;  // (starts that fall)
            tile += step * (63 - __builtin_clzll(below));
            if (step == 1) break;
        }
        const uint32_t from = at - seq_begin - tiles_units(a, whole, tile), units = whole + by_ratio(a, tile);
        if (from >= units) return;  // (starts that fall)
        const uint32_t count = min(units - from, stretch_end - at);
        const bool alone = count == units;
        const uint32_t record = 2 * stretch + (at == stretch_begin ? 0 : 1);
        if (at == seq_begin && kvh == 0 && tid == 0) a.plan[b] = u4{per, seq_begin, whole, 1};  // for the join
        at += count;
        const uint32_t start = a.p.batch.row_starts ? a.p.batch.row_starts[b] : b;
        const uint32_t f = tile * kManyRows + 32 * wave + col;
        const uint32_t t = by_ratio(a, f), r = f - t * a.ratio;
        const bool active = t < tokens;
        const auto place = [&](uint32_t token) {  // its position, at most the tables' last
            const uint64_t p = (uint64_t)first + min(token, tokens - 1);
            return p < a.held ? (uint32_t)p : a.held - 1;
        };
        // Positions up to limit for this lane's row, up to `common` for every
        // row of the wavefront, up to `furthest` for some; `end` of the tile.
        const uint32_t limit = place(t);
        const uint32_t wave_first = tile * kManyRows + 32 * wave;
        const bool busy = by_ratio(a, wave_first) < tokens;
        const uint32_t common = uniform(place(by_ratio(a, wave_first)));
        const uint32_t furthest = uniform(place(by_ratio(a, wave_first + 31)));
        const uint32_t begin = from * kUnit;
        uint32_t end = uniform(place(by_ratio(a, tile * kManyRows + kManyRows - 1))) + 1;
        if (begin >= end) continue;  // (no row of the tile sees this part)
        if (end - begin > count * kUnit) end = begin + count * kUnit;

        const uint32_t *table = a.p.batch.tables + (size_t)b * a.p.batch.table_pages;
        // Wavefront 0 looks the pool rows up, lane by position.
        struct Place {
            uint32_t page, within;
        };
        const auto lookup = [&](uint32_t base) {
            const uint32_t p = min(base + lane, end - 1);
            const uint32_t page = a.page_shift < 32 ? p >> a.page_shift : p / c.page_size;
            return Place{table[page], p - page * c.page_size};
        };
        const auto put_rows = [&](const Place &p, uint32_t base, uint32_t slot) {
            const bool has_row = (p.page < c.pages) & (base + lane < end);
            const uint32_t safe = has_row ? p.page * c.page_size + p.within : 0;
            const uint64_t there = __ballot(has_row);
            reinterpret_cast<uint32_t *>(lds + Lay::kRows)[slot * kManyPositions + lane] = safe * (kv_width / 16);
            reinterpret_cast<uint32_t *>(lds + Lay::kPoolRows)[slot * kManyPositions + lane] = safe;
            if (lane == 0) reinterpret_cast<uint64_t *>(lds + Lay::kThere)[slot] = there;
        };
        // A tile on its way: raw codes and scales.
        uint4 k_raw[G];
        uint32_t v_raw[kValueItems][8];
        uint16_t scale_raw[G];
        const uint8_t *k_base = c.k_codes + kvh * D, *v_base = c.v_codes + kvh * D;
        const uint16_t *scale_base = reinterpret_cast<const uint16_t *>(wave == 0 ? c.k_scales : c.v_scales) + kvh * G;
        const auto load = [&](uint32_t slot) {
            const int tid = anew(threadIdx.x);
            const uint32_t *rows = reinterpret_cast<const uint32_t *>(lds + Lay::kRows) + slot * kManyPositions;
            if (wave < 2) {
                const size_t pool_row = reinterpret_cast<const uint32_t *>(lds + Lay::kPoolRows)[slot * kManyPositions + lane];
#pragma unroll
                for (int g = 0; g < G; ++g) scale_raw[g] = scale_base[pool_row * gpr + g];
            }
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const uint32_t piece = tid + 256 * j;
                k_raw[j] = *reinterpret_cast<const uint4 *>(k_base + ((size_t)rows[piece / kPieces] << 4) + 16 * (piece % kPieces));
            }
#pragma unroll
            for (int j = 0; j < kValueItems; ++j) {
                const int item = tid + 256 * j, eight = item / (D / 4), quad = item % (D / 4);
                if (2 * D % 256 != 0 && item >= 2 * D) break;
                // Positions 16 s + 4 h + 0..3 and 16 s + 8 + 4 h + 0..3 of eight 2 s + h.
                const u4 r0 = *reinterpret_cast<const u4 *>(rows + 16 * (eight / 2) + 4 * (eight & 1));
                const u4 r1 = *reinterpret_cast<const u4 *>(rows + 16 * (eight / 2) + 8 + 4 * (eight & 1));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v_raw[j][i] = *reinterpret_cast<const uint32_t *>(v_base + ((size_t)r0[i] << 4) + 4 * quad);
                    v_raw[j][4 + i] = *reinterpret_cast<const uint32_t *>(v_base + ((size_t)r1[i] << 4) + 4 * quad);
                }
            }
        };
        const auto convert = [&](uint32_t buffer) {
            uint8_t *buf = lds + buffer * Lay::kBuffer;
            const int tid = anew(threadIdx.x);
#pragma unroll
            for (int j = 0; j < G; ++j) {
                const int piece = tid + 256 * j, row = piece / (int)kPieces, chunk = 2 * (piece % (int)kPieces);
                uint8_t *dst = buf + Lay::kKeys + row * (2 * D);
                *reinterpret_cast<h8 *>(dst + 16 * (chunk ^ Lay::key_turn(row))) = codes8(k_raw[j].x, k_raw[j].y);
                *reinterpret_cast<h8 *>(dst + 16 * ((chunk + 1) ^ Lay::key_turn(row))) = codes8(k_raw[j].z, k_raw[j].w);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int j = 0; j < kValueItems; ++j) {
                const int item = tid + 256 * j, eight = item / (D / 4), quad = item % (D / 4);
                if (2 * D % 256 != 0 && item >= 2 * D) break;
                uint8_t *dst = buf + Lay::kValues;
                *reinterpret_cast<h8 *>(dst + (4 * quad) * 128 + 16 * (eight ^ Lay::value_turn(4 * quad))) = codes_across<0>(v_raw[j]);
                *reinterpret_cast<h8 *>(dst + (4 * quad + 1) * 128 + 16 * (eight ^ Lay::value_turn(4 * quad + 1))) = codes_across<1>(v_raw[j]);
                *reinterpret_cast<h8 *>(dst + (4 * quad + 2) * 128 + 16 * (eight ^ Lay::value_turn(4 * quad + 2))) = codes_across<2>(v_raw[j]);
                *reinterpret_cast<h8 *>(dst + (4 * quad + 3) * 128 + 16 * (eight ^ Lay::value_turn(4 * quad + 3))) = codes_across<3>(v_raw[j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (wave == 1) {
                // Value scales that are no number count as 0 here, and the
                // rows that see them are told apart in use(). (A position of
                // zero scales counts as one of f16's least: its weight still
                // belongs to the sum.)
                float vm = 0x1p-24f;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const float vs = fabsf(dev::f16_bits_to_f32(scale_raw[g]));
                    const bool bad = !(vs < INFINITY);
                    const uint64_t some = __ballot(bad);
                    if (lane == 0) reinterpret_cast<uint64_t *>(buf + Lay::kBad)[g] = some;
                    if (bad) scale_raw[g] = 0;
                    vm = fmaxf(vm, bad ? 0.0f : vs);
                }
                const float inverse = 1.0f / vm;
                float *weights = reinterpret_cast<float *>(buf + Lay::kWeights);
                weights[lane] = __builtin_amdgcn_logf(vm);
                weights[kManyPositions + lane] = inverse;
                float *ratios = reinterpret_cast<float *>(buf + Lay::kRatios) + lane / 4 * (4 * G) + lane % 4;
#pragma unroll
                for (int g = 0; g < G; ++g) ratios[4 * g] = dev::f16_bits_to_f32(scale_raw[g]) * inverse;
            }
            if (wave == 0) {
                uint16_t *scales = reinterpret_cast<uint16_t *>(buf + Lay::kScales) + lane / 4 * (4 * G) + lane % 4;
#pragma unroll
                for (int g = 0; g < G; ++g)  // (an infinity: NaN, as in the few rows' form)
                    scales[4 * g] = (scale_raw[g] & 0x7c00u) == 0x7c00u ? (uint16_t)0x7e00u : scale_raw[g];
            }
        };

        // The query rows' two terms, times log2(e) / sqrt(D) and what brings
        // products with the codes back, scaled by a power of two a row to
        // below 2^8; the scores by `fix` afterwards.
        const size_t row = (size_t)start + t;
        h8 qh[G][4], ql[G][4];
        float fix;
        {
            f4 x[G][4][2];
            float top = 0.0f;
            const float *src = a.p.query + (active ? row * a.p.query_stride + (kvh * a.ratio + r) * D + 8 * half : 0);
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const f4 y = active ? *reinterpret_cast<const f4 *>(src + 64 * g + 16 * k + 4 * i) : f4{0.0f, 0.0f, 0.0f, 0.0f};
                        x[g][k][i] = y;
                        top = fmaxf(top, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
                    }
            top = fmaxf(top, dev::xor_lane<32>(top));
            int e = 0;
            if (top > 0.0f && top < INFINITY) (void)__builtin_frexpf(top, &e);
            e = e < -100 ? -100 : e > 126 ? 126 : e;  // (what undoes it is finite)
            const float up = a.scaling * __builtin_ldexpf(1.0f, 8 - e);
            fix = __builtin_ldexpf(kCodeScale, e - 8);
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const f4 y = x[g][k][i] * up;
                        const float z[4] = {y.x, y.y, y.z, y.w};
                        u2 hi, lo;
                        two_terms(z, hi, lo);
                        const h4 h = __builtin_bit_cast(h4, hi), l = __builtin_bit_cast(h4, lo);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            qh[g][k][4 * i + j] = h[j];
                            ql[g][k][4 * i + j] = l[j];
                        }
                    }
        }

        float low = -INFINITY, l = 0.0f;
        uint32_t not_numbers = 0;  // bit g: the row sees a value scale that is none
        f16v acc[G][2];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i) acc[g][i] = f16v{};

        // A block of 32 positions: base + 32 blk on.
        const auto use = [&](uint32_t buffer, int blk, uint32_t base, uint32_t there) {
            // (Products before staging where a SIMD's two wavefronts meet:
            // 134 -> 131 us for the chunk in a long run.)
            __builtin_amdgcn_s_setprio(1);
            const uint8_t *buf = lds + buffer * Lay::kBuffer;
            const int col = anew(lane & 31), half = anew(lane >> 5);
            // This lane's four positions 8 i + 4 half of the block: key or
            // value scales over vm, and log2(vm) or 1 / vm.
            const uint8_t *scales = buf + Lay::kScales + (8 * blk + half) * (8 * G);
            const auto scale4 = [&](int g, int i) { return *reinterpret_cast<const h4 *>(scales + i * (16 * G) + 8 * g); };
            const uint8_t *ratios = buf + Lay::kRatios + (8 * blk + half) * (16 * G);
            const auto ratio4 = [&](int g, int i) { return *reinterpret_cast<const f4 *>(ratios + i * (32 * G) + 16 * g); };
            const uint8_t *weights = buf + Lay::kWeights + (32 * blk + 4 * half) * 4;
            const auto weight4 = [&](int which, int i) { return *reinterpret_cast<const f4 *>(weights + which * (4 * kManyPositions) + 32 * i); };
            // A chunk's place differs from the lane's first one in the bits
            // of the chunk's number: one exclusive or, no sum. (Chunk 8 g + 2 k
            // + half of key row 32 blk + col; chunk 4 blk + i + half of value
            // row 64 g + 32 k + col, whose turn is the column's and 4 g + 2 k.)
            const int key_at = (32 * blk + col) * (2 * D) + 16 * (half ^ Lay::key_turn(col));
            const int value_at = col * 128 + 16 * ((half ^ Lay::value_turn(col) ^ 4 * blk) & 7);
            const auto key_chunk = [&](int g, int k) {
                const int chunk = D % 128 == 0 ? key_at ^ 16 * (8 * g + 2 * k) : (key_at ^ 16 * (2 * k)) + 128 * g;
                return *reinterpret_cast<const h8 *>(buf + Lay::kKeys + chunk);
            };
            uint64_t bad = 0;
#pragma unroll
            for (int g = 0; g < G; ++g) bad |= reinterpret_cast<const uint64_t *>(buf + Lay::kBad)[g];
            const bool some_bad = uniform((uint32_t)(bad >> 32 * blk)) != 0;
            // A group's chunks are read while the one before is multiplied.
            h8 key[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) key[k] = key_chunk(0, k);
            float s[16];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                f16v x = f16v{};
                h8 next[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x = mma32(key[k], ql[g][k], x);
                    x = mma32(key[k], qh[g][k], x);
                    if (g + 1 < G) next[k] = key_chunk(g + 1, k);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const h4 ks = scale4(g, i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[4 * i + j] = fmaf((float)ks[j], x[4 * i + j], g == 0 ? 0.0f : s[4 * i + j]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) key[k] = next[k];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f4 lv = weight4(0, i);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[4 * i + j] = fmaf(s[4 * i + j], fix, lv[j]);
            }
            // (Branches around scores and weights only: one around the sums
            // would hold them twice, and spill.)
            if (there != ~0u || base + 31 > common || some_bad) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t within = 8 * i + 4 * half + j;
                        if (!(there >> within & 1u) || base + within > limit) s[4 * i + j] = -INFINITY;
                    }
                if (some_bad) {
                    uint32_t seen = there;
                    if (base + 31 > limit) seen &= base > limit ? 0u : ~0u >> (31 - (limit - base));
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const uint32_t none = (uint32_t)(reinterpret_cast<const uint64_t *>(buf + Lay::kBad)[g] >> 32 * blk);
                        not_numbers |= (none & seen) != 0 ? 1u << g : 0u;
                    }
                }
            }
            const auto value_chunk = [&](int g, int k, int i) {
                return *reinterpret_cast<const h8 *>(buf + Lay::kValues + (64 * g + 32 * k) * 128 + (value_at ^ 16 * ((i ^ (4 * g + 2 * k)) & 7)));
            };
            h8 value[G][2];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int k = 0; k < 2; ++k) value[g][k] = value_chunk(g, k, 0);
            __builtin_amdgcn_sched_barrier(0);
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[i]);
            mx = fmaxf(mx, dev::xor_lane<32>(mx));
            // `low` moves when some row's maximum is past it by 2^15, 2^3
            // more than it was put below one, or the row has none yet.
            if (__ballot(mx - low > 15.0f)) {
                const float below = mx - 12.0f;
                const float to = fmaxf(low, mx - below > 14.0f ? mx : below);  // (16 and more: f32's steps there)
                const float less = exp2_fast(low - (to == -INFINITY ? 0.0f : to));
                l *= less;
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[g][i][j] *= less;
                low = to;
            }
            const float against = low == -INFINITY ? 0.0f : low;
            // 16 positions at a time: weights, then their products, the next
            // ones' values on their way meanwhile.
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const f4 rv[2] = {weight4(1, i), weight4(1, i + 1)};
                f4 vs[G][2];
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int k = 0; k < 2; ++k) vs[g][k] = ratio4(g, i + k);
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = exp2_fast(s[4 * i + j] - against);
                    l = fmaf(p[j], rv[j / 4][j & 3], l);
                }
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    float w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = settled(p[j] * vs[g][j / 4][j & 3]);
                    h8 hi, lo;
#pragma unroll
                    for (int j = 0; j < 8; ++j) hi[j] = (_Float16)w[j];
#pragma unroll
                    for (int j = 0; j < 8; ++j) lo[j] = rest(w[j], hi[j]);
#pragma unroll
                    for (int k = 0; k < 2; ++k) acc[g][k] = mma32(value[g][k], lo, acc[g][k]);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        acc[g][k] = mma32(value[g][k], hi, acc[g][k]);
                        if (i == 0) value[g][k] = value_chunk(g, k, 2);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            __builtin_amdgcn_s_setprio(0);
        };

        // (The last part's reads of the buffers are done: its use() is behind
        // a barrier for all but the last tile, and the rows' slots are not
        // read in use().)
        __syncthreads();
        Place ahead{};
        if (wave == 0) {
            const Place p0 = lookup(begin), p1 = lookup(begin + kManyPositions), p2 = lookup(begin + 2 * kManyPositions);
            ahead = lookup(begin + 3 * kManyPositions);
            put_rows(p0, begin, 0);
            put_rows(p1, begin + kManyPositions, 1);
            put_rows(p2, begin + 2 * kManyPositions, 2);
        }
        __syncthreads();
        load(0);
        convert(0);
        load(1);
        uint32_t i = 0;
        for (uint32_t base = begin; base < end; base += kManyPositions, ++i) {
            __syncthreads();
            if (wave == 0) {
                put_rows(ahead, base + 3 * kManyPositions, (i + 3) & 3);
                ahead = lookup(base + 4 * kManyPositions);
            }
            convert((i + 1) & 1);
            __builtin_amdgcn_sched_barrier(0);
            load((i + 2) & 3);
            __builtin_amdgcn_sched_barrier(0);
            const uint64_t there = reinterpret_cast<const uint64_t *>(lds + Lay::kThere)[i & 3];
#pragma unroll 1
            for (int blk = 0; blk < 2; ++blk)
                if (busy && base + 32 * blk <= furthest) use(i & 1, blk, base + 32 * blk, (uint32_t)(there >> 32 * blk));
        }

        if (!active) continue;
        l += dev::xor_lane<32>(l);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float more = not_numbers >> g & 1u ? __builtin_nanf("") : 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[g][i][j] += more;
        }
        // Lane: dimensions 64 g + 32 k + 8 i + 4 half + 0..3 of its row.
        if (!alone) {
            const size_t rec = ((size_t)record * c.kv_heads + kvh) * kManyRows + 32 * wave + col;
            if (half == 0) {
                a.sums_many[2 * rec] = low;
                a.sums_many[2 * rec + 1] = l;
            }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<f4 *>(a.values_many + rec * D + 64 * g + 32 * k + 8 * q + 4 * half) =
                            f4{acc[g][k][4 * q], acc[g][k][4 * q + 1], acc[g][k][4 * q + 2], acc[g][k][4 * q + 3]} * kCodeScale;
            continue;
        }
        const float inv = l == 0.0f ? 0.0f : kCodeScale / l;
        float *out = a.p.out + (row * a.p.heads + kvh * a.ratio + r) * D + 4 * half;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<f4 *>(out + 64 * g + 32 * k + 8 * q) =
                        f4{acc[g][k][4 * q], acc[g][k][4 * q + 1], acc[g][k][4 * q + 2], acc[g][k][4 * q + 3]} * inv;
    }
}

// Joins the records of a query row (one wavefront) in the order of its
// positions. Rows whose tile one workgroup took whole were written by it.
// Bound by latency: the chain row, plan, records; 3.6 us for one row of 16
// heads, 11 for 512.
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const KernelArgs a, uint32_t rows) {
    constexpr int G = D / 64;
    const int lane = threadIdx.x & 63;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t row = uniform((uint32_t)(unit / a.p.heads)), h = uniform((uint32_t)(unit % a.p.heads));
    if (row >= rows) return;
    uint32_t b, t;
    if (!paged_row(a.p.batch, row, lane, b, t)) return;
    b = uniform(b);
    t = uniform(t);
    const u4 plan = a.plan[b];
    const uint64_t seen64 = (uint64_t)a.p.batch.first[b] + t + 1;
    const uint32_t seen = seen64 < a.held ? (uint32_t)seen64 : a.held;
    // (Starts that fall can leave a sequence without a plan. Whatever an
    // earlier call left there, the form is one that this call runs, and
    // stretches are held to that form's records.)
    const bool many = paged::joins_many(plan.w, a.few_rows);
    const uint32_t per = max(plan.x, 1u), tile_rows = many ? kManyRows : kTileRows;
    const uint32_t kvh = h / a.ratio, f = t * a.ratio + (h - kvh * a.ratio);
    const uint32_t tile = f / tile_rows, slot = f - tile * tile_rows;
    // The tile's units.
    const uint32_t units = many ? plan.z + by_ratio(a, tile) : plan.z;
    const uint32_t begin = plan.y + (many ? tiles_units(a, plan.z, tile) : tile * units);
    const uint32_t first = begin / per, last = (begin + units - 1) / per;
    if (first == last) return;
    // Stretches that hold positions this row sees.
    const uint32_t most = many ? a.stretches_most_many : a.stretches_most;
    const uint32_t used = min(min(last, (begin + (seen - 1) / kUnit) / per) - first + 1, most);
    const float *sums = many ? a.sums_many : a.sums, *values = many ? a.values_many : a.values;
    float M = -INFINITY, L = 0.0f, acc[G];
#pragma unroll
    for (int g = 0; g < G; ++g) acc[g] = 0.0f;
    for (uint32_t s0 = 0; s0 < used; s0 += 4) {
        float m[4], l[4], v[4][G];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t s = min(first + min(s0 + k, used - 1), most - 1);
            const size_t rec = ((size_t)(2 * s + (s * per < begin ? 1 : 0)) * a.p.cache.kv_heads + kvh) * tile_rows + slot;
            m[k] = sums[2 * rec];
            l[k] = sums[2 * rec + 1];
#pragma unroll
            for (int g = 0; g < G; ++g) v[k][g] = values[rec * D + 64 * g + lane];
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

// Workgroups that a CU holds at once, by the kernels' registers.
uint32_t resident_few(uint32_t head_dim) { return head_dim == 64 ? 3 : 2; }
uint32_t resident_many(uint32_t head_dim) { return head_dim == 64 ? 3 : head_dim == 128 ? 2 : 1; }

// Stretches of a key/value head: as many workgroups as the device holds.
uint32_t wanted_stretches(int cus, const PagedAttentionArgs &a, uint32_t resident) {
    const uint32_t groups = resident * (uint32_t)(cus > 0 ? cus : 256);
    return groups > a.cache.kv_heads ? groups / a.cache.kv_heads : 1;
}

// Stretches at most: the division's rounding, and a whole round of the dies.
uint32_t most_stretches(int cus, const PagedAttentionArgs &a, uint32_t resident) {
    return (wanted_stretches(cus, a, resident) + 2 + kDies - 1) / kDies * kDies;
}

paged::Forms forms_of(const PagedAttentionArgs &a) {
    return paged::forms_of(a.batch, a.heads / a.cache.kv_heads, (uint64_t)a.batch.table_pages * a.cache.page_size);
}

// Two records a stretch and head, each of a tile's rows.
uint64_t record_rows_few(int cus, const PagedAttentionArgs &a) {
    return forms_of(a).few ? 2ull * most_stretches(cus, a, resident_few(a.cache.head_dim)) * a.cache.kv_heads * kTileRows : 0;
}
uint64_t record_rows_many(int cus, const PagedAttentionArgs &a) {
    return forms_of(a).many ? 2ull * most_stretches(cus, a, resident_many(a.cache.head_dim)) * a.cache.kv_heads * kManyRows : 0;
}

template <int D>
hipError_t launch_attention(hipStream_t s, const KernelArgs &k) {
    const qwh_paged_batch &b = k.p.batch;
    const paged::Forms forms = forms_of(k.p);
    const uint32_t rows = b.row_starts ? b.rows : b.batch;
    const uint64_t join = ((uint64_t)rows * k.p.heads + 3) / 4;
    const uint64_t few = (uint64_t)k.stretches_most * k.p.cache.kv_heads, many = (uint64_t)k.stretches_most_many * k.p.cache.kv_heads;
    if (few > 0xffffffu || many > 0xffffffu || join > 0xffffffu) return hipErrorInvalidValue;
    if (forms.many) {
        constexpr int bytes = ManyLayout<D>::kBytes;
        static_assert(bytes <= 160 * 1024, "a CU's LDS");
        const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void *>(paged_many_kernel<D>),
                                                   hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (err != hipSuccess) return err;
        paged_many_kernel<D><<<(uint32_t)many, 256, bytes, s>>>(k);
    }
    if (forms.few) paged_few_kernel<D><<<(uint32_t)few, 256, 0, s>>>(k);
    // (Few rows over tables of one unit: nothing to join.)
    if (forms.many || k.held > kUnit) paged_join_kernel<D><<<(uint32_t)join, 256, 0, s>>>(k, rows);
    return hipGetLastError();
}

}  // namespace

size_t paged_attention_scratch_bytes(int cus, const PagedAttentionArgs &a) {
    return a.batch.batch * sizeof(u4) +
           (record_rows_few(cus, a) + record_rows_many(cus, a)) * (a.cache.head_dim + 2) * sizeof(float);
}

hipError_t launch_paged_attention(hipStream_t s, int cus, const PagedAttentionArgs &a, void *scratch, size_t scratch_bytes) {
    if (paged_attention_scratch_bytes(cus, a) > scratch_bytes) return hipErrorInvalidValue;
    KernelArgs k{};
    const uint32_t D = a.cache.head_dim;
    k.p = a;
    k.held = a.batch.table_pages * a.cache.page_size;  // (check_positions)
    k.ratio = a.heads / a.cache.kv_heads;
    k.ratio_magic = k.ratio == 1 ? 0 : (uint32_t)((1ull << 32) / k.ratio) + 1;
    k.page_shift = (a.cache.page_size & (a.cache.page_size - 1)) ? 32 : (uint32_t)__builtin_ctz(a.cache.page_size);
    k.few_rows = paged::few_rows(forms_of(a));
    k.stretches_most = most_stretches(cus, a, resident_few(D));
    k.inverse_stretches = 1.0f / (float)wanted_stretches(cus, a, resident_few(D));
    k.stretches_most_many = most_stretches(cus, a, resident_many(D));
    k.inverse_stretches_many = 1.0f / (float)wanted_stretches(cus, a, resident_many(D));
    k.scaling = kLog2e / sqrtf((float)D);
    k.plan = static_cast<u4 *>(scratch);
    k.values = reinterpret_cast<float *>(k.plan + a.batch.batch);
    k.sums = k.values + record_rows_few(cus, a) * D;
    k.values_many = k.sums + record_rows_few(cus, a) * 2;
    k.sums_many = k.values_many + record_rows_many(cus, a) * D;
    switch (a.cache.head_dim) {
    case 64: return launch_attention<64>(s, k);
    case 128: return launch_attention<128>(s, k);
    case 192: return launch_attention<192>(s, k);
    case 256: return launch_attention<256>(s, k);
    default: return hipErrorNotSupported;
    }
}

}  // namespace qwh
