// Drawing tokens from logits by temperature, top-k, top-p and min-p
// (qwh_sample_rows).
//
// Everything a draw asks for is a place in one order of the row, the largest
// logit first and the lower index first among equal ones: the sum of the
// first k weights (top-k), where the running sum reaches top_p times that
// (top-p), how many weights are at least min_p of the largest, and where the
// running sum passes u times what is left. The row is never sorted. A first
// launch goes over the logits once, 4096 of them a workgroup, and leaves for
// each such part a histogram over steps of a quarter octave of the weight
// (count and sum of weights) and its tokens of the best steps, up to 256 of
// them, by step. A second launch, a workgroup a row, adds the histograms and
// then needs only the tokens of the steps in which a place lies: mostly those
// kept beside the histograms, put in order in LDS.
//
// Steps and weights: y = l * 4 / (T ln 2) in 64 bits; step floor(y), the same
// grid in every part; within a step a token weighs 2^((y - floor(y)) / 4), 1
// to 2^(1/4), in whole multiples of 2^-37, and the step itself is a power of
// 2^(1/4) that comes in when steps are added. Within a step sums are integers,
// so the order of the LDS atomics does not matter, and count and sum share one
// 64-bit word and one atomic. Running sums over steps and tokens are 64-bit
// floats in a fixed order. Every sum, of a histogram, a step's split or a list,
// is of the same multiples, and the largest logit's step weighs 1: sums of
// tokens that share it are whole numbers of one weight, however they are added,
// and where top_p's or u's part of the whole is such a sum, the token is the one
// that the definition says. (Sums are compared as equal within 2^-47, which is
// what 64-bit additions may leave of larger ones: kReach, kPast.) Otherwise a
// draw differs from one in real numbers only where u falls within 4e-12 of a
// border (half a multiple; logits of more than 10^4 temperatures, whose y has
// fewer bits behind the point: in proportion more); with 32-bit weights, about
// one draw in 1000 of an unfiltered row of 151936 would.
//
// The first launch is bound by its vector instructions, f64 among them (64
// rows of 151936, 39 MB: 20 us; one row 5.4; parts of 8192 logits, 27 and 12),
// the second by latency: a chain of rounds over one workgroup, 14 us where the
// kept tokens are few, up to 45 where a place lies in the bulk of an
// unfiltered row and the workgroup goes over all its logits once more, 18 us
// at what one CU can have in flight.
#include <cmath>

#include "common.h"
#include "device.h"
#include "sample_plan.h"

namespace qwh {
namespace {

constexpr uint32_t kPart = 4096;       // logits of a first-pass workgroup
constexpr uint32_t kBins = 256;
constexpr uint32_t kDead = kBins - 1;  // the step of tokens that are not drawn, 63 octaves and more below the largest
constexpr uint32_t kShort = 256;       // tokens kept beside a part's histogram
constexpr uint32_t kList = 12288;      // tokens that the second pass takes into LDS
constexpr uint32_t kOrder = 256;       // and of these, puts in order
constexpr int kThreads = 1024;
constexpr int kUnitBits = 37;          // of a weight of 1 in a step's sum
constexpr int kCountShift = 50;        // 4096 * 2^(1/4) * 2^37 < 2^50: the count stands above the sum
constexpr double kReach = 1.0 - 0x1p-47, kPast = 1.0 + 0x1p-47;  // what a sum has to reach, or pass, for a part of it
constexpr uint32_t kPartsAtOnce = 32768;  // of a launch (152 MB of scratch)

// Order-preserving bits of a logit (0: NaN, never drawn); -0 counts as 0.
__device__ __forceinline__ uint32_t logit_key(float l) {
    if (l != l) return 0u;
    const uint32_t u = __float_as_uint(l + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float key_logit(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

constexpr uint32_t kKeyMinusInf = 0x007fffffu, kKeyPlusInf = 0xff800000u;

__device__ __forceinline__ bool is_greedy(const qwh_sampling &p) { return !(p.temperature > 0.0f) || p.top_k == 1; }

// 4 / (T ln 2).
__device__ __forceinline__ double steps_per_logit(float temperature) { return 5.770780163555853 / (double)temperature; }

// a * b, not fused into what it is added to.
__device__ __forceinline__ double rounded_product(double a, double b) {
#pragma clang fp contract(off)
    return a * b;
}

// A constant in scalar registers: as a literal it would be moved into the
// result of each multiply-add first.
__device__ __forceinline__ double held(double c) {
    asm("" : "+s"(c));
    return c;
}

// 2^(f / 4) for f in [0, 1), times `scale` and plus `add`: e^t about the middle
// of the range, t = (f - 1/2) ln(2) / 4 below 0.087 in magnitude, by its series
// to t^7 / 7! (the next term is below 9e-14, a unit of a step's sum 7e-12).
struct QuarterPower {
    double step, half, c7, c6, c5, c4, c3, c2, c1, add;

    __device__ __forceinline__ QuarterPower(double scale, double add_) {
        constexpr double kStep = 0.17328679513998633, kMiddle = 1.0905077326652577;  // ln(2) / 4, 2^(1/8)
        const double s = kMiddle * scale;
        step = held(kStep);
        half = held(-0.5 * kStep);
        c7 = held(s * (1.0 / 5040));
        c6 = held(s * (1.0 / 720));
        c5 = held(s * (1.0 / 120));
        c4 = held(s * (1.0 / 24));
        c3 = held(s * (1.0 / 6));
        c2 = held(s * 0.5);
        c1 = held(s);
        add = held(add_);
    }
    __device__ __forceinline__ double operator()(double f) const {
        const double t = fma(f, step, half);
        double e = fma(c7, t, c6);
        e = fma(e, t, c5);
        e = fma(e, t, c4);
        e = fma(e, t, c3);
        e = fma(e, t, c2);
        e = fma(e, t, c1);
        e = fma(e, t, c1);
        return e + add;
    }
};

// The same in whole units of 2^-kUnitBits: the sum with 2^52 rounds to them.
constexpr double kUnits = (double)(1ull << kUnitBits);
__device__ __forceinline__ double quarter_power(double f) { return (QuarterPower(kUnits, 0x1p52)(f) - 0x1p52) * (1.0 / kUnits); }

// Weights against a reference step (infinite where the largest logit is: then
// such logits weigh 1 and others nothing).
struct Weights {
    double c, reference;
    bool infinite;

    __device__ Weights(double c_, uint32_t top_key)
        : c(c_), reference(floor(rounded_product((double)key_logit(top_key), c_))), infinite(top_key == kKeyPlusInf) {}
    // A logit's step below the reference, at most kDead, and its weight
    // within the step.
    __device__ uint32_t bin(uint32_t key, double &within) const {
        within = 1.0;
        if (key <= kKeyMinusInf) return kDead;
        if (infinite) return key == kKeyPlusInf ? 0 : kDead;
        double f;
        const uint32_t b = finite_bin(key_logit(key), f);
        within = quarter_power(f);
        return b;
    }
    // A logit's step and place f within it, 2^(f / 4) the weight, where the
    // largest is finite. (NaN and -infinity come out at kDead by themselves.)
    __device__ __forceinline__ uint32_t finite_bin(float l, double &f) const {
        // (The product rounded first, as the reference's is: fused, the
        // largest finite logits would leave its rounding error.)
        const double y = rounded_product((double)l, c), step = floor(y);
        f = y - step;
        return (uint32_t)fmin(reference - step, (double)kDead);
    }
    __device__ uint32_t bin(uint32_t key) const {
        if (key <= kKeyMinusInf) return kDead;
        if (infinite) return key == kKeyPlusInf ? 0 : kDead;
        return (uint32_t)fmin(reference - floor(rounded_product((double)key_logit(key), c)), (double)kDead);
    }
    // The steps between a part's largest and this one's (kDead: none of the
    // part's tokens counts).
    __device__ uint32_t shift(uint32_t part_top) const {
        if (part_top <= kKeyMinusInf) return kDead;
        if (infinite) return part_top == kKeyPlusInf ? 0 : kDead;
        return bin(part_top);
    }
};

// A step's weight, 2^(-bin / 4).
__device__ __forceinline__ double step_weight(uint32_t bin) {
    const double odd = bin & 1 ? 0.8408964152537145 : 1.0, half = bin & 2 ? 0.7071067811865476 : 1.0;
    return ldexp(odd * half, -(int)(bin >> 2));
}

// What the first pass leaves of a part.
struct Part {
    uint64_t best;            // (key, ~index) of the largest
    uint32_t kept_bins, pad;  // `tokens` has all of the steps below kept_bins
    uint64_t sum[kBins];      // a step's count << kCountShift, and its sum in units
    uint16_t upto[kBins];     // tokens up to and with the step
    uint64_t tokens[kShort];  // (~key, index), by step
};

__device__ __forceinline__ uint64_t wave_largest(uint64_t v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const uint64_t o = __shfl_xor((unsigned long long)v, m, 64);
        v = o > v ? o : v;
    }
    return v;
}

__global__ __launch_bounds__(256) void sample_parts_kernel(const float *logits, uint32_t count, const qwh_sampling *params,
                                                           Part *parts) {
    __shared__ unsigned long long sums[kBins];
    __shared__ uint32_t place[kBins];
    __shared__ uint64_t wave_best[4];
    __shared__ uint32_t wave_sum[4], kept_bins;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *row = logits + (size_t)blockIdx.y * count;
    Part &part = parts[(size_t)blockIdx.y * gridDim.x + blockIdx.x];
    const uint32_t first = blockIdx.x * kPart, n = min(kPart, count - first);
    const qwh_sampling p = params[blockIdx.y];
    sums[tid] = 0;
    if (tid == 0) kept_bins = 0;
    // Sixteen logits a thread, four in a row: 16-byte loads where the row
    // allows them.
    float l[16];
    const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15u) == 0 && n == kPart;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t at = 1024 * k + 4 * tid;
        if (aligned) {
            const float4 v = *reinterpret_cast<const float4 *>(row + first + at);
            l[4 * k] = v.x;
            l[4 * k + 1] = v.y;
            l[4 * k + 2] = v.z;
            l[4 * k + 3] = v.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) l[4 * k + j] = at + j < n ? row[first + at + j] : -INFINITY;
        }
    }
    // The largest (NaN apart), then the lowest index that has it.
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, l[i]);
    uint32_t at_top = 15;
#pragma unroll
    for (int i = 15; i >= 0; --i)
        if (l[i] == top) at_top = i;
    uint64_t best = (uint64_t)logit_key(top) << 32 | (uint32_t) ~(first + 1024 * (at_top / 4) + 4 * tid + at_top % 4);
    best = wave_largest(best);
    if (lane == 0) wave_best[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) best = wave_best[w] > best ? wave_best[w] : best;
    const uint32_t top_key = (uint32_t)(best >> 32);
    if (tid == 0) part.best = best;
    if (is_greedy(p) || top_key <= kKeyMinusInf) return;  // (nothing else of it is read)
    const Weights w(steps_per_logit(p.temperature), top_key);
    uint8_t bin[16];
    if (w.infinite) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            bin[i] = l[i] == INFINITY ? 0 : (uint8_t)kDead;
            if (bin[i] == 0) atomicAdd(&sums[0], (unsigned long long)(1ull << kCountShift | 1ull << kUnitBits));
        }
    } else {
        // A weight as a whole number of units: the sum with 2^52 rounds to
        // one and holds it in its low bits. (Eight chains side by side, no
        // branch between them.)
        const QuarterPower units(kUnits, 0x1p52);
#pragma unroll
        for (int i0 = 0; i0 < 16; i0 += 8) {
            uint64_t add[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                double f;
                bin[i0 + i] = (uint8_t)w.finite_bin(l[i0 + i], f);
                // (2^52's own bits give way to the count of 1.)
                add[i] = __builtin_bit_cast(uint64_t, units(f)) - (0x433ull << 52) + (1ull << kCountShift);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (bin[i0 + i] < kDead) atomicAdd(&sums[bin[i0 + i]], (unsigned long long)add[i]);
        }
    }
    __syncthreads();
    // The steps whose tokens fit the short list.
    const uint64_t sum = sums[tid];
    uint32_t upto = (uint32_t)(sum >> kCountShift);
    const uint32_t own = upto;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(upto, d, 64);
        if (lane >= d) upto += o;
    }
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    for (int i = 0; i < wave; ++i) upto += wave_sum[i];
    part.sum[tid] = sum;
    part.upto[tid] = (uint16_t)upto;
    place[tid] = upto - own;
    const uint64_t fits = __ballot(upto <= kShort && tid < (int)kDead);
    if (lane == 0 && fits) atomicMax(&kept_bins, 64 * wave + (uint32_t)__popcll(fits));
    __syncthreads();
    const uint32_t below = kept_bins;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (bin[i] < below) {
            const uint32_t at = atomicAdd(&place[bin[i]], 1u);
            part.tokens[at] = (uint64_t)~logit_key(l[i]) << 32 | (first + 1024 * (i / 4) + 4 * tid + i % 4);
        }
    if (tid == 0) part.kept_bins = below;
}

struct RowShared {
    double mass[kBins];      // before each step; at kDead: all
    uint32_t count[kBins];
    uint64_t list[kList];
    uint64_t picked[kOrder], ordered[kOrder];
    double run[kOrder];      // running sums of the ordered tokens
    uint32_t split_n[kThreads];            // (of histograms: counts,
    unsigned long long split_m[kThreads];  // and sums)
    uint32_t raw[kThreads];
    uint16_t shift[kThreads], kept[kThreads];  // of the first parts
    double wave_m[16];
    uint32_t wave_n[16], wave_step[kBins / 64];
    uint64_t wave_best[16];
    uint32_t listed, raw_parts, found, found_index, edge[2], last_live;
    uint32_t found_count, counted, tie;
    double found_mass;
};

// Inclusive sums over the workgroup, in thread order.
__device__ __forceinline__ void block_scan(RowShared &sh, uint32_t &n, double &m) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t n2 = __shfl_up(n, d, 64);
        const double m2 = __shfl_up(m, d, 64);
        if (lane >= d) {
            n += n2;
            m += m2;
        }
    }
    __syncthreads();
    if (lane == 63) {
        sh.wave_n[wave] = n;
        sh.wave_m[wave] = m;
    }
    __syncthreads();
    uint32_t n0 = 0;
    double m0 = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64 - 1; ++w) {
        const uint32_t n2 = sh.wave_n[w];
        const double m2 = sh.wave_m[w];
        n0 += w < wave ? n2 : 0;
        m0 += w < wave ? m2 : 0.0;
    }
    n += n0;
    m += m0;
}

struct Row {
    const float *logits;
    uint32_t count, n_parts, top_key;
    const Part *parts;
    Weights w;
};

// The smallest key whose step is at most `bin`, by a whole wavefront: up to
// the row's largest, whose step is 0, steps never rise with the key, so 64
// keys at a time bracket it.
__device__ uint32_t first_key(const Weights &w, uint32_t top_key, uint32_t bin) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t low = 0, high = top_key;  // below low: not; from high on: yes
    while (high - low > 0) {
        const uint64_t step = (high - low + 63) / 64;
        const uint64_t key = low + lane * step;
        const bool yes = key >= high || w.bin((uint32_t)key) <= bin;
        const uint64_t all = __ballot(yes);
        const int at = all ? __builtin_ctzll(all) : 64;
        const uint64_t found = low + at * step;
        if (step == 1) return (uint32_t)(found < high ? found : high);
        high = found < high ? found : high;
        low = at ? low + (at - 1) * step + 1 : low;
    }
    return (uint32_t)low;
}

// The keys of steps lo .. hi: between edge[0] and edge[1], both included.
__device__ __forceinline__ void find_edges(RowShared &sh, const Row &row, uint32_t lo, uint32_t hi) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if (wave < 2) {
        const uint32_t edge = wave == 0  ? first_key(row.w, row.top_key, hi)
                              : lo == 0 ? row.top_key
                                        : first_key(row.w, row.top_key, lo - 1) - 1;
        if ((threadIdx.x & 63) == 0) sh.edge[wave] = edge;
    }
    __syncthreads();
}

// Calls f(key, index) for the row's tokens of steps lo .. hi (below kDead)
// with keys from low to high, each once (`whole`: whole steps; the keys are
// then found here where they are needed): eight lanes a part on its short
// list, where that has all of them, then a wavefront on each half of the
// others' logits.
template <typename F>
__device__ __forceinline__ void each_token(RowShared &sh, const Row &row, uint32_t lo, uint32_t hi, bool whole, uint32_t low,
                                           uint32_t high, F f) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr uint32_t kHalf = kPart / 2;
    const bool aligned = (reinterpret_cast<uintptr_t>(row.logits) & 15u) == 0;
    for (uint32_t base = 0; base < row.n_parts; base += kThreads) {
        const uint32_t held = min((uint32_t)kThreads, row.n_parts - base);
        __syncthreads();
        if (tid == 0) sh.raw_parts = 0;
        __syncthreads();
        for (uint32_t i = tid / 8; i < held; i += kThreads / 8) {
            const Part &part = row.parts[base + i];
            const uint32_t s = base ? row.w.shift((uint32_t)(part.best >> 32)) : sh.shift[i];
            if (s > hi) continue;
            const uint32_t kept = base ? part.kept_bins : sh.kept[i];
            const uint32_t begin = lo > s ? part.upto[lo - s - 1] : 0, end = part.upto[hi - s];
            if (begin >= end) continue;
            if (hi - s < kept) {
                for (uint32_t k = begin + tid % 8; k < end; k += 8) {
                    const uint64_t token = part.tokens[k];
                    const uint32_t key = (uint32_t)(~token >> 32);
                    if (whole || (key >= low && key <= high)) f(key, (uint32_t)token);
                }
            } else if (tid % 8 == 0) {
                sh.raw[atomicAdd(&sh.raw_parts, 1u)] = base + i;
            }
        }
        __syncthreads();
        const uint32_t halves = 2 * sh.raw_parts;
        if (whole && halves) {
            find_edges(sh, row, lo, hi);
            whole = false;
            low = sh.edge[0];
            high = sh.edge[1];
        }
        for (uint32_t r = wave; r < halves; r += kThreads / 64) {
            const uint32_t begin = sh.raw[r / 2] * kPart + r % 2 * kHalf;
            if (begin >= row.count) continue;
            const uint32_t n = min(kHalf, row.count - begin);
            const float *from = row.logits + begin;
            if (aligned && n == kHalf) {
                float4 l[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) l[j] = *reinterpret_cast<const float4 *>(from + 256 * j + 4 * lane);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float four[4] = {l[j].x, l[j].y, l[j].z, l[j].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t key = logit_key(four[i]);
                        if (key >= low && key <= high) f(key, begin + 256 * j + 4 * lane + i);
                    }
                }
            } else {
                for (uint32_t k = lane; k < n; k += 256) {
                    float l[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) l[j] = from[min(k + 64 * j, n - 1)];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t key = logit_key(l[j]);
                        if (k + 64 * j < n && key >= low && key <= high) f(key, begin + k + 64 * j);
                    }
                }
            }
        }
    }
    __syncthreads();
}

// Takes the tokens of steps lo .. hi (not `whole`: of them, with keys from low
// to high) into the list.
__device__ __noinline__ void collect(RowShared &sh, const Row &row, uint32_t lo, uint32_t hi, bool whole, uint32_t low,
                                     uint32_t high) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    each_token(sh, row, lo, hi, whole, low, high, [&](uint32_t key, uint32_t i) {
        const uint32_t at = atomicAdd(&sh.listed, 1u);
        if (at < kList) sh.list[at] = (uint64_t)~key << 32 | i;
    });
}

// The list's n tokens (at most kOrder) with keys from low to high in order in
// sh.ordered, sh.run their running sums on top of `before`.
__device__ __noinline__ void order_listed(RowShared &sh, const Row &row, uint32_t low, uint32_t high, uint32_t n, double before) {
    const uint32_t tid = threadIdx.x;
    __syncthreads();
    const uint32_t all = min(sh.listed, kList);
    const uint64_t *tokens = sh.list;
    if (all > n) {
        tokens = sh.picked;
        if (tid == 0) sh.counted = 0;
        __syncthreads();
        for (uint32_t i = tid; i < all; i += kThreads) {
            const uint64_t token = sh.list[i];
            const uint32_t key = (uint32_t)(~token >> 32);
            if (key >= low && key <= high) {
                const uint32_t at = atomicAdd(&sh.counted, 1u);
                if (at < kOrder) sh.picked[at] = token;
            }
        }
        __syncthreads();
    }
    // A token's place is the number of smaller ones (all differ).
    if (tid < n) {
        const uint64_t own = tokens[tid];
        uint32_t rank = 0;
#pragma unroll 8
        for (uint32_t k = 0; k < n; ++k) rank += tokens[k] < own;
        sh.ordered[rank] = own;
    }
    __syncthreads();
    double run = 0.0, within;
    if (tid < n) {
        const uint32_t bin = row.w.bin((uint32_t)(~sh.ordered[tid] >> 32), within);
        run = step_weight(bin) * within;
    }
    uint32_t none = 0;
    block_scan(sh, none, run);
    if (tid < n) sh.run[tid] = before + run;
    __syncthreads();
}

// The first entry of the ordered list (of n) whose running sum reaches
// (`past`: exceeds) `at`; the last if none does.
__device__ uint32_t reach(RowShared &sh, uint32_t n, double at, bool past) {
    __syncthreads();
    if (threadIdx.x == 0) sh.found = n - 1;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const bool here = past ? sh.run[i] > at : sh.run[i] >= at;
        const bool before = i > 0 && (past ? sh.run[i - 1] > at : sh.run[i - 1] >= at);
        if (here && !before) atomicMin(&sh.found, i);
    }
    __syncthreads();
    return sh.found;
}

// The step in which the count (`by_mass`: the sum) reaches `at` (past:
// exceeds it): the first with tokens of which that holds (may_hold), the last
// step with tokens if none does.
__device__ uint32_t step_of(RowShared &sh, bool by_mass, double at, bool past) {
    const uint32_t b = threadIdx.x;
    bool here = false;
    if (b < kDead) {
        const double upto = by_mass ? sh.mass[b + 1] : (double)sh.count[b + 1];
        here = sample::may_hold(sh.count[b], sh.count[b + 1], upto, at, past);
    }
    const uint64_t all = __ballot(here);
    __syncthreads();
    if (b < kBins && b % 64 == 0) sh.wave_step[b / 64] = all ? b + (uint32_t)__builtin_ctzll(all) : kDead;
    __syncthreads();
    uint32_t first = sh.last_live;
#pragma unroll
    for (uint32_t w = 0; w < kBins / 64; ++w) first = min(first, sh.wave_step[w]);
    return first;
}

// A place in step `bin`: the entry where the count (by_mass: sum) reaches
// `at` (past: exceeds it). found_index, and count and sum up to it. `listed`:
// the list has the step's tokens (and perhaps others).
__device__ __noinline__ void place_in(RowShared &sh, const Row &row, uint32_t bin, bool by_mass, double at, bool past,
                                      bool listed) {
    const uint32_t tid = threadIdx.x;
    uint32_t nb = sh.count[bin], n = sh.count[bin + 1] - nb;
    double mb = sh.mass[bin];
    // (Few tokens that the list does not have are all that it then has.)
    uint32_t low = 0, high = row.top_key;
    const bool whole = !listed && n <= kOrder;
    if (!whole) {
        find_edges(sh, row, bin, bin);
        low = sh.edge[0];
        high = sh.edge[1];
    }
    // The range of keys split into up to 1024 equal ones, and the one that
    // has the place again, until it has few tokens or one key. (Sums in units:
    // 2^26 weights of up to 2^(1/4) fit 64 bits.)
    const double unit = step_weight(bin) * (1.0 / kUnits);
    while (true) {
        if (!listed && n <= kList) {
            collect(sh, row, bin, bin, whole, low, high);
            listed = true;
        }
        if (n <= kOrder || low >= high) break;
        const uint32_t width = 32 - __builtin_clz(high - low), shift = width > 10 ? width - 10 : 0;
        __syncthreads();
        sh.split_n[tid] = 0;
        sh.split_m[tid] = 0;
        __syncthreads();
        const auto add = [&](uint32_t key, uint32_t) {
            const uint32_t d = (high - key) >> shift;
            double within;
            (void)row.w.bin(key, within);
            atomicAdd(&sh.split_n[d], 1u);
            atomicAdd(&sh.split_m[d], (unsigned long long)(within * kUnits));
        };
        if (listed) {
            const uint32_t all = min(sh.listed, kList);
            for (uint32_t i = tid; i < all; i += kThreads) {
                const uint64_t token = sh.list[i];
                const uint32_t key = (uint32_t)(~token >> 32);
                if (key >= low && key <= high) add(key, (uint32_t)token);
            }
            __syncthreads();
        } else {
            each_token(sh, row, bin, bin, false, low, high, add);
        }
        const uint32_t mine = sh.split_n[tid];
        const double mass = (double)sh.split_m[tid] * unit;
        uint32_t run_n = mine;
        double run_m = mass;
        block_scan(sh, run_n, run_m);
        if (tid == 0) sh.found = kThreads;
        __syncthreads();
        const double v = by_mass ? mb + run_m : (double)nb + run_n;
        if (mine && (past ? v > at : v >= at)) atomicMin(&sh.found, tid);
        __syncthreads();
        if (sh.found == kThreads) {  // (uniform; the sums' last bits)
            __syncthreads();
            if (tid == 0) sh.found = 0;
            __syncthreads();
            if (mine) atomicMax(&sh.found, tid);
            __syncthreads();
        }
        const uint32_t d = sh.found;
        if (tid == d) {
            sh.found_count = run_n - mine;
            sh.found_mass = run_m - mass;
        }
        __syncthreads();
        high -= d << shift;
        low = max(low, high - min(high, (1u << shift) - 1));
        n = sh.split_n[d];
        nb += sh.found_count;
        mb += sh.found_mass;
    }
    if (n <= kOrder) {
        order_listed(sh, row, low, high, n, mb);
        const uint32_t k = by_mass ? reach(sh, n, at, past) : (uint32_t)fmin(fmax(at - nb, 1.0), (double)n) - 1;
        __syncthreads();
        if (tid == 0) {
            sh.found_index = (uint32_t)sh.ordered[k];
            sh.found_count = nb + k + 1;
            sh.found_mass = sh.run[k];
        }
        __syncthreads();
        return;
    }
    // Tokens of one logit, in index order, all of one weight: which of them.
    double w;
    (void)row.w.bin(low, w);
    w *= step_weight(bin);
    double nth = by_mass ? (past ? floor((at - mb) / w) + 1.0 : ceil((at - mb) / w)) : at - nb;
    nth = fmin(fmax(nth, 1.0), (double)n);
    const uint32_t which = (uint32_t)nth;
    uint32_t seen = 0;  // of them before this stretch
    for (uint32_t base = 0; base < row.count; base += kThreads) {
        const uint32_t i = base + tid;
        uint32_t run = i < row.count && logit_key(row.logits[i]) == low ? 1u : 0u;
        const uint32_t own = run;
        double none = 0.0;
        block_scan(sh, run, none);
        if (own && seen + run == which) sh.found_index = i;
        if (tid == kThreads - 1u) sh.tie = run;
        __syncthreads();
        seen += sh.tie;
        __syncthreads();
        if (seen >= which) break;
    }
    if (tid == 0) {
        sh.found_count = (uint32_t)(nb + which);
        sh.found_mass = mb + which * w;
    }
    __syncthreads();
}

__global__ __launch_bounds__(kThreads) void sample_rows_kernel(const float *logits, uint32_t count, uint32_t n_parts,
                                                               const qwh_sampling *params, const float *uniform,
                                                               const Part *all_parts, uint32_t *ids) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_row[];
    RowShared &sh = *reinterpret_cast<RowShared *>(lds_row);
    const int tid = threadIdx.x;
    const qwh_sampling p = params[blockIdx.x];
    const Part *parts = all_parts + (size_t)blockIdx.x * n_parts;
    // The largest logit, the lowest index among equal ones.
    uint64_t best = 0;
    for (uint32_t i = tid; i < n_parts; i += kThreads) best = parts[i].best > best ? parts[i].best : best;
    best = wave_largest(best);
    if ((tid & 63) == 0) sh.wave_best[tid >> 6] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) best = sh.wave_best[w] > best ? sh.wave_best[w] : best;
    const uint32_t top_key = (uint32_t)(best >> 32);
    if (is_greedy(p) || top_key <= kKeyMinusInf) {
        if (tid == 0) ids[blockIdx.x] = top_key <= kKeyMinusInf ? 0u : ~(uint32_t)best;
        return;
    }
    const Row row{logits + (size_t)blockIdx.x * count, count, n_parts, top_key, parts,
                  Weights(steps_per_logit(p.temperature), top_key)};
    // The parts' histograms, each shifted by its own largest step: four
    // threads a step, every fourth part each. Parts' sums share the grid of
    // steps, so they are added as integers.
    {
        const uint32_t b = tid & (kBins - 1), group = tid / kBins;
        uint32_t n = 0;
        uint64_t m = 0;
        for (uint32_t base = 0; base < n_parts; base += kThreads) {
            __syncthreads();
            if (base + tid < n_parts) {
                const Part &part = parts[base + tid];
                const uint32_t kept = part.kept_bins, s = row.w.shift((uint32_t)(part.best >> 32));
                sh.raw[tid] = s;
                if (base == 0) {
                    sh.shift[tid] = (uint16_t)s;
                    sh.kept[tid] = (uint16_t)kept;
                }
            }
            __syncthreads();
            const uint32_t held = min((uint32_t)kThreads, n_parts - base);
            for (uint32_t i0 = group; i0 < held; i0 += 8 * (kThreads / kBins)) {
                uint64_t read[8];
                uint32_t s[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t i = i0 + k * (kThreads / kBins);
                    s[k] = i < held ? sh.raw[i] : kDead;
                    read[k] = parts[base + min(i, held - 1)].sum[b >= s[k] ? b - s[k] : 0];
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    // (A part all of whose tokens are dead has written no sums.)
                    const uint64_t sum = s[k] > b || b >= kDead ? 0 : read[k];
                    n += (uint32_t)(sum >> kCountShift);
                    m += sum & ((1ull << kCountShift) - 1);
                }
            }
        }
        sh.split_n[tid] = n;
        sh.split_m[tid] = m;
        __syncthreads();
        uint32_t run_n = 0;
        double run_m = 0.0;
        if (group == 0) {
            for (uint32_t g = 1; g < kThreads / kBins; ++g) {
                n += sh.split_n[g * kBins + b];
                m += sh.split_m[g * kBins + b];
            }
            run_n = n;
            run_m = (double)m * (step_weight(b) * (1.0 / kUnits));
        }
        block_scan(sh, run_n, run_m);
        if (group == 0) {
            // Before the step; the next step's is this one's end, exactly.
            if (b + 1 < kBins) {
                sh.count[b + 1] = run_n;
                sh.mass[b + 1] = run_m;
            }
            if (b == 0) {
                sh.count[0] = 0;
                sh.mass[0] = 0.0;
            }
        }
        __syncthreads();
        if (tid < (int)kDead && sh.count[tid + 1] == sh.count[kDead] && sh.count[tid] != sh.count[kDead]) sh.last_live = tid;
        __syncthreads();
    }
    const uint32_t live = sh.count[kDead];
    const bool by_k = p.top_k > 0 && p.top_k < live, by_p = p.top_p < 1.0f;
    const double least = p.min_p > 0.0f ? (double)fminf(p.min_p, 1.0f) : 0.0;
    const double top = (double)key_logit(top_key), heat = (double)p.temperature;
    const auto enough = [&](uint32_t key) {
        return row.w.infinite || exp(((double)key_logit(key) - top) / heat) >= least;
    };
    const float u = uniform[blockIdx.x];
    const double draw = u > 0.0f ? fmin((double)u, 1.0) : 0.0;
    // The last step that any rule can keep a token of.
    uint32_t last = sh.last_live;
    if (by_k) last = min(last, step_of(sh, false, (double)p.top_k, false));
    else if (by_p) last = min(last, step_of(sh, true, (double)p.top_p * kReach * sh.mass[kDead], false));
    else if (least > 0.0 && !row.w.infinite) last = min(last, (uint32_t)fmin(row.w.reference - floor(top * row.w.c + 4.0 * log2(least)) + 1.0, (double)(kDead - 1)));
    // All that may be kept, if it fits the list.
    const uint32_t n = sh.count[last + 1];
    const bool listed = (by_k || by_p || least > 0.0) && n <= kList;
    if (listed) {
        collect(sh, row, 0, last, true, 0, 0);
    }
    if (listed && n <= kOrder) {
        // The rules one after another on its running sums.
        order_listed(sh, row, 0, row.top_key, n, 0.0);
        uint32_t tokens = by_k ? min(p.top_k, n) : n;
        if (by_p) {
            const double whole = by_k ? sh.run[tokens - 1] : sh.mass[kDead];
            tokens = min(tokens, reach(sh, tokens, (double)p.top_p * kReach * whole, false) + 1);
        }
        if (least > 0.0) {
            __syncthreads();
            if (tid == 0) sh.counted = 0;
            __syncthreads();
            uint32_t mine = 0;
            for (uint32_t i = tid; i < tokens; i += kThreads) mine += enough((uint32_t)(~sh.ordered[i] >> 32));
            if (mine) atomicAdd(&sh.counted, mine);
            __syncthreads();
            tokens = max(sh.counted, 1u);
        }
        const double kept = sh.run[tokens - 1];
        const uint32_t k = draw >= 1.0 ? tokens - 1 : reach(sh, tokens, draw * kPast * kept, true);
        __syncthreads();
        if (tid == 0) ids[blockIdx.x] = (uint32_t)sh.ordered[min(k, tokens - 1)];
        return;
    }
    // Otherwise each place by itself.
    double kept = sh.mass[kDead];
    uint32_t tokens = live;
    if (by_k) {
        place_in(sh, row, step_of(sh, false, (double)p.top_k, false), false, (double)p.top_k, false, listed);
        tokens = sh.found_count;
        kept = sh.found_mass;
    }
    if (by_p) {
        const double at = (double)p.top_p * kReach * kept;
        place_in(sh, row, step_of(sh, true, at, false), true, at, false, listed);
        tokens = sh.found_count;
        kept = sh.found_mass;
    }
    if (least > 0.0 && !row.w.infinite) {
        // Tokens of at least min_p: all of the steps above its own and the
        // one before that, and those of the next three that are.
        const double at = row.w.reference - floor(top * row.w.c + 4.0 * log2(least)) - 1.0;
        const uint32_t lo = (uint32_t)fmin(fmax(at, 0.0), (double)(kDead - 1)), hi = min(lo + 2, kDead - 1);
        __syncthreads();
        if (tid == 0) sh.counted = 0;
        __syncthreads();
        each_token(sh, row, lo, hi, true, 0, 0, [&](uint32_t key, uint32_t) {
            if (enough(key)) atomicAdd(&sh.counted, 1u);
        });
        const uint32_t reaching = max(sh.count[lo] + sh.counted, 1u);
        if (reaching < tokens) {
            tokens = reaching;
            place_in(sh, row, step_of(sh, false, (double)tokens, false), false, (double)tokens, false, listed);
            kept = sh.found_mass;
        }
    }
    if (draw >= 1.0) place_in(sh, row, step_of(sh, false, (double)tokens, false), false, (double)tokens, false, listed);
    else {
        const double at = draw * kPast * kept;
        place_in(sh, row, step_of(sh, true, at, true), true, at, true, listed);
    }
    if (tid == 0) ids[blockIdx.x] = sh.found_index;
}

uint32_t parts_of(uint32_t count) { return (count + kPart - 1) / kPart; }
uint32_t rows_at_once(uint32_t rows, uint32_t count) {
    const uint32_t most = kPartsAtOnce / parts_of(count);
    return most < 1 ? 1 : rows < most ? rows : most;
}

}  // namespace

size_t sample_scratch_bytes(uint32_t rows, uint32_t count) {
    return (size_t)rows_at_once(rows, count) * parts_of(count) * sizeof(Part);
}

hipError_t launch_sample_rows(hipStream_t s, const float *logits, uint32_t rows, uint32_t count, const qwh_sampling *params,
                              const float *uniform, void *scratch, uint32_t *ids) {
    const uint32_t n_parts = parts_of(count), at_once = rows_at_once(rows, count);
    Part *parts = static_cast<Part *>(scratch);
    const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void *>(sample_rows_kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(RowShared));
    if (err != hipSuccess) return err;
    for (uint32_t r = 0; r < rows; r += at_once) {
        const uint32_t n = rows - r < at_once ? rows - r : at_once;
        const float *from = logits + (size_t)r * count;
        sample_parts_kernel<<<dim3(n_parts, n), 256, 0, s>>>(from, count, params + r, parts);
        sample_rows_kernel<<<n, kThreads, sizeof(RowShared), s>>>(from, count, n_parts, params + r, uniform + r, parts, ids + r);
    }
    return hipGetLastError();
}

}  // namespace qwh
