// Drawing tokens from logits by temperature, top-k, top-p and min-p
// (qwh_sample_rows).
//
// Everything a draw asks for is a place in one order of the row, the largest
// logit first and the lower index first among equal ones: the sum of the
// first k weights (top-k), where the running sum reaches top_p times that
// (top-p), how many weights are at least min_p of the largest, and where the
// running sum passes u times what is left. The row is never sorted: a
// histogram over 2047 steps of the logit below the largest (count and sum of
// weights a step) says in which step such a place lies, and only that step's
// tokens are put in order.
//
// Weights are exp in 64 bits, rounded to whole multiples of 2^-s of the
// largest (s = 62 less the bits of the row's length, so that a row's sum
// fits 64 bits): integer sums are the same in any order, so histograms may be
// filled with atomics and still every run draws the same token, and with 44
// bits at a vocabulary of 151936 a draw differs from one in real numbers only
// where u falls within about 1e-13 of a border.
#include <cfloat>

#include "common.h"
#include "device.h"

namespace qwh {
namespace {

constexpr int kThreads = 1024;
constexpr uint32_t kBins = 2048;          // the last: tokens without a weight
constexpr uint32_t kList = 4096;          // tokens of a step that are put in order in LDS

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

// What turns a row's logits into weights.
struct RowWeights {
    double top, heat;    // the largest logit, the temperature
    double bins_per_nat;
    int shift;           // s
    bool infinite;       // the largest is +infinity

    __device__ double below(uint32_t key) const { return (top - (double)key_logit(key)) / heat; }
    // exp(-below), of the row's largest.
    __device__ double weight(uint32_t key) const {
        if (key <= kKeyMinusInf) return 0.0;
        if (infinite) return key == kKeyPlusInf ? 1.0 : 0.0;
        return exp(-below(key));
    }
    __device__ uint64_t fixed(double w) const { return (uint64_t)rint(ldexp(w, shift)); }
    // The step of a key: never falls as the logit falls. Past 2^-(s + 1) of
    // the largest there is no weight left.
    __device__ uint32_t bin(uint32_t key) const {
        if (key <= kKeyMinusInf) return kBins - 1;
        if (infinite) return key == kKeyPlusInf ? 0u : kBins - 1;
        return (uint32_t)fmin(below(key) * bins_per_nat, (double)(kBins - 1));
    }
};

__device__ __forceinline__ RowWeights row_weights(uint32_t top_key, float temperature, uint32_t count) {
    RowWeights r;
    r.top = (double)key_logit(top_key);
    r.heat = (double)temperature;
    r.infinite = top_key == kKeyPlusInf;
    r.shift = 62 - (32 - __builtin_clz(count));
    r.bins_per_nat = (double)(kBins - 1) / ((r.shift + 1) * 0.69314718055994530942);
    return r;
}

// Calls f(key, index) for the row's elements, some of them by each thread.
template <typename F>
__device__ __forceinline__ void each_logit(const float *row, uint32_t count, F f) {
    if ((reinterpret_cast<uintptr_t>(row) & 15u) == 0) {
        const uint32_t quads = count / 4;
        for (uint32_t i = threadIdx.x; i < quads; i += kThreads) {
            const float4 v = reinterpret_cast<const float4 *>(row)[i];
            f(logit_key(v.x), 4 * i);
            f(logit_key(v.y), 4 * i + 1);
            f(logit_key(v.z), 4 * i + 2);
            f(logit_key(v.w), 4 * i + 3);
        }
        const uint32_t i = 4 * quads + threadIdx.x;
        if (i < count) f(logit_key(row[i]), i);
        return;
    }
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) f(logit_key(row[i]), i);
}

struct SampleShared {
    uint32_t count[kBins];   // per step; then before the step
    uint64_t mass[kBins];
    uint64_t list[kList];    // (~key, index): ascending is the row's order
    uint64_t wave[16];
    uint32_t wave_n[16];
    uint64_t best;
    uint32_t listed, at_least, found_bin, found_index, tie_index;
    uint32_t found_count;
    uint64_t found_mass, total;
    uint32_t live;
    uint32_t digits[256];
    uint64_t digit_mass[256];
};

// Inclusive sums over the workgroup, in thread order.
__device__ __forceinline__ void block_scan(SampleShared &sh, uint32_t &n, uint64_t &m) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t n2 = __shfl_up(n, d, 64);
        const uint64_t m2 = __shfl_up((unsigned long long)m, d, 64);
        if (lane >= d) {
            n += n2;
            m += m2;
        }
    }
    __syncthreads();
    if (lane == 63) {
        sh.wave_n[wave] = n;
        sh.wave[wave] = m;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        n += sh.wave_n[w];
        m += sh.wave[w];
    }
}

// Where a place is asked for: the first token of the order at which the
// running count, or the running sum, reaches `at` (at least 1).
struct Place {
    bool by_mass;
    uint64_t at;
    __device__ bool reached(uint32_t n, uint64_t m) const { return (by_mass ? m : n) >= at; }
};

// The place in the row: found_index the token there, found_count and
// found_mass the running count and sum with it. It lies in some step (the
// caller asks for no place behind the last token with a weight).
__device__ void find_place(SampleShared &sh, const float *row, uint32_t count, const RowWeights &rw, const Place &p) {
    const int tid = threadIdx.x;
    __syncthreads();
    // sh.count / sh.mass hold what lies before each step (and at [kBins - 1]
    // the totals).
    for (uint32_t b = tid; b + 1 < kBins; b += kThreads)
        if (!p.reached(sh.count[b], sh.mass[b]) && p.reached(sh.count[b + 1], sh.mass[b + 1])) sh.found_bin = b;
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    const uint32_t bin = sh.found_bin;
    const uint32_t n0 = sh.count[bin], n = sh.count[bin + 1] - n0;
    const uint64_t m0 = sh.mass[bin];
    if (n <= kList) {
        each_logit(row, count, [&](uint32_t key, uint32_t i) {
            if (rw.bin(key) == bin) sh.list[atomicAdd(&sh.listed, 1u)] = (uint64_t)~key << 32 | i;
        });
        uint32_t padded = 2;
        while (padded < n) padded *= 2;
        for (uint32_t i = n + tid; i < padded; i += kThreads) sh.list[i] = ~0ull;
        for (uint32_t size = 2; size <= padded; size *= 2) {
            for (uint32_t step = size / 2; step >= 1; step /= 2) {
                __syncthreads();
                for (uint32_t k = tid; k < padded / 2; k += kThreads) {
                    const uint32_t i = 2 * k - (k & (step - 1)), j = i + step;
                    const uint64_t x = sh.list[i], y = sh.list[j];
                    if ((x > y) == ((i & size) == 0)) {
                        sh.list[i] = y;
                        sh.list[j] = x;
                    }
                }
            }
        }
        __syncthreads();
        // Running sums over the ordered list, four tokens a thread.
        uint32_t mine = 0;
        uint64_t w[4], sum = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t i = 4 * tid + k;
            w[k] = 0;
            if (i < n) {
                w[k] = rw.fixed(rw.weight((uint32_t)(~sh.list[i] >> 32)));
                ++mine;
                sum += w[k];
            }
        }
        uint32_t run_n = mine;
        uint64_t run_m = sum;
        block_scan(sh, run_n, run_m);
        run_n += n0 - mine;
        run_m += m0 - sum;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t i = 4 * tid + k;
            if (i >= n) break;
            const bool before = p.reached(run_n, run_m);
            ++run_n;
            run_m += w[k];
            if (!before && p.reached(run_n, run_m)) {
                sh.found_index = (uint32_t)sh.list[i];
                sh.found_count = run_n;
                sh.found_mass = run_m;
            }
        }
        __syncthreads();
        return;
    }
    // More tokens than the list holds: the key at the place digit by digit,
    // each pass a histogram of the step's tokens that share the digits so far.
    uint32_t prefix = 0, nb = n0;
    uint64_t mb = m0;
    for (int digit = 3; digit >= 0; --digit) {
        for (int i = tid; i < 256; i += kThreads) {
            sh.digits[i] = 0;
            sh.digit_mass[i] = 0;
        }
        __syncthreads();
        each_logit(row, count, [&](uint32_t key, uint32_t) {
            if (rw.bin(key) != bin || (digit < 3 && (key >> (8 * digit + 8)) != prefix)) return;
            const uint32_t d = 255u - ((key >> (8 * digit)) & 255u);
            atomicAdd(&sh.digits[d], 1u);
            atomicAdd(reinterpret_cast<unsigned long long *>(&sh.digit_mass[d]), (unsigned long long)rw.fixed(rw.weight(key)));
        });
        __syncthreads();
        const uint32_t mine = tid < 256 ? sh.digits[tid] : 0;
        const uint64_t mass = tid < 256 ? sh.digit_mass[tid] : 0;
        uint32_t run_n = mine;
        uint64_t run_m = mass;
        block_scan(sh, run_n, run_m);
        if (!p.reached(nb + run_n - mine, mb + run_m - mass) && p.reached(nb + run_n, mb + run_m)) {
            sh.found_bin = 255u - tid;
            sh.found_count = nb + run_n - mine;
            sh.found_mass = mb + run_m - mass;
        }
        __syncthreads();
        prefix = prefix << 8 | sh.found_bin;
        nb = sh.found_count;
        mb = sh.found_mass;
        __syncthreads();
    }
    // Tokens of one logit, in index order, all of one weight: which of them.
    const uint64_t w = rw.fixed(rw.weight(prefix));
    uint32_t low = 1, high = count;  // the place's number among them
    while (low < high) {
        const uint32_t mid = low + (high - low) / 2;
        if (p.reached(nb + mid, mb + mid * w)) high = mid;
        else low = mid + 1;
    }
    uint32_t seen = 0;  // of them before this stretch
    for (uint32_t base = 0; base < count; base += kThreads) {
        const uint32_t i = base + tid;
        uint32_t run = i < count && logit_key(row[i]) == prefix ? 1u : 0u;
        const uint32_t own = run;
        uint64_t none = 0;
        block_scan(sh, run, none);
        if (own && seen + run == low) sh.found_index = i;
        if (tid == kThreads - 1) sh.tie_index = run;
        __syncthreads();
        seen += sh.tie_index;
        __syncthreads();
        if (seen >= low) break;
    }
    if (tid == 0) {
        sh.found_count = nb + low;
        sh.found_mass = mb + low * w;
    }
    __syncthreads();
}

__global__ __launch_bounds__(kThreads) void sample_rows_kernel(const float *logits, uint32_t count, const qwh_sampling *params,
                                                               const float *uniform, uint32_t *ids) {
    __shared__ SampleShared sh;
    const int tid = threadIdx.x;
    const float *row = logits + (size_t)blockIdx.x * count;
    const qwh_sampling p = params[blockIdx.x];
    // The largest logit, the lowest index among equal ones.
    uint64_t best = 0;
    each_logit(row, count, [&](uint32_t key, uint32_t i) {
        const uint64_t v = (uint64_t)key << 32 | (uint32_t)~i;
        best = v > best ? v : best;
    });
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const uint64_t o = __shfl_xor((unsigned long long)best, m, 64);
        best = o > best ? o : best;
    }
    if ((tid & 63) == 0) sh.wave[tid >> 6] = best;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) best = sh.wave[w] > best ? sh.wave[w] : best;
    __syncthreads();
    const uint32_t top_key = (uint32_t)(best >> 32);
    if (!(p.temperature > 0.0f) || top_key <= kKeyMinusInf || p.top_k == 1) {
        if (tid == 0) ids[blockIdx.x] = top_key <= kKeyMinusInf ? 0u : ~(uint32_t)best;
        return;
    }
    const RowWeights rw = row_weights(top_key, p.temperature, count);
    const double least = p.min_p > 0.0f ? (double)fminf(p.min_p, 1.0f) : 0.0;
    for (uint32_t b = tid; b < kBins; b += kThreads) {
        sh.count[b] = 0;
        sh.mass[b] = 0;
    }
    if (tid == 0) sh.at_least = 0;
    __syncthreads();
    uint32_t mine = 0;
    each_logit(row, count, [&](uint32_t key, uint32_t) {
        const uint32_t b = rw.bin(key);
        if (b == kBins - 1) return;
        const double w = rw.weight(key);
        atomicAdd(&sh.count[b], 1u);
        atomicAdd(reinterpret_cast<unsigned long long *>(&sh.mass[b]), (unsigned long long)rw.fixed(w));
        mine += w >= least;
    });
    if (mine) atomicAdd(&sh.at_least, mine);
    __syncthreads();
    {
        // Sums before each step.
        const uint32_t n0 = sh.count[2 * tid], n1 = sh.count[2 * tid + 1];
        const uint64_t m0 = sh.mass[2 * tid], m1 = sh.mass[2 * tid + 1];
        uint32_t n = n0 + n1;
        uint64_t m = m0 + m1;
        block_scan(sh, n, m);
        sh.count[2 * tid] = n - n0 - n1;
        sh.mass[2 * tid] = m - m0 - m1;
        sh.count[2 * tid + 1] = n - n1;
        sh.mass[2 * tid + 1] = m - m1;
    }
    __syncthreads();
    const uint32_t live = sh.count[kBins - 1];
    uint64_t kept = sh.mass[kBins - 1];  // the sum of the first `tokens`
    uint32_t tokens = live;
    if (p.top_k > 0 && p.top_k < live) {
        find_place(sh, row, count, rw, Place{false, p.top_k});
        tokens = sh.found_count;
        kept = sh.found_mass;
    }
    if (p.top_p < 1.0f) {
        // A token is kept while the sum before it is below top_p * kept: the
        // last one is where the sum reaches it.
        const double reach = fmax((double)p.top_p * (double)kept, 1.0);
        find_place(sh, row, count, rw, Place{true, (uint64_t)ceil(reach)});
        tokens = sh.found_count;
        kept = sh.found_mass;
    }
    const uint32_t least_tokens = least > 0.0 ? (sh.at_least > 1 ? sh.at_least : 1u) : tokens;
    if (least_tokens < tokens) {
        find_place(sh, row, count, rw, Place{false, least_tokens});
        kept = sh.found_mass;
    }
    const float u = uniform[blockIdx.x];
    // The first token past u * kept; from u = 1 on the last one with a weight.
    const double target = (u > 0.0f ? fmin((double)u, 1.0) : 0.0) * (double)kept;
    const uint64_t past = (uint64_t)target;
    find_place(sh, row, count, rw, Place{true, past < kept ? past + 1 : kept});
    if (tid == 0) ids[blockIdx.x] = sh.found_index;
}

}  // namespace

size_t sample_scratch_bytes(uint32_t, uint32_t) { return 256; }

hipError_t launch_sample_rows(hipStream_t s, const float *logits, uint32_t rows, uint32_t count, const qwh_sampling *params,
                              const float *uniform, void *, uint32_t *ids) {
    sample_rows_kernel<<<rows, kThreads, 0, s>>>(logits, count, params, uniform, ids);
    return hipGetLastError();
}

}  // namespace qwh
