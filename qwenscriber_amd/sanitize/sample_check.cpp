// CPU check of the step in which sampling looks for a place (sample_plan.h),
// built with g++ and its sanitizers: over running sums added in the order in
// which sample.hip's workgroup adds them, the step for every sum and the
// numbers next to it has tokens, reaches what is asked for, and has none
// before it that does by more than the sums' last bits. Exit status 0 when
// every case holds.
#include <cmath>
#include <cstdio>
#include <random>
#include <vector>

#include "../csrc/sample_plan.h"

namespace {

constexpr uint32_t kBins = 256, kDead = kBins - 1;
long cases = 0, failures = 0, falls = 0, rises = 0;

void expect(bool ok, const char *what, long a = 0, long b = 0) {
    ++cases;
    if (ok) return;
    if (++failures <= 20) std::printf("FAIL %s (%ld, %ld)\n", what, a, b);
}

// block_scan's sums of its first four wavefronts: within one by doubling
// distances, then the wavefronts before it one after another.
std::vector<double> scan(const std::vector<double> &x) {
    std::vector<double> m = x;
    for (uint32_t w = 0; w < kBins; w += 64)
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const std::vector<double> old = m;
            for (uint32_t l = d; l < 64; ++l) m[w + l] = old[w + l] + old[w + l - d];
        }
    std::vector<double> out(kBins);
    for (uint32_t b = 0; b < kBins; ++b) {
        double before = 0.0;
        for (uint32_t w = 0; w < b / 64; ++w) before += m[64 * w + 63];
        out[b] = m[b] + before;
    }
    return out;
}

void histogram(std::mt19937_64 &rng) {
    // A row's steps: a bulk of tokens far down, few above it, some steps of
    // none.
    std::vector<uint32_t> count(kBins + 1, 0);
    std::vector<double> weight(kBins, 0.0);
    std::uniform_real_distribution<double> uniform(0.0, 1.0);
    const double middle = 20 + 60 * uniform(rng), width = 4 + 20 * uniform(rng), tokens = std::exp(2 + 10 * uniform(rng));
    for (uint32_t b = 0; b < kDead; ++b) {
        const double expected = tokens / width * std::exp(-0.5 * std::pow((b - middle) / width, 2));
        const uint32_t n = b == 0 ? 1 : (uint32_t)std::poisson_distribution<long>(expected + 0.01)(rng);
        count[b + 1] = count[b] + n;
        uint64_t units = 0;
        for (uint32_t i = 0; i < n; ++i) units += (uint64_t)((1.0 + 0.189 * uniform(rng)) * 0x1p37);
        weight[b] = (double)units * std::pow(2.0, -0.25 * b) / 0x1p37;
    }
    count[kBins] = count[kDead];
    const std::vector<double> upto = scan(weight);
    uint32_t last_live = 0;
    for (uint32_t b = 0; b < kDead; ++b)
        if (count[b + 1] > count[b]) last_live = b;
    for (uint32_t b = 1; b < kDead; ++b) {
        falls += upto[b] < upto[b - 1];
        rises += count[b + 1] == count[b] && upto[b] > upto[b - 1];
    }
    for (uint32_t k = 0; k < kDead; ++k)
        for (const double at : {upto[k], std::nextafter(upto[k], 0.0), std::nextafter(upto[k], 1e300), upto[k] * 0.999})
            for (const bool past : {false, true}) {
                uint32_t found = last_live;
                bool some = false;
                for (uint32_t b = kDead; b-- > 0;)
                    if (qwh::sample::may_hold(count[b], count[b + 1], upto[b], at, past)) found = b, some = true;
                expect(count[found + 1] > count[found], "a step without tokens", found, k);
                expect(found <= last_live, "a step behind the last", found, k);
                expect(!some || (past ? upto[found] > at : upto[found] >= at), "a step that does not reach", found, k);
                // (Every earlier one's sum is below, or above by last bits.)
                for (uint32_t b = 0; b < found; ++b)
                    expect(upto[b] <= at * (1 + 0x1p-50) || count[b + 1] == count[b], "a later step than the first", found, b);
            }
}

}  // namespace

int main() {
    std::mt19937_64 rng(11);
    for (int round = 0; round < 150; ++round) histogram(rng);
    expect(falls > 0 && rises > 0, "histograms whose sums fall, and rise over an empty step", falls, rises);
    std::printf("sample: %ld cases, %ld failures, %ld sums that fall, %ld that rise over an empty step\n", cases, failures, falls, rises);
    return failures ? 1 : 0;
}
