// Where a place of a row's order lies among the histogram's steps: shared by
// sample.hip and sanitize/sample_check.cpp, which holds it on the CPU.
#pragma once

#include <cstdint>

namespace qwh {
namespace sample {

// Whether the place that the running sum (or count) reaches `at` (past:
// exceeds it) at may lie in a step, `upto` being the sum up to and with it: the
// place is in the first step of which this holds. A scan over a workgroup adds
// in another order for each step, so neighbouring sums may fall or rise by
// their last bits, also over a step without tokens: such a step has no place.
constexpr bool may_hold(uint32_t count_before, uint32_t count_upto, double upto, double at, bool past) {
    return count_upto > count_before && (past ? upto > at : upto >= at);
}

}  // namespace sample
}  // namespace qwh
