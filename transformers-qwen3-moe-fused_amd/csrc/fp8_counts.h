// Row counts of the experts, cut where their sum passes the rows there are.  Plain constant-expression arithmetic, for host and
// device.
//
// Counts come from device memory as the caller left them: they may be negative, or sum to more than any integer holds.  Every
// one is first brought to 0 .. rows (2^31 - 1 at most), then summed up to and including each expert's with sums that stay at 2^32 - 1:
// where a sum has come to that, less the expert's own count it is 2^31 at least, past every row.  So what an expert gets are the
// rows between two sums brought to `room`, whatever the counts are.
#pragma once

#include <stdint.h>

namespace mfl {

constexpr uint32_t fp8_count_of(int64_t size, uint32_t rows) { return size <= 0 ? 0u : size < (int64_t)rows ? (uint32_t)size : rows; }
constexpr uint32_t fp8_sum(uint32_t a, uint32_t b) { return a + b < a ? 0xffffffffu : a + b; }
// from the sum up to and including an expert's count: the row behind its last one, and its first one
constexpr uint32_t fp8_end(uint32_t sum, uint32_t room) { return sum < room ? sum : room; }
constexpr uint32_t fp8_begin(uint32_t sum, uint32_t count, uint32_t room) { return fp8_end(sum - count, room); }

}  // namespace mfl
