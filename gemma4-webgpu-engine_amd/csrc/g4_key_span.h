// Which keys the rows of an attention tile may see. Host and device share the arithmetic; no runtime calls, so
// a CPU test can walk it.
#ifndef G4_KEY_SPAN_H
#define G4_KEY_SPAN_H

#include <cstdint>

namespace g4 {

// A window that reaches behind every position is none: with windows below max_kv (2^30 at most) differences
// of a position and a window stay in 32 bits.
constexpr int effective_window(int window, int max_kv) { return window >= max_kv ? 0 : window; }

// Keys [lo, hi) that rows at positions p0 <= p1 may see, lo a multiple of `unit` (a power of two). Negative
// positions (a sequence with more rows than positions) see none; lo <= hi.
struct KeySpan {
    int lo, hi;
};
constexpr KeySpan key_span(int p0, int p1, int window, int unit) {
    const int lo = window > 0 && p0 >= window ? (p0 - window + 1) & ~(unit - 1) : 0;
    return {lo, p1 < 0 ? 0 : p1 + 1};
}

}  // namespace g4

#endif
