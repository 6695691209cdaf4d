// CPU driver for the keys of an attention tile (gemma4-webgpu-engine_amd/csrc/g4_key_span.h): windows up to
// INT32_MAX and positions on either side of 0, against the definition in 64 bits. Built and run by
// tests/test_key_span.py; prints "ok" and exits 0 when it holds.
#include <climits>
#include <cstdint>
#include <cstdio>
#include <initializer_list>

#include "g4_key_span.h"

static bool sees(int64_t p, int64_t j, int64_t window) { return j <= p && (!window || j > p - window); }

int main() {
    const int windows[] = {0, 1, 2, 31, 32, 33, 100, 511, 512, 1 << 20, (1 << 30) - 1, 1 << 30, INT_MAX - 40, INT_MAX - 1, INT_MAX};
    const int ends[] = {-(1 << 30), -100000, -33, -8, -3, -2, -1, 0, 1, 30, 31, 32, 33, 95, 600, 4095, (1 << 30) - 1};
    for (int max_kv : {1, 7, 64, 601, 4096, 1 << 30})
        for (int given : windows) {
            const int window = g4::effective_window(given, max_kv);
            if (window < 0 || window >= max_kv) return std::printf("FAIL: window %d of %d positions\n", window, max_kv), 1;
            for (int p1 : ends)
                for (int rows : {1, 2, 5, 32, 128, 1000}) {
                    if (p1 >= max_kv || p1 < INT_MIN + rows) continue;
                    const int p0 = p1 - rows + 1;
                    const g4::KeySpan K = g4::key_span(p0, p1, window, 32);
                    if (K.lo < 0 || K.lo % 32 || K.lo > K.hi || K.hi > max_kv)
                        return std::printf("FAIL: [%d, %d) of rows %d..%d, window %d\n", K.lo, K.hi, p0, p1, given), 1;
                    // the last row sees the last key of the span, nothing sees the one behind it
                    if (K.hi != (p1 < 0 ? 0 : p1 + 1)) return std::printf("FAIL: end %d of rows ..%d\n", K.hi, p1), 1;
                    for (int64_t p = p0; p <= p1; ++p)  // no row sees a key before the span
                        for (int64_t j : {(int64_t)0, (int64_t)K.lo - 33, (int64_t)K.lo - 1})
                            if (j >= 0 && j < K.lo && sees(p, j, given))
                                return std::printf("FAIL: key %lld of row %lld, window %d\n", (long long)j, (long long)p, given), 1;
                    for (int64_t p = p0; p <= p1; ++p)  // the window put for the call hides what the given one hides
                        for (int64_t j : {(int64_t)0, (int64_t)K.lo, p - given, p - given + 1, p, p + 1})
                            if (j >= 0 && j < max_kv && sees(p, j, given) != sees(p, j, window))
                                return std::printf("FAIL: window %d as %d\n", given, window), 1;
                }
        }
    std::printf("ok\n");
    return 0;
}
