// The arithmetic of logits in 64 bits, for the verification of drafts and for sampling: the softcap, and 2^z for the
// weights of a softmax. A drawn token is the one of up to millions whose running sum passes a given point: sums
// that are 1e-7 off would often name its neighbour.
#pragma once

#include "g4_internal.h"

namespace g4 {

// a b + k with k in scalar registers (the compiler would copy it to vector ones first, two moves a step).
__device__ __forceinline__ double fma_k(double a, double b, double k) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(k));
    return r;
}

// The softcap, tanh(x / cap) cap: |x| <= cap / 2 as x + x t P(t), t = (x / cap)^2 (a polynomial fitted on Chebyshev
// nodes, 8e-14 t x off, 11 operations), past that 1 - 2 / (e^2a + 1), which would lose digits where a is small. A
// row's maximum, the bulk of its sums and the judged logits all go through the same two, so that the maximum's
// exponent is 0 and no other's is above: at a temperature of 1e-12 a difference of 1e-13 would count. (Neither falls
// as x grows: below half the cap the values of neighbouring f32 logits are 2^-25 of them apart and 2^-44 off.)
// first: the polynomial's first coefficient, which a loop may keep in a vector register. Cap: cap, inv_cap2 and half_cap, a
// little less than half the cap.
constexpr double kNearCapFirst = 0.00039943422382545215;
template <class Cap>
__device__ __forceinline__ double near_cap(double x, const Cap &A, double first = kNearCapFirst) {
    const double t = x * x * A.inv_cap2;
    double c = first;
    c = fma_k(c, t, -0.0013843999024647944);
    c = fma_k(c, t, 0.0035776163994480498);
    c = fma_k(c, t, -0.008861575554686911);
    c = fma_k(c, t, 0.021869384578835853);
    c = fma_k(c, t, -0.053968250756296965);
    c = fma_k(c, t, 0.1333333332954187);
    c = fma_k(c, t, -0.3333333333332598);
    return __builtin_fma(x, t * c, x);
}
__device__ __forceinline__ double far_cap(double x, double cap) {
    const double a = fabs(x) / cap;
    return copysign(cap * (1.0 - 2.0 / (exp(2.0 * a) + 1.0)), x);
}
template <class Cap>
__device__ __forceinline__ double softcap64(float x, const Cap &A) {
    if (A.cap == 0.0) return x;
    return fabsf(x) > A.half_cap ? far_cap(x, A.cap) : near_cap(x, A);
}
// |x| past what near_cap is good for, -infinity (no weight) not included
template <class Cap>
__device__ __forceinline__ bool is_far(float x, const Cap &A) { return fabsf(x) > A.half_cap && x > -INFINITY; }

// 2^z: z = n + f, |f| <= 1/2, a polynomial in f (fitted like the softcap's, relative error 1.1e-12) and n into the
// exponent; below 2^-1000 that (too small to count, and the exponent stays normal), and for a NaN.
__device__ __forceinline__ double pow2(double z) {
    z = fmax(z, -1000.0);
    const double r = z + 0x1.8p52;  // n in the low word
    const double f = z - (r - 0x1.8p52);
    double e = 1.3259689002093833e-06;
    e = fma_k(e, f, 1.531008106933654e-05);
    e = fma_k(e, f, 0.00015403433582607232);
    e = fma_k(e, f, 0.0013333450560096254);
    e = fma_k(e, f, 0.009618129194093111);
    e = fma_k(e, f, 0.05550410941217064);
    e = fma_k(e, f, 0.24022650695640319);
    e = fma_k(e, f, 0.6931471805459295);
    e = fma_k(e, f, 1.0000000000000135);
    return __hiloint2double(__double2hiint(e) + (int)((uint32_t)__double2loint(r) << 20), __double2loint(e));
}

// NaN: no weight, as -infinity.
__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }

}  // namespace g4
