// What the kernels over rows of logits share: the exponential, differences of scaled logits, 16-byte vectors as they were loaded, and entries
// ordered by value and index.
#pragma once
#include <type_traits>

#include "typed.cuh"

namespace b2 {

constexpr float LOG2E = 1.4426950408889634f;
constexpr unsigned FULL = 0xffffffffu;

// The hardware's exponential, whatever the logits' type: its error of 2^-22 goes into a sum whose own roundings are as large (38400 rows of 259 fp32: 4.2e-8 off in
// the mean, a plain form with expf 4.1e-8).  Results below 2^-126 are 0.
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float max_nan(float a, float b) { float y; asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b)); return y; }
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// z of two logits less what both subtract, z rounded.  Packed products and sums become one packed FMA in the assembler, rounding modifiers or not, and that
// subtracts from the unrounded product; one that is an FMA already, with -0 for its addend, stays as it is.  The -0 is made from the scale, where it can not be
// seen to be one.  With a scale that is a power of two the product needs no rounding, and the one FMA is right (8192 rows of 50001 with four alternatives: 180 us a pass, with
// two instructions 185 us).
struct Exact {
    Pair s, off;
    __device__ __forceinline__ Pair operator()(float x, float y) const { return fma2(pair(x, y), s, off); }
};
struct Rounded {
    Pair s, off, none;
    __device__ __forceinline__ Rounded(Pair s_, Pair off_, float scale) : s(s_), off(off_) {
        const float zero = __fmul_rn(scale, -0.0f);
        none = pair(zero, zero);
    }
    __device__ __forceinline__ Pair operator()(float x, float y) const { return add2(fma2(pair(x, y), s, none), off); }
};
// the same by two products of their own
struct Apart {
    float s; Pair off;
    __device__ __forceinline__ Pair operator()(float x, float y) const { return add2(pair(__fmul_rn(x, s), __fmul_rn(y, s)), off); }
};
// f(function of two logits of type T), the one that the scale asks for: the product of a logit of b bits and a scale of 24 - b bits needs no rounding
template <typename T, typename F> __device__ __forceinline__ void less_of_type(float scale, float minus, F &&f) {
    constexpr unsigned BITS = sizeof(T) == 4 ? 0x7fffffu : std::is_same<T, __half>::value ? 0x7ffu : 0xffu;
    const Pair off = pair(-minus, -minus);
    if ((__float_as_uint(scale) & BITS) == 0) f(Exact{pair(scale, scale), off});
    else f(Apart{scale, off});
}
// f(function of two logits), the one that the scale asks for
template <typename F> __device__ __forceinline__ void less_of(float scale, float minus, F &&f) {
    const Pair s = pair(scale, scale), off = pair(-minus, -minus);
    if ((__float_as_uint(scale) & 0x7fffffu) == 0) f(Exact{s, off});
    else f(Rounded(s, off, scale));
}

// fp32 gradients with the exponential of the full accuracy, 16-bit ones with the hardware's: its error of 2^-22 is lost in their rounding (and a probability
// below 2^-126 is 0)
template <typename T> __device__ __forceinline__ Pair exp_pair(Pair x) {
    const float2 v = halves(sizeof(T) == 4 ? x : mul2(x, pair(LOG2E, LOG2E)));
    return sizeof(T) == 4 ? pair(expf(v.x), expf(v.y)) : pair(ex2(v.x), ex2(v.y));
}

// ---- running sums of exponentials --------------------------------------------------------------------------------------------------
struct Sum { float m, s; };      // largest z met (-inf: none, and s is 0), sum of e^(z - m).  NaN in m stays, whatever is met behind it
__device__ __forceinline__ void rise(Sum &a, float m) {
    if (a.m != neg_inf()) {
        const float r = ex2((a.m - m) * LOG2E);
        a.s = r == 0.0f ? 0.0f : r * a.s;
    }
    a.m = max_nan(a.m, m);
}
__device__ __forceinline__ Sum join(Sum a, Sum b) {
    const float m = max_nan(a.m, b.m);
    if (m == neg_inf()) return a;
    if (b.m != neg_inf()) rise(b, m); else b.s = 0.0f;
    rise(a, m);
    return {m, a.s + b.s};
}
template <int TEAM> __device__ __forceinline__ Sum team_join(Sum a) {
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1) a = join(a, {__shfl_xor_sync(FULL, a.m, o), __shfl_xor_sync(FULL, a.s, o)});
    return a;
}

// ---- vectors of 16 bytes as they were loaded ------------------------------------------------------------------------------------------
template <typename T> struct Raw;
template <> struct Raw<float> {
    static constexpr unsigned NONE = 0xff800000u;      // -inf in every place of a word
    static __device__ __forceinline__ void values(float (&z)[4], const uint4 &q) {
        z[0] = __uint_as_float(q.x); z[1] = __uint_as_float(q.y); z[2] = __uint_as_float(q.z); z[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ float largest(unsigned a) { return __uint_as_float(a); }
};
template <> struct Raw<__nv_bfloat16> {
    static constexpr unsigned NONE = 0xff80ff80u;
    static __device__ __forceinline__ float2 two(unsigned a) { return make_float2(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u)); }
    static __device__ __forceinline__ void values(float (&z)[8], const uint4 &q) {
        const float2 a = two(q.x), b = two(q.y), c = two(q.z), d = two(q.w);
        z[0] = a.x; z[1] = a.y; z[2] = b.x; z[3] = b.y; z[4] = c.x; z[5] = c.y; z[6] = d.x; z[7] = d.y;
    }
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { unsigned y; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b)); return y; }
    static __device__ __forceinline__ float largest(unsigned a) { const float2 v = two(a); return max_nan(v.x, v.y); }
};
template <> struct Raw<__half> {
    static constexpr unsigned NONE = 0xfc00fc00u;
    static __device__ __forceinline__ float2 two(unsigned a) { return __half22float2(*reinterpret_cast<const __half2 *>(&a)); }
    static __device__ __forceinline__ void values(float (&z)[8], const uint4 &q) {
        const float2 a = two(q.x), b = two(q.y), c = two(q.z), d = two(q.w);
        z[0] = a.x; z[1] = a.y; z[2] = b.x; z[3] = b.y; z[4] = c.x; z[5] = c.y; z[6] = d.x; z[7] = d.y;
    }
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { unsigned y; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b)); return y; }
    static __device__ __forceinline__ float largest(unsigned a) { const float2 v = two(a); return max_nan(v.x, v.y); }
};
template <typename T> __device__ __forceinline__ unsigned larger_of(const uint4 &q) {
    typedef Raw<T> R;
    return R::larger(R::larger(q.x, q.y), R::larger(q.z, q.w));
}

// ---- entries in order ------------------------------------------------------------------------------------------------------------------
// An entry is one 64-bit key: the value as an ordered integer above, the complement of its index below; larger is better.  0 is no entry.
typedef unsigned long long Key;
__device__ __forceinline__ unsigned ordered(float z) {
    const unsigned b = __float_as_uint(z + 0.0f);           // -0 counts as 0
    return z != z ? FULL : (b ^ ((b >> 31) ? FULL : 0x80000000u));
}
__device__ __forceinline__ float ordered_value(unsigned o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : FULL)); }
__device__ __forceinline__ Key make_key(float z, int index) { return ((Key)ordered(z) << 32) | (unsigned)~index; }
__device__ __forceinline__ float key_value(Key k) { return ordered_value((unsigned)(k >> 32)); }
__device__ __forceinline__ int key_index(Key k) { return (int)~(unsigned)k; }

}  // namespace b2
