// Device arithmetic of the gated feed-forward block's operators, shared by their own kernels and by the contraction kernels'
// epilogues: the activations with their derivatives, and the counter-based generator behind dropout.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

namespace d8k {

// values of the activation argument (D8K_ACT_* in d8k.h)
enum : int { kActSilu = 0, kActGelu = 1, kActGeluTanh = 2, kActRelu = 3, kActSigmoid = 4, kActCount = 5 };

// 1 / (1 + exp(-a)).  FAST (results that are rounded to fp16, whose step is 2^-11): the hardware exponential and a division
// without the last rounding, a few 2^-22 together; 0 below -80, where exp(80) keeps the division in its full range and under 2^-115 is
// nothing beside fp16's 2^-25.  Otherwise the library's exponential and an IEEE division, for negative arguments as e / (1 + e) with
// e = exp(a), which follows the result down to the smallest floats (1 / (1 + exp(-a)) would lose it where exp(-a) overflows).
template <bool FAST>
__device__ __forceinline__ float sigmoid_of(float a) {
    if constexpr (FAST) {
        if (a < -80.0f) return 0.0f;
        return __fdividef(1.0f, 1.0f + __expf(-a));
    } else {
        const float e = expf(-fabsf(a)), r = 1.0f / (1.0f + e);
        return a < 0.0f ? e * r : r;
    }
}
// s = 1 / (1 + exp(-a)) and c = 1 - s, both to a few steps of themselves: 1 / (1 + e) and e / (1 + e) with e = exp(-|a|).  Formed as 1 - s, c would
// be off by the spacing of floats around 1 (0.9 % of it at a = 12) and 0 from a = 17 on.
template <bool FAST>
__device__ __forceinline__ void sigmoid_and_rest(float a, float& s, float& c) {
    const float e = FAST ? __expf(-fabsf(a)) : expf(-fabsf(a));
    const float large = FAST ? __fdividef(1.0f, 1.0f + e) : 1.0f / (1.0f + e), small = e * large;
    s = a < 0.0f ? small : large;
    c = a < 0.0f ? large : small;
}

// value = act(a); slope = act'(a) when wanted.  gelu goes through erfc, gelu_tanh through a sigmoid ((1 + tanh z) / 2 = sigmoid(2 z)):
// both forms keep the relative accuracy of the negative tail, where 1 + erf and 1 + tanh cancel.  FAST: the normal distribution's tail
// beyond |a| is exp(-a^2 / 2) q(|a|), and q a polynomial of degree 7 in 1 / (1 + 0.264 |a|) without a constant, fitted for the least largest
// relative error over |a| <= 14 (linear programming on 1200 Chebyshev points: 5.8e-7 as fitted, 8.9e-7 with these coefficients in 32 bits); the
// library's erfc made the fp16 product of 1531 x 1024 by two of 1024 x 4096 a third longer than the other activations.  Factors beyond +-110 count as 110 where what they multiply has
// vanished (exp(-104) is below the smallest float; an infinite projection times a vanished factor would be a NaN).
template <int ACT, bool FAST, bool SLOPE>
__device__ __forceinline__ void activation(float a, float& value, float& slope) {
    const float lo = a < -110.0f ? -110.0f : a;
    const float b = lo > 110.0f ? 110.0f : lo;
    if constexpr (ACT == kActSilu || ACT == kActSigmoid) {
        float s, c = 0.0f;
        if constexpr (SLOPE) sigmoid_and_rest<FAST>(a, s, c);
        else s = sigmoid_of<FAST>(a);
        value = ACT == kActSilu ? lo * s : s;
        if (SLOPE) slope = ACT == kActSilu ? fmaf(b * s, c, s) : s * c;
    } else if constexpr (ACT == kActGeluTanh) {
        const float c2 = 1.5957691216057308f;  // 2 sqrt(2 / pi)
        const float b2 = b * b, z = c2 * b * fmaf(0.044715f, b2, 1.0f);
        float s, c = 0.0f;
        if constexpr (SLOPE) sigmoid_and_rest<FAST>(z, s, c);
        else s = sigmoid_of<FAST>(z);
        value = lo * s;
        if (SLOPE) slope = fmaf(b * s * c, c2 * fmaf(0.134145f, b2, 1.0f), s);
    } else if constexpr (ACT == kActGelu) {
        float cdf, e;
        if constexpr (FAST) {
            const float x = fabsf(b), t = __fdividef(1.0f, fmaf(0.26445794f, x, 1.0f));
            e = __expf(-0.5f * b * b);
            float q = -0.068581074f;
            q = fmaf(q, t, 0.19961888f);
            q = fmaf(q, t, -0.071617506f);
            q = fmaf(q, t, 0.14575285f);
            q = fmaf(q, t, 0.08163642f);
            q = fmaf(q, t, 0.10782069f);
            q = fmaf(q, t, 0.10536946f);
            const float tail = e * (q * t);
            cdf = b < 0.0f ? tail : 1.0f - tail;
        } else {
            cdf = 0.5f * erfcf(-0.7071067811865476f * b);
            if (SLOPE) e = expf(-0.5f * b * b);
        }
        value = lo * cdf;
        if (SLOPE) slope = fmaf(b * 0.3989422804014327f, e, cdf);
    } else {  // relu: a NaN stays one, so that a diverged projection shows
        value = a <= 0.0f ? 0.0f : a;
        if (SLOPE) slope = a > 0.0f ? 1.0f : 0.0f;
    }
}

// f(std::integral_constant<int, act>): one branch around a whole group of elements.  A branch per element would keep the compiler from
// overlapping the elements' exponentials and divisions, and an epilogue has too few warps to hide them otherwise.
template <class F>
__device__ __forceinline__ void with_activation(int act, F f) {
    switch (act) {
        case kActSilu: f(std::integral_constant<int, kActSilu>()); break;
        case kActGelu: f(std::integral_constant<int, kActGelu>()); break;
        case kActGeluTanh: f(std::integral_constant<int, kActGeluTanh>()); break;
        case kActRelu: f(std::integral_constant<int, kActRelu>()); break;
        default: f(std::integral_constant<int, kActSigmoid>()); break;
    }
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC 2011): four 32-bit words from a
// 128-bit counter under a 64-bit key.  The words of one counter are dropout's decisions for four consecutive elements, so a
// mask is a function of (seed, offset, element) and is computed again wherever it is needed instead of being stored.
// The high word of the group index is an argument of its own: where it is the same for a whole launch (and offset and seed are),
// the two products of the first rounds that do not depend on the low word leave the loops, 2 of 20.
__device__ __forceinline__ uint4 philox4x32(uint32_t group_lo, uint32_t group_hi, unsigned long long offset, unsigned long long seed) {
    uint32_t c0 = group_lo, c1 = group_hi;
    uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint32_t a_hi = __umulhi(c0, 0xD2511F53u), a_lo = c0 * 0xD2511F53u;
        const uint32_t b_hi = __umulhi(c2, 0xCD9E8D57u), b_lo = c2 * 0xCD9E8D57u;
        c0 = b_hi ^ c1 ^ k0;
        c1 = b_lo;
        c2 = a_hi ^ c3 ^ k1;
        c3 = a_lo;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ uint4 philox4x32(unsigned long long group, unsigned long long offset, unsigned long long seed) {
    return philox4x32(static_cast<uint32_t>(group), static_cast<uint32_t>(group >> 32), offset, seed);
}

// What a kernel needs to decide element i: it stays when word i % 4 of counter (i / 4, offset) is at least `threshold`
// (p * 2^32), and is then multiplied by `scale` (1 / (1 - p)).  `counter` (device memory, may be null) is added to `offset` when the kernel
// runs, so that a captured graph draws new masks at every replay.
struct DropSpec {
    unsigned long long seed, offset;
    const unsigned long long* counter;
    uint32_t threshold;
    int some;  // 0: p == 1, nothing stays
    float scale;
};
__device__ __forceinline__ unsigned long long drop_offset(const DropSpec& d) { return d.offset + (d.counter ? *d.counter : 0ull); }
__device__ __forceinline__ bool drop_keeps(const DropSpec& d, uint32_t word) { return d.some && word >= d.threshold; }

}  // namespace d8k
