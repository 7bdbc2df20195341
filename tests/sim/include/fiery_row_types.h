// TEST INFRASTRUCTURE: CPU stand-in for fiery_amd/csrc/fiery_row_types.h, same semantics in integer arithmetic.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>

namespace fiery {

inline unsigned f16_bits(float v) {                                    // round to nearest even, as v_cvt_f16_f32
    unsigned u;
    __builtin_memcpy(&u, &v, 4);
    const unsigned sign = (u >> 16) & 0x8000u, a = u & 0x7fffffffu;
    if (a > 0x7f800000u) return sign | 0x7e00u;
    if (a >= 0x477ff000u) return sign | 0x7c00u;                        // 65520 and more: infinity
    if (a < 0x38800000u) {                                              // below 2^-14: multiples of 2^-24
        float m;
        __builtin_memcpy(&m, &a, 4);
        return sign | static_cast<unsigned>(std::nearbyint(std::ldexp(static_cast<double>(m), 24)));
    }
    return sign | ((a - 0x38000000u + 0xfffu + ((a >> 13) & 1u)) >> 13);
}
inline float f16_value(unsigned bits) {
    const unsigned e = (bits >> 10) & 31u, m = bits & 0x3ffu;
    const double s = (bits & 0x8000u) ? -1.0 : 1.0;
    if (e == 31u) return m ? static_cast<float>(NAN) : static_cast<float>(s * INFINITY);
    return static_cast<float>(s * (e ? std::ldexp(1024.0 + m, static_cast<int>(e) - 25) : std::ldexp(static_cast<double>(m), -24)));
}
inline unsigned bf16_one_bits(float f) {
    unsigned u;
    __builtin_memcpy(&u, &f, 4);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
inline unsigned bf16_pair_bits(float lo, float hi) { return bf16_one_bits(lo) | (bf16_one_bits(hi) << 16); }

inline float lanes_sum(float v, int lanes) {
    for (int m = 1; m < lanes; m <<= 1) v += __shfl_xor(v, m);
    return v;
}
inline bool any_lane(bool p) { return lanes_sum(p ? 1.0f : 0.0f, 64) != 0.0f; }
inline float rsq_estimate(float x) { return 1.0f / std::sqrt(x); }
inline unsigned funnel_halves(unsigned hi, unsigned lo, unsigned halves) {
    return static_cast<unsigned>(((static_cast<unsigned long long>(hi) << 32) | lo) >> (16 * halves));
}

}  // namespace fiery
