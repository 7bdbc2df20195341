// 16-bit element types and lane exchanges of the row operators (layer norm, dropout) for gfx950.
// Included with angle brackets: the CPU simulator of tests/sim/ supplies a plain C++ stand-in of the same name.
#pragma once
#include <hip/hip_runtime.h>

namespace fiery {

// fp32 -> the nearest fp16 / bf16 value's bits (round to nearest even; one v_cvt each), and back (exact)
__device__ __forceinline__ unsigned f16_bits(float v) {
    const _Float16 h = static_cast<_Float16>(v);
    unsigned short r;
    __builtin_memcpy(&r, &h, 2);
    return r;
}
__device__ __forceinline__ float f16_value(unsigned bits) {
    const unsigned short b = static_cast<unsigned short>(bits);
    _Float16 h;
    __builtin_memcpy(&h, &b, 2);
    return static_cast<float>(h);
}
__device__ __forceinline__ unsigned bf16_pair_bits(float lo, float hi) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
    unsigned r;
    __builtin_memcpy(&r, &v, 4);
    return r;
}

}  // namespace fiery
