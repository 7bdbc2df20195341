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

// Sum over aligned groups of `lanes` (1, 2, 4 .. 64; the same in the whole wavefront) neighbouring lanes, the same in all of
// them.  No LDS: data-parallel moves inside rows of 16 (quad permutations, then mirrors - by then all lanes of a half hold the
// same sum), gfx950's row swaps across them.
template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    if (lanes > 1) {
        v += lane_move<0xB1>(v);                        // quad_perm [1, 0, 3, 2]
        if (lanes > 2) {
            v += lane_move<0x4E>(v);                    // quad_perm [2, 3, 0, 1]
            if (lanes > 4) {
                v += lane_move<0x141>(v);               // row_half_mirror
                if (lanes > 8) {
                    v += lane_move<0x140>(v);           // row_mirror
                    if (lanes > 16) {
                        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
                        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
                        if (lanes > 32) {
                            const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
                            v = __uint_as_float(q[0]) + __uint_as_float(q[1]);
                        }
                    }
                }
            }
        }
    }
    return v;
}

// whether it holds in any lane of the wavefront
__device__ __forceinline__ bool any_lane(bool p) { return __builtin_amdgcn_ballot_w64(p) != 0; }

// v_rsq_f32: 1 / sqrt(x) to about an ulp, for x well inside the range of normal numbers
__device__ __forceinline__ float rsq_estimate(float x) { return __builtin_amdgcn_rsqf(x); }
// the low word of (hi:lo) >> (16 * halves), halves 0 or 1
__device__ __forceinline__ unsigned funnel_halves(unsigned hi, unsigned lo, unsigned halves) { return __builtin_amdgcn_alignbit(hi, lo, halves * 16u); }

}  // namespace fiery
