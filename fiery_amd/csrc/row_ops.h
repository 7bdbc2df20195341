// What the row operators share (layer_norm_kernel.h, dropout.hip): element types, loads and stores of eight columns, the
// counter-based generator behind the dropout masks.
//
// A row's columns are dealt to lanes in UNITS of eight: 16 bytes of a 16-bit type, 32 of fp32, and exactly the columns that one
// call of the generator serves.  Addresses need no alignment beyond the element's (gfx950's global accesses take any), so odd
// widths and row strides use the same wide accesses; only the last unit of a row whose width is not a multiple of eight goes
// in pieces of four, two and one.
#pragma once
#include <fiery_row_types.h>

#include <type_traits>

#include "common.h"

namespace fiery {

struct F32 {
    typedef float store;
};
struct BF16 {
    typedef unsigned short store;
    static __device__ __forceinline__ float value(unsigned b) {
        const unsigned u = b << 16;
        float f;
        __builtin_memcpy(&f, &u, 4);
        return f;
    }
    static __device__ __forceinline__ unsigned pair(float lo, float hi) { return bf16_pair_bits(lo, hi); }
};
struct F16 {
    typedef unsigned short store;
    static __device__ __forceinline__ float value(unsigned b) { return f16_value(b); }
    static __device__ __forceinline__ unsigned pair(float lo, float hi) { return f16_bits(lo) | (f16_bits(hi) << 16); }
};

constexpr int kUnit = 8;

// the values that a unit has once it is stored as S
template <typename S>
__device__ __forceinline__ void as_stored(const float (&v)[kUnit], float (&out)[kUnit]) {
#pragma unroll
    for (int j = 0; j < kUnit; j += 2) {
        if constexpr (sizeof(typename S::store) == 4) {
            out[j] = v[j];
            out[j + 1] = v[j + 1];
        } else {
            const unsigned w = S::pair(v[j], v[j + 1]);
            out[j] = S::value(w & 0xffffu);
            out[j + 1] = S::value(w >> 16);
        }
    }
}

// N consecutive elements (8, 4, 2 or 1), any alignment of the element's own
template <typename T, int N>
__device__ __forceinline__ void load_n(const typename T::store* p, float* v) {
    if constexpr (sizeof(typename T::store) == 4) {
        if constexpr (N == 8) {
            __builtin_memcpy(v, p, 16);
            __builtin_memcpy(v + 4, p + 4, 16);
        } else {
            __builtin_memcpy(v, p, 4 * N);
        }
    } else if constexpr (N == 1) {
        v[0] = T::value(p[0]);
    } else {
        unsigned w[N / 2];
        __builtin_memcpy(w, p, 2 * N);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            v[2 * i] = T::value(w[i] & 0xffffu);
            v[2 * i + 1] = T::value(w[i] >> 16);
        }
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(typename T::store* p, const float* v) {
    if constexpr (sizeof(typename T::store) == 4) {
        if constexpr (N == 8) {
            __builtin_memcpy(p, v, 16);
            __builtin_memcpy(p + 4, v + 4, 16);
        } else {
            __builtin_memcpy(p, v, 4 * N);
        }
    } else if constexpr (N == 1) {
        p[0] = static_cast<unsigned short>(T::pair(v[0], 0.f) & 0xffffu);
    } else {
        unsigned w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = T::pair(v[2 * i], v[2 * i + 1]);
        __builtin_memcpy(p, w, 2 * N);
    }
}

// The first `count` (0 .. 8) of a unit's elements; the others come out as zeros.  Nothing past them is touched.
template <typename T>
__device__ __forceinline__ void load_unit(const typename T::store* p, int count, float (&v)[kUnit]) {
    if (count == kUnit) {
        load_n<T, 8>(p, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < kUnit; ++j) v[j] = 0.f;
    if (count <= 0) return;
    float four[4] = {0.f, 0.f, 0.f, 0.f}, two[2] = {0.f, 0.f}, one[1] = {0.f};
    if (count & 4) load_n<T, 4>(p, four);
    if (count & 2) load_n<T, 2>(p + (count & 4), two);
    if (count & 1) load_n<T, 1>(p + (count & 6), one);
    const bool h4 = count & 4, h2 = count & 2;
    v[0] = h4 ? four[0] : h2 ? two[0] : one[0];
    v[1] = h4 ? four[1] : h2 ? two[1] : 0.f;
    v[2] = h4 ? four[2] : h2 ? one[0] : 0.f;
    v[3] = four[3];
    v[4] = h4 ? (h2 ? two[0] : one[0]) : 0.f;
    v[5] = h4 && h2 ? two[1] : 0.f;
    v[6] = h4 && h2 ? one[0] : 0.f;
}
template <typename T>
__device__ __forceinline__ void store_unit(typename T::store* p, int count, const float (&v)[kUnit]) {
    if (count == kUnit) {
        store_n<T, 8>(p, v);
        return;
    }
    if (count <= 0) return;
    const bool h4 = count & 4, h2 = count & 2;
    if (h4) store_n<T, 4>(p, v);
    if (h2) {
        const float two[2] = {h4 ? v[4] : v[0], h4 ? v[5] : v[1]};
        store_n<T, 2>(p + (count & 4), two);
    }
    if (count & 1) {
        const float one[1] = {h4 ? (h2 ? v[6] : v[4]) : (h2 ? v[2] : v[0])};
        store_n<T, 1>(p + (count & 6), one);
    }
}

// one element of a tensor whose type is known at run time (parameters: read once per lane, outside the loops)
__device__ __forceinline__ float load_typed(const void* p, int type, long long i) {
    if (type == FIERY_TYPE_F32) return static_cast<const float*>(p)[i];
    const unsigned b = static_cast<const unsigned short*>(p)[i];
    return type == FIERY_TYPE_BF16 ? BF16::value(b) : F16::value(b);
}
__device__ __forceinline__ void store_typed(void* p, int type, long long i, float v) {
    if (type == FIERY_TYPE_F32)
        static_cast<float*>(p)[i] = v;
    else
        static_cast<unsigned short*>(p)[i] =
            static_cast<unsigned short>((type == FIERY_TYPE_BF16 ? BF16::pair(v, 0.f) : F16::pair(v, 0.f)) & 0xffffu);
}

// n / d for n < 2^31 by one wide multiplication (Granlund, Montgomery 1994: the multiplier rounded up, its excess bit as an add)
struct FastDiv {
    unsigned d, m, s;
};
inline FastDiv fast_div(unsigned d) {
    FastDiv f{d, 0, 0};
    while ((1ull << f.s) < d) ++f.s;
    f.m = static_cast<unsigned>(((1ull << 32) * ((1ull << f.s) - d)) / d + 1);
    return f;
}
__device__ __forceinline__ unsigned div_by(unsigned n, FastDiv f) {
    const unsigned t = static_cast<unsigned>((static_cast<unsigned long long>(n) * f.m) >> 32);
    return (t + n) >> f.s;
}

// ---- the dropout mask -----------------------------------------------------------------------------------------------------
// Sixteen bits per value from Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011):
// counter (column / 8, mask row, call low, call high), key (seed low, seed high), column c takes word (c % 8) / 2, its low half
// where c is even.  Kept iff the half is >= threshold = round(65536 p); scale = 65536 / (65536 - threshold), so the expectation
// is exact for the probability that is drawn.  Sixteen bits and not 32: one call (20 wide multiplications, a quarter of the
// vector rate) then serves eight values instead of four, and a bf16 pass stays bound by memory.
struct DropArgs {
    const long long* rng;                // device: {seed, call}
    long long* rng_used;                 // device, may be null: {seed, call + call_add} as this launch used them
    long long call_add;
    unsigned threshold;                  // 0: nothing is dropped, no generator runs
    float scale;
    FastDiv rows_per_mask;               // rows that share one mask row (1: every row its own)
    int one_column;                      // every column takes column 0's number
};

struct DropKey {
    unsigned seed_lo, seed_hi, call_lo, call_hi;
};
__device__ __forceinline__ DropKey drop_key(const DropArgs& d) {
    const unsigned long long seed = static_cast<unsigned long long>(d.rng[0]);
    const unsigned long long call = static_cast<unsigned long long>(d.rng[1]) + static_cast<unsigned long long>(d.call_add);
    return {static_cast<unsigned>(seed), static_cast<unsigned>(seed >> 32), static_cast<unsigned>(call), static_cast<unsigned>(call >> 32)};
}
// (the first thread of the first workgroup: what the backward pass reads, whatever the program does to `rng` meanwhile)
__device__ __forceinline__ void drop_note(const DropArgs& d) {
    if (d.rng_used && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
        d.rng_used[0] = d.rng[0];
        d.rng_used[1] = static_cast<long long>(static_cast<unsigned long long>(d.rng[1]) + static_cast<unsigned long long>(d.call_add));
    }
}

__device__ __forceinline__ uint4 philox(unsigned c0, unsigned c1, unsigned c2, unsigned c3, unsigned k0, unsigned k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const unsigned long long p = 0xD2511F53ull * c0, q = 0xCD9E8D57ull * c2;
        const unsigned n0 = static_cast<unsigned>(q >> 32) ^ c1 ^ k0, n2 = static_cast<unsigned>(p >> 32) ^ c3 ^ k1;
        c1 = static_cast<unsigned>(q);
        c3 = static_cast<unsigned>(p);
        c0 = n0;
        c2 = n2;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    uint4 r;
    r.x = c0;
    r.y = c1;
    r.z = c2;
    r.w = c3;
    return r;
}
// bit j of the result: column 8 * unit + j of the row is kept
__device__ __forceinline__ unsigned drop_bits(const DropArgs& d, const DropKey& k, unsigned row, unsigned unit) {
    const unsigned mask_row = d.rows_per_mask.d > 1 ? div_by(row, d.rows_per_mask) : row;
    const uint4 w = philox(d.one_column ? 0u : unit, mask_row, k.call_lo, k.call_hi, k.seed_lo, k.seed_hi);
    if (d.one_column) return (w.x & 0xffffu) >= d.threshold ? 0xffu : 0u;
    unsigned bits = 0;
    bits |= (w.x & 0xffffu) >= d.threshold ? 1u : 0u;
    bits |= (w.x >> 16) >= d.threshold ? 2u : 0u;
    bits |= (w.y & 0xffffu) >= d.threshold ? 4u : 0u;
    bits |= (w.y >> 16) >= d.threshold ? 8u : 0u;
    bits |= (w.z & 0xffffu) >= d.threshold ? 16u : 0u;
    bits |= (w.z >> 16) >= d.threshold ? 32u : 0u;
    bits |= (w.w & 0xffffu) >= d.threshold ? 64u : 0u;
    bits |= (w.w >> 16) >= d.threshold ? 128u : 0u;
    return bits;
}
// (a select and not a product: a dropped infinity or NaN leaves a zero)
__device__ __forceinline__ void drop_unit(const DropArgs& d, const DropKey& k, unsigned row, unsigned unit, float (&v)[kUnit]) {
    if (d.threshold == 0) return;
    const unsigned bits = drop_bits(d, k, row, unit);
#pragma unroll
    for (int j = 0; j < kUnit; ++j) v[j] = (bits >> j) & 1u ? v[j] * d.scale : 0.f;
}

// host side: the arguments of one call, or an error text
inline const char* drop_args(DropArgs& d, const void* rng, void* rng_used, int64_t call, int threshold, int64_t rows_per_mask, int one_column) {
    if (threshold < 0 || threshold > 65536) return "threshold outside 0 .. 65536";
    if (threshold > 0 && !rng) return "null rng";
    if (rows_per_mask < 1 || rows_per_mask >= (1ll << 31)) return "bad rows_per_mask";
    d.rng = static_cast<const long long*>(rng);
    d.rng_used = threshold > 0 ? static_cast<long long*>(rng_used) : nullptr;
    d.call_add = call;
    d.threshold = static_cast<unsigned>(threshold);
    d.scale = threshold < 65536 ? 65536.f / static_cast<float>(65536 - threshold) : 0.f;
    d.rows_per_mask = fast_div(static_cast<unsigned>(rows_per_mask));
    d.one_column = one_column ? 1 : 0;
    return nullptr;
}

inline bool row_type(int t) { return t == FIERY_TYPE_F32 || t == FIERY_TYPE_BF16 || t == FIERY_TYPE_F16; }

}  // namespace fiery
