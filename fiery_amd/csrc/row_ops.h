// What the row operators share (layer_norm_kernel.h, dropout.hip): element types, loads and stores of eight columns, the
// counter-based generator behind the dropout masks.
//
// A row's columns are dealt to lanes in UNITS of eight: 16 bytes of a 16-bit type, 32 of fp32, and exactly the columns that one
// call of the generator serves.  Addresses need no alignment beyond the element's (gfx950's global accesses take any), so odd
// widths and row strides use the same wide accesses.
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

// (values, not references: a conditional of two array elements is a conditional address, which keeps the array out of registers)
template <typename V>
__device__ __forceinline__ V pick(bool first, V a, V b) {
    return first ? a : b;
}

// A unit as it lies in memory: loads are issued well before unpack() makes their values.  `count` (0 .. 8) of its columns belong
// to the row, the others come out as zeros and nothing past them is touched.  A last unit with fewer than eight is read as the
// row's last eight columns, so every lane makes the same access, and shifted into place by unpack(); rows narrower than a unit
// go in pieces.  RAGGED: the width is no multiple of eight (0: it is, and none of this is compiled in); 1: every wavefront holds last
// units, all lanes take the shift; 2: few do, and a branch keeps it (and its masks' registers) out of the others; 3:
// rows narrower than a unit.  `live`: whether there is a row
// at all (apart from `count`, which is then the same for all rows of a lane and its comparisons leave the loop).
template <int RAGGED>
__device__ __forceinline__ int unit_count(int C, long long unit) {
    const long long left = C - unit * kUnit;
    return left >= kUnit ? kUnit : RAGGED && left > 0 ? static_cast<int>(left) : 0;
}
template <typename T>
struct Raw {
    unsigned w[sizeof(typename T::store) * kUnit / 4];
};
template <typename T>
__device__ __forceinline__ Raw<T> load_pieces(const typename T::store* p, int count) {
    constexpr int kWords = sizeof(typename T::store) * kUnit / 4;
    Raw<T> r = {};
    const bool h4 = count & 4, h2 = count & 2;
    unsigned four[kWords / 2] = {}, two[kWords / 4] = {}, one = 0;
    if (h4) __builtin_memcpy(four, p, sizeof(four));
    if (h2) __builtin_memcpy(two, p + (count & 4), sizeof(two));
    if (count & 1) {
        typename T::store e = p[count & 6];
        if constexpr (sizeof(e) == 4)
            __builtin_memcpy(&one, &e, 4);
        else
            one = e;
    }
    if constexpr (sizeof(typename T::store) == 4) {
        r.w[0] = pick(h4, four[0], pick(h2, two[0], one));
        r.w[1] = pick(h4, four[1], two[1]);
        r.w[2] = pick(h4, four[2], pick(h2, one, 0u));
        r.w[3] = four[3];
        r.w[4] = pick(h4, pick(h2, two[0], one), 0u);
        r.w[5] = pick(h4, two[1], 0u);
        r.w[6] = pick(h4 && h2, one, 0u);
    } else {
        r.w[0] = pick(h4, four[0], pick(h2, two[0], one));
        r.w[1] = pick(h4, four[1], pick(h2, one, 0u));
        r.w[2] = pick(h4, pick(h2, two[0], one), 0u);
        r.w[3] = pick(h4 && h2, one, 0u);
    }
    return r;
}
template <typename T, int RAGGED>
__device__ __forceinline__ Raw<T> load_raw(const typename T::store* p, bool live, int count) {
    if (RAGGED == 3) return load_pieces<T>(p, live ? count : 0);
    Raw<T> r = {};
    if (live && count > 0) {
        if (RAGGED) p -= kUnit - count;
        __builtin_memcpy(&r.w[0], p, 16);
        if constexpr (sizeof(typename T::store) == 4) __builtin_memcpy(&r.w[4], p + 4, 16);
    }
    return r;
}
template <typename T, int RAGGED>
__device__ __forceinline__ void unpack(Raw<T> r, int count, float (&v)[kUnit]) {
    constexpr int kWords = sizeof(typename T::store) * kUnit / 4;
    const unsigned off = (RAGGED == 1 || RAGGED == 2) && count > 0 ? kUnit - count : 0;
    if (RAGGED == 1 || (RAGGED == 2 && off)) {
        unsigned words = off;
        if constexpr (kWords == 4) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) r.w[i] = funnel_halves(i + 1 < kWords ? r.w[i + 1] : 0u, r.w[i], off & 1u);
            words >>= 1;
        }
#pragma unroll
        for (int step = kWords / 2; step > 0; step >>= 1)
#pragma unroll
            for (int i = 0; i < kWords; ++i) r.w[i] = pick((words & step) != 0, i + step < kWords ? r.w[i + step] : 0u, r.w[i]);
    }
#pragma unroll
    for (int j = 0; j < kUnit; ++j) {
        if constexpr (kWords == 8)
            __builtin_memcpy(&v[j], &r.w[j], 4);
        else
            v[j] = T::value(j & 1 ? r.w[j / 2] >> 16 : r.w[j / 2] & 0xffffu);
    }
}
template <typename T, int RAGGED>
__device__ __forceinline__ void load_unit(const typename T::store* p, int count, float (&v)[kUnit]) {
    unpack<T, RAGGED>(load_raw<T, RAGGED>(p, true, count), count, v);
}
// (a store of less than a unit goes in pieces)
template <typename T, int RAGGED>
__device__ __forceinline__ void store_unit(typename T::store* p, int count, const float (&v)[kUnit]) {
    if (RAGGED ? count == kUnit : count > 0) {
        store_n<T, 8>(p, v);
        return;
    }
    if (!RAGGED || count <= 0) return;
    const bool h4 = count & 4, h2 = count & 2;
    if (h4) store_n<T, 4>(p, v);
    if (h2) {
        const float two[2] = {pick(h4, v[4], v[0]), pick(h4, v[5], v[1])};
        store_n<T, 2>(p + (count & 4), two);
    }
    if (count & 1) {
        const float one[1] = {pick(h4, pick(h2, v[6], v[4]), pick(h2, v[2], v[0]))};
        store_n<T, 1>(p + (count & 6), one);
    }
}

// parameters, whose type is known at run time only: read once per lane, outside the loops
template <int RAGGED>
__device__ __forceinline__ void load_typed(const void* p, int type, long long c, int count, float otherwise, float (&v)[kUnit]) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < kUnit; ++j) v[j] = otherwise;
    } else if (type == FIERY_TYPE_F32) {
        load_unit<F32, RAGGED>(static_cast<const float*>(p) + c, count, v);
    } else if (type == FIERY_TYPE_BF16) {
        load_unit<BF16, RAGGED>(static_cast<const unsigned short*>(p) + c, count, v);
    } else {
        load_unit<F16, RAGGED>(static_cast<const unsigned short*>(p) + c, count, v);
    }
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
// The words of one unit of a row.
__device__ __forceinline__ uint4 drop_words(const DropArgs& d, const DropKey& k, unsigned row, unsigned unit) {
    const unsigned mask_row = d.rows_per_mask.d > 1 ? div_by(row, d.rows_per_mask) : row;
    uint4 w = philox(d.one_column ? 0u : unit, mask_row, k.call_lo, k.call_hi, k.seed_lo, k.seed_hi);
    if (d.one_column) {
        w.x = (w.x << 16) | (w.x & 0xffffu);
        w.y = w.z = w.w = w.x;
    }
    return w;
}
// One unit of a row.  (A select and not a product: a dropped infinity or NaN leaves a zero.  Each half is compared in the upper
// half of a word, with 65536 threshold - 1: 2^32 - 1 where everything is dropped.)
__device__ __forceinline__ void drop_unit(const DropArgs& d, const DropKey& k, unsigned row, unsigned unit, float (&v)[kUnit]) {
    if (d.threshold == 0) return;
    const uint4 w = drop_words(d, k, row, unit);
    const unsigned word[4] = {w.x, w.y, w.z, w.w}, limit = d.threshold * 65536u - 1u;
#pragma unroll
    for (int j = 0; j < kUnit; ++j) v[j] = (j & 1 ? word[j / 2] : word[j / 2] << 16) > limit ? v[j] * d.scale : 0.f;
}
// The same in two steps, for a mask that is used twice (threshold > 0): bit j is set where column j is kept.
__device__ __forceinline__ unsigned drop_bits(const DropArgs& d, const DropKey& k, unsigned row, unsigned unit) {
    const uint4 w = drop_words(d, k, row, unit);
    const unsigned word[4] = {w.x, w.y, w.z, w.w};
    unsigned bits = 0;
#pragma unroll
    for (int j = kUnit - 1; j >= 0; --j) {
        const unsigned half = j & 1 ? word[j / 2] >> 16 : word[j / 2] & 0xffffu;
        bits = bits + bits + ((d.threshold - 1u - half) >> 31);             // (integers: lane masks fill the scalar registers; 4001 bf16 columns 108 us, not 126)
    }
    return bits;
}
__device__ __forceinline__ void drop_by(const DropArgs& d, unsigned bits, float (&v)[kUnit]) {
#pragma unroll
    for (int j = 0; j < kUnit; ++j) {
        unsigned u;
        const float scaled = v[j] * d.scale;
        __builtin_memcpy(&u, &scaled, 4);
        u &= 0u - (bits >> j & 1u);
        __builtin_memcpy(&v[j], &u, 4);
    }
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

struct DropoutArgs {
    const void* x;
    const void* residual;
    void* y;
    long long x_ld, res_ld, y_ld;
    int C;
    unsigned first, total;               // of a launch: its first row, its rows * units per row
    FastDiv units;
    DropArgs drop;
};
void dropout_rows(DropoutArgs a, int64_t rows, int x_type, int y_type, hipStream_t stream);          // dropout.hip

inline bool row_type(int t) { return t == FIERY_TYPE_F32 || t == FIERY_TYPE_BF16 || t == FIERY_TYPE_F16; }

}  // namespace fiery
