// Layer norm over the channels of pixel-major rows, forward and backward, alone or behind residual + dropout (JOIN).
//
//   h = x                                    (alone)         h = residual + drop(x)          (JOIN; mask: row_ops.h)
//   mean = sum h / C,  var = sum (h - mean)^2 / C,  rstd = 1 / sqrt(var + eps),  xhat = (h - mean) rstd,  y = xhat gamma + beta
//   backward:  gg = dy gamma,  dh' = [dh +] rstd (gg - (sum gg + xhat sum gg xhat) / C),
//              dx = dh' (alone) or drop(dh'), dresidual = dh' (JOIN);  dgamma = sum over rows of dy xhat,  dbeta = sum dy.
//
// Memory-bound: every tensor is read once and written once.  A row lives in registers between its load and its store, so the
// two sums (mean, then squared distances from it: no cancellation) cost no second pass.  A row is dealt to lanes in units of
// eight columns (row_ops.h): a power-of-two group of up to 64 lanes of one wavefront (C <= 1024, no barrier), a workgroup (up
// to 8192), or, past that, a workgroup that walks the row three times.
// The mean itself is corrected by the mean of the distances from it, and the variance by that correction's square: the sum of a row's
// values is rounded (1000 values of 12345.678 had a mean off by 0.002, y by 0.5).  Where the correction is no small part of the
// variance (values closer together than their sum's rounding: constant rows), the distances are taken once more.  It costs one value
// more in the second exchange: 90,720 x 128 fp16 forward 11.2 us, 10.3 without; 8192 x 4096 bf16 27 and 26, joined 53 and 52.
// The backward pass deals a lane the same columns for all its rows, so dgamma and dbeta grow in registers; every workgroup
// leaves one partial row and k_norm_finish adds them in a fixed order in double.  Sums and statistics are fp32; what is
// stored in 16 bits is rounded once, at the store.
// With a 16-bit stream y comes from the h before its rounding, while the statistics that are kept are those of the h that is
// stored, which is what the backward pass reads: its xhat then sums to zero and has its variance, and the gradient is the norm's
// at that h.  (With the other statistics a row of small variance beside a large mean had an xhat off by |mean| rstd / 256.)
// That gradient carries h's rounding: dgamma's error grows with |mean| rstd.  SUM (16-bit streams, the caller's choice): the backward
// pass makes h again from x and residual, unrounded, under the statistics of that h; one tensor more to read (480,000 x 64 bf16: 82 us
// against 65; 8192 x 4096 bf16: 90 - 95 against 73 - 80, both with the sum of the partial rows).
//
// Measured (one MI355X; a large copy reaches 5.35 TB/s): 480,000 x 64 fp32 forward 46 us = 5.4 TB/s, backward 69 + 5 us = 5.0 TB/s,
// joined 95 and 120 + 5 us = 5.2 and 4.9 TB/s; 8192 x 4096 bf16 29 and 39 + 4 us = 4.7 TB/s, joined 52 and (SUM) 87 + 5 us = 5.1 and 4.4 TB/s,
// beside an fp32 stream 72 and 102 + 5 us = 5.6 and 4.9 TB/s; 90,720 x 128 fp16 forward 11 - 12 us = 3.9 TB/s.  Counter traffic is the
// operands' and the partial rows'.  240,000 x 35 bf16: 14 and 19 + 5 us = 2.4 and 2.1 TB/s, joined 30 and (SUM) 39 + 5 us, bound by
// instructions: the layout puts five units on eight lanes.  3000 x 10,000 bf16 (three walks): 45 and 45 + 22 + 10 us = 2.7 and 1.2 TB/s,
// joined 104 and (SUM) 127 + 32 + 10 us: the walks after the first come out of the caches.
#pragma once
#include "row_ops.h"

namespace fiery {

struct NormFwdArgs {
    const void* x;
    const void* residual;
    const void* gamma;
    const void* beta;
    void* y;
    void* h;
    float* mean;                         // [rows], may be null (no backward pass will follow)
    float* rstd;
    long long x_ld, res_ld, y_ld, h_ld;
    int rows, C, lane_bits, param_type;
    float eps, inv_c;
    int of_sum;                          // mean, rstd: of the h before its rounding (a backward pass with x and residual follows)
    DropArgs drop;
};

struct NormBwdArgs {
    const void* dy;
    const void* dh;                      // JOIN: gradient of h itself, may be null
    const void* h;                       // the rows that were normalised (alone: x; SUM: the residual)
    const void* x;                       // SUM only
    const void* gamma;
    const float* mean;
    const float* rstd;
    void* dx;                            // may be null
    void* dres;                          // JOIN, may be null
    float* partial;                      // [workgroups][2][round_up(C, 8)]: dgamma, dbeta of a workgroup's rows; null: not wanted
    void* dgamma;                        // written here by a single workgroup
    void* dbeta;
    long long dy_ld, dh_ld, h_ld, x_ld, dx_ld, dres_ld;
    int rows, C, lane_bits, param_type;
    float inv_c;
    DropArgs drop;
};

namespace {

// Sum over the lanes that share a row, the same in all of them.  THREADS > 0: over the workgroup, through one of two slots used in
// turn (a slot is written again only behind the barrier of the call in between).
constexpr int kSums = 4;                 // values of one exchange, at most
template <int THREADS, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int lanes, float (*slots)[kSums][16], int& turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum(v[i], THREADS ? 64 : lanes);
    if constexpr (THREADS > 0) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) slots[turn][i][wave] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < THREADS / 64; ++w) v[i] += slots[turn][i][w];
        }
        turn ^= 1;
    }
}

// A row's mean and variance from a first mean and the sums of the distances from it and of their squares.  `again`: the squares have to
// be taken from the corrected mean (also where their sum overflowed).
struct Moments {
    float mean, var;
    bool again;
};
__device__ __forceinline__ Moments moments_of(float first, float distances, float squares, float inv_c) {
    const float off = distances * inv_c, raw = squares * inv_c, part = off * off;
    return {first + off, fmaf(-off, off, raw), !(part <= raw * 0x1p-20f && raw <= 3.4028234e38f)};
}

// 1 / sqrt(x) of a variance plus eps: the hardware's estimate and one Newton step, or the exact functions at the ends of the range
__device__ __forceinline__ float rstd_of(float x) {
    if (!(x > 1e-30f && x < 1e30f)) return 1.f / sqrtf(x);
    const float r = rsq_estimate(x);
    return fmaf(r * fmaf(-x * r, r, 1.f), 0.5f, r);
}

// one unit of h: x alone, or residual + drop(x), written out as it is read
template <typename T, typename S, bool JOIN, int RAGGED>
__device__ __forceinline__ void load_h(const NormFwdArgs& a, const DropKey& key, long long row, bool live, int unit, int count, bool write, float (&v)[kUnit]) {
    const long long c = static_cast<long long>(unit) * kUnit;
    const Raw<T> x = load_raw<T, RAGGED>(static_cast<const typename T::store*>(a.x) + row * a.x_ld + c, live, count);
    if constexpr (!JOIN) {
        unpack<T, RAGGED>(x, count, v);
    } else {
        const Raw<S> residual = load_raw<S, RAGGED>(static_cast<const typename S::store*>(a.residual) + row * a.res_ld + c, live, count);
        float r[kUnit];
        unpack<T, RAGGED>(x, count, v);
        unpack<S, RAGGED>(residual, count, r);
        drop_unit(a.drop, key, static_cast<unsigned>(row), static_cast<unsigned>(unit), v);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) v[j] += r[j];
        if (write && live) store_unit<S, RAGGED>(static_cast<typename S::store*>(a.h) + row * a.h_ld + c, count, v);
    }
}

template <int RAGGED>
__device__ __forceinline__ void distances(const float (&v)[kUnit], int count, float mean, float& e, float& q) {
    if (RAGGED == 1 || RAGGED == 3 || (RAGGED == 2 && count < kUnit)) {
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
            const float d = j < count ? v[j] - mean : 0.f;
            e += d;
            q += d * d;
        }
    } else if (count) {
        float p = 0.f;
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
            const float d = v[j] - mean;
            e += d;
            p += d * d;
        }
        q += p;
    }
}
// (each value times 1 / C, not their sum: no overflow where the mean is finite)
__device__ __forceinline__ void add_means(const float (&v)[kUnit], float inv_c, float& s) {
#pragma unroll
    for (int j = 0; j < kUnit; ++j) s = fmaf(v[j], inv_c, s);
}
template <typename S>
__device__ __forceinline__ void add_stored(const float (&v)[kUnit], float inv_c, float& s) {
    float r[kUnit];
    as_stored<S>(v, r);
    add_means(r, inv_c, s);
}
// distances of h (sums 0, 1) and, with TWO, of the stored h (sums 2, 3)
template <typename S, bool TWO, int RAGGED, int N>
__device__ __forceinline__ void add_distances(const float (&v)[kUnit], int count, float mean, float stored_mean, float (&d)[N]) {
    distances<RAGGED>(v, count, mean, d[0], d[1]);
    if constexpr (TWO) {
        float r[kUnit];
        as_stored<S>(v, r);
        distances<RAGGED>(r, count, stored_mean, d[2], d[3]);
    }
}
template <typename T, typename S, bool JOIN, int NV, int THREADS, int RAGGED>
__global__ __launch_bounds__(THREADS ? THREADS : 256) void k_norm_fwd(NormFwdArgs a) {
    __shared__ float slots[2][kSums][16];
    int turn = 0;
    const int lanes = THREADS ? THREADS : 1 << a.lane_bits;
    const int sub = static_cast<int>(threadIdx.x) & (lanes - 1);
    const int per_block = THREADS ? 1 : 256 >> a.lane_bits;
    const int mine = THREADS ? 0 : static_cast<int>(threadIdx.x) >> a.lane_bits;
    DropKey key = {0, 0, 0, 0};
    if constexpr (JOIN) {
        if (a.drop.threshold) key = drop_key(a.drop);
        drop_note(a.drop);
    }
    float ga[NV][kUnit], be[NV][kUnit];
    int count[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int unit = i * lanes + sub;
        count[i] = unit_count<RAGGED>(a.C, unit);
        load_typed<RAGGED>(a.gamma, a.param_type, static_cast<long long>(unit) * kUnit, count[i], 1.f, ga[i]);
        load_typed<RAGGED>(a.beta, a.param_type, static_cast<long long>(unit) * kUnit, count[i], 0.f, be[i]);
    }
    // (every lane of a wavefront walks the loop as often as its neighbours: the exchanges need all of them)
    for (long long first = static_cast<long long>(blockIdx.x) * per_block; first < a.rows; first += static_cast<long long>(gridDim.x) * per_block) {
        const long long row = first + mine;
        const bool live = row < a.rows;
        constexpr bool two = JOIN && sizeof(typename S::store) == 2;            // the stored h has statistics of its own
        float v[NV][kUnit];
        constexpr int kStored = two ? 2 : 0;                                    // where the kept statistics' sums are
        float s[two ? 2 : 1] = {}, d[2 + kStored] = {};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            load_h<T, S, JOIN, RAGGED>(a, key, row, live, i * lanes + sub, count[i], true, v[i]);
            add_means(v[i], a.inv_c, s[0]);
            if constexpr (two) add_stored<S>(v[i], a.inv_c, s[1]);
        }
        row_sums<THREADS>(s, lanes, slots, turn);
#pragma unroll
        for (int i = 0; i < NV; ++i) add_distances<S, two, RAGGED>(v[i], count[i], s[0], s[kStored / 2], d);
        row_sums<THREADS>(d, lanes, slots, turn);
        Moments m = moments_of(s[0], d[0], d[1], a.inv_c), k = moments_of(s[kStored / 2], d[kStored], d[kStored + 1], a.inv_c);
        // (a workgroup's lanes agree; a wavefront's hold several rows, and all of them are needed for the exchange)
        if (THREADS ? m.again || k.again : any_lane(m.again || k.again)) {
            float f[2 + kStored] = {};
#pragma unroll
            for (int i = 0; i < NV; ++i) add_distances<S, two, RAGGED>(v[i], count[i], m.mean, k.mean, f);
            row_sums<THREADS>(f, lanes, slots, turn);
            if (m.again) m.var = f[1] * a.inv_c;
            if (k.again) k.var = f[kStored + 1] * a.inv_c;
        }
        const float mean = m.mean, rstd = rstd_of(m.var + a.eps);
        if (a.mean && live && sub == 0) {
            const bool stored = two && !a.of_sum;
            a.mean[row] = stored ? k.mean : mean;
            a.rstd[row] = stored ? rstd_of(k.var + a.eps) : rstd;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float out[kUnit];
#pragma unroll
            for (int j = 0; j < kUnit; ++j) out[j] = (v[i][j] - mean) * rstd * ga[i][j] + be[i][j];
            if (live) store_unit<T, RAGGED>(static_cast<typename T::store*>(a.y) + row * a.y_ld + static_cast<long long>(i * lanes + sub) * kUnit, count[i], out);
        }
    }
}

// Rows past what the registers of a workgroup hold: three walks over the row (sum, squared distances, result); the second and
// third come out of the caches.
template <typename T, typename S, bool JOIN>
__global__ __launch_bounds__(1024) void k_norm_fwd_long(NormFwdArgs a) {
    __shared__ float slots[2][kSums][16];
    int turn = 0;
    const int units = (a.C + kUnit - 1) / kUnit;
    DropKey key = {0, 0, 0, 0};
    if constexpr (JOIN) {
        if (a.drop.threshold) key = drop_key(a.drop);
        drop_note(a.drop);
    }
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        constexpr bool two = JOIN && sizeof(typename S::store) == 2;
        constexpr int kStored = two ? 2 : 0;
        float v[kUnit], s[two ? 2 : 1] = {};
        for (int u = threadIdx.x; u < units; u += blockDim.x) {
            load_h<T, S, JOIN, 2>(a, key, row, true, u, unit_count<2>(a.C, u), true, v);
            add_means(v, a.inv_c, s[0]);
            if constexpr (two) add_stored<S>(v, a.inv_c, s[1]);
        }
        row_sums<1024>(s, 64, slots, turn);
        Moments m = {s[0], 0.f, false}, k = {s[kStored / 2], 0.f, false};
        for (int walk = 0; walk < 2; ++walk) {
            float d[2 + kStored] = {};
            for (int u = threadIdx.x; u < units; u += blockDim.x) {
                const int count = unit_count<2>(a.C, u);
                load_h<T, S, JOIN, 2>(a, key, row, true, u, count, false, v);
                add_distances<S, two, 2>(v, count, m.mean, k.mean, d);
            }
            row_sums<1024>(d, 64, slots, turn);
            if (walk == 0) {
                m = moments_of(s[0], d[0], d[1], a.inv_c);
                k = moments_of(s[kStored / 2], d[kStored], d[kStored + 1], a.inv_c);
                if (!m.again && !k.again) break;
            } else {
                if (m.again) m.var = d[1] * a.inv_c;
                if (k.again) k.var = d[kStored + 1] * a.inv_c;
            }
        }
        const float mean = m.mean, rstd = rstd_of(m.var + a.eps);
        if (a.mean && threadIdx.x == 0) {
            const bool stored = two && !a.of_sum;
            a.mean[row] = stored ? k.mean : mean;
            a.rstd[row] = stored ? rstd_of(k.var + a.eps) : rstd;
        }
        for (int u = threadIdx.x; u < units; u += blockDim.x) {
            const int count = unit_count<2>(a.C, u);
            load_h<T, S, JOIN, 2>(a, key, row, true, u, count, false, v);
            float ga[kUnit], be[kUnit];
            load_typed<2>(a.gamma, a.param_type, static_cast<long long>(u) * kUnit, count, 1.f, ga);
            load_typed<2>(a.beta, a.param_type, static_cast<long long>(u) * kUnit, count, 0.f, be);
#pragma unroll
            for (int j = 0; j < kUnit; ++j) v[j] = (v[j] - mean) * rstd * ga[j] + be[j];
            store_unit<T, 2>(static_cast<typename T::store*>(a.y) + row * a.y_ld + static_cast<long long>(u) * kUnit, count, v);
        }
    }
}

// SUM: the unit of h from the residual's (in v) and x's; -> which of its columns are kept
template <typename T, int RAGGED>
__device__ __forceinline__ unsigned sum_again(const NormBwdArgs& a, const DropKey& key, long long row, int unit, int count, const Raw<T>& x, float (&v)[kUnit]) {
    float d[kUnit];
    unpack<T, RAGGED>(x, count, d);
    unsigned bits = 0;
    if (a.drop.threshold) {
        bits = drop_bits(a.drop, key, static_cast<unsigned>(row), static_cast<unsigned>(unit));
        drop_by(a.drop, bits, d);
    }
#pragma unroll
    for (int j = 0; j < kUnit; ++j) v[j] = d[j] + v[j];
    return bits;
}

// xhat of the columns that are none is (0 - mean) rstd, and 0 times it would be NaN in the row's sums where that overflows
__device__ __forceinline__ void clear_far(float (&xhat)[kUnit], int count, float mean, float rstd) {
    if (fabsf(mean * rstd) <= 3.4028234e38f) return;
#pragma unroll
    for (int j = 0; j < kUnit; ++j) xhat[j] = j < count ? xhat[j] : 0.f;
}

// One unit of the backward pass's results from its dy (gg = dy gamma), xhat and the row's sums.
template <typename T, typename S, bool JOIN, int RAGGED, bool SUM>
__device__ __forceinline__ void store_grads(const NormBwdArgs& a, const DropKey& key, long long row, int unit, int count, const float (&gg)[kUnit],
                                            const float (&xhat)[kUnit], const Raw<S>& dh, unsigned bits, float rstd, float m1, float m2) {
    const long long c = static_cast<long long>(unit) * kUnit;
    float out[kUnit];
#pragma unroll
    for (int j = 0; j < kUnit; ++j) out[j] = rstd * (gg[j] - (m1 + xhat[j] * m2));
    if constexpr (JOIN) {
        if (a.dh) {
            float d[kUnit];
            unpack<S, RAGGED>(dh, count, d);
#pragma unroll
            for (int j = 0; j < kUnit; ++j) out[j] += d[j];
        }
        if (a.dres) store_unit<S, RAGGED>(static_cast<typename S::store*>(a.dres) + row * a.dres_ld + c, count, out);
        if (!a.dx) return;
        if constexpr (!SUM)
            drop_unit(a.drop, key, static_cast<unsigned>(row), static_cast<unsigned>(unit), out);
        else if (a.drop.threshold)
            drop_by(a.drop, bits, out);
    } else {
        if (!a.dx) return;
    }
    store_unit<T, RAGGED>(static_cast<typename T::store*>(a.dx) + row * a.dx_ld + c, count, out);
}

template <typename T, typename S, bool JOIN, int NV, int THREADS, int RAGGED, bool SUM>
__global__ __launch_bounds__(THREADS ? THREADS : 256) void k_norm_bwd(NormBwdArgs a) {
    typedef typename std::conditional<JOIN, S, T>::type H;
    __shared__ float slots[2][kSums][16];
    int turn = 0;
    const int lanes = THREADS ? THREADS : 1 << a.lane_bits;
    const int sub = static_cast<int>(threadIdx.x) & (lanes - 1);
    const int per_block = THREADS ? 1 : 256 >> a.lane_bits;
    const int mine = THREADS ? 0 : static_cast<int>(threadIdx.x) >> a.lane_bits;
    DropKey key = {0, 0, 0, 0};
    if constexpr (JOIN)
        if (a.drop.threshold) key = drop_key(a.drop);
    float ga[NV][kUnit], dg[NV][kUnit], db[NV][kUnit];
    int count[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        count[i] = unit_count<RAGGED>(a.C, i * lanes + sub);
        load_typed<RAGGED>(a.gamma, a.param_type, static_cast<long long>(i * lanes + sub) * kUnit, count[i], 1.f, ga[i]);
#pragma unroll
        for (int j = 0; j < kUnit; ++j) dg[i][j] = db[i][j] = 0.f;
    }
    // the next row's values are on their way while this row's sums go round the lanes
    const long long step = static_cast<long long>(gridDim.x) * per_block;
    Raw<H> h_next[NV];
    Raw<T> g_next[NV];
    Raw<S> d_next[NV] = {};
    Raw<T> x_next[SUM ? NV : 1] = {};
    float mean_next = 0.f, rstd_next = 0.f;
    const auto fetch = [&](long long first) {
        const long long row = first + mine;
        const bool live = row < a.rows;
        const long long at = live ? row : 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int unit = i * lanes + sub;
            h_next[i] = load_raw<H, RAGGED>(static_cast<const typename H::store*>(a.h) + at * a.h_ld + static_cast<long long>(unit) * kUnit, live, count[i]);
            g_next[i] = load_raw<T, RAGGED>(static_cast<const typename T::store*>(a.dy) + at * a.dy_ld + static_cast<long long>(unit) * kUnit, live, count[i]);
            if constexpr (SUM) x_next[i] = load_raw<T, RAGGED>(static_cast<const typename T::store*>(a.x) + at * a.x_ld + static_cast<long long>(unit) * kUnit, live, count[i]);
            if (JOIN && a.dh) d_next[i] = load_raw<S, RAGGED>(static_cast<const typename S::store*>(a.dh) + at * a.dh_ld + static_cast<long long>(unit) * kUnit, live, count[i]);
        }
        mean_next = live ? a.mean[row] : 0.f;                                      // (a row that is none has xhat 0, whatever row 0 holds)
        rstd_next = live ? a.rstd[row] : 0.f;
    };
    const long long begin = static_cast<long long>(blockIdx.x) * per_block;
    if (begin < a.rows) fetch(begin);
    for (long long first = begin; first < a.rows; first += step) {
        const long long row = first + mine;
        const bool live = row < a.rows;
        const long long at = live ? row : 0;
        const float mean = mean_next, rstd = rstd_next;
        float gg[NV][kUnit], xhat[NV][kUnit], s[2] = {0.f, 0.f};
        Raw<S> dh[NV];
        unsigned bits[NV] = {};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            dh[i] = d_next[i];
            unpack<H, RAGGED>(h_next[i], count[i], xhat[i]);
            if constexpr (SUM) bits[i] = sum_again<T, RAGGED>(a, key, at, i * lanes + sub, count[i], x_next[i], xhat[i]);
            unpack<T, RAGGED>(g_next[i], count[i], gg[i]);
        }
        if (first + step < a.rows) fetch(first + step);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < kUnit; ++j) xhat[i][j] = (xhat[i][j] - mean) * rstd;
            clear_far(xhat[i], count[i], mean, rstd);                              // (past the row gg is 0)
#pragma unroll
            for (int j = 0; j < kUnit; ++j) {
                dg[i][j] += gg[i][j] * xhat[i][j];
                db[i][j] += gg[i][j];
                gg[i][j] *= ga[i][j];
                s[0] += gg[i][j];
                s[1] += gg[i][j] * xhat[i][j];
            }
        }
        row_sums<THREADS>(s, lanes, slots, turn);
        const float m1 = s[0] * a.inv_c, m2 = s[1] * a.inv_c;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (live && count[i]) store_grads<T, S, JOIN, RAGGED, SUM>(a, key, at, i * lanes + sub, count[i], gg[i], xhat[i], dh[i], bits[i], rstd, m1, m2);
    }
    if (!a.partial && !a.dgamma && !a.dbeta) return;
    const int width = (a.C + kUnit - 1) / kUnit * kUnit;
    bool writes = true;
    if constexpr (THREADS == 0) {
        // the lanes that hold the same columns: those of this wavefront, then the other three wavefronts', in order
        __shared__ float others[3][NV * 64 * kUnit][2];
        const int wave = static_cast<int>(threadIdx.x) >> 6, lane = static_cast<int>(threadIdx.x) & 63;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < kUnit; ++j) {
                for (int m = lanes; m < 64; m <<= 1) {
                    dg[i][j] += __shfl_xor(dg[i][j], m);
                    db[i][j] += __shfl_xor(db[i][j], m);
                }
                if (wave > 0 && lane < lanes) {
                    const int c = (i * lanes + lane) * kUnit + j;
                    others[wave - 1][c][0] = dg[i][j];
                    others[wave - 1][c][1] = db[i][j];
                }
            }
        __syncthreads();
        writes = wave == 0 && lane < lanes;
        if (writes) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < kUnit; ++j)
                    for (int w = 0; w < 3; ++w) {
                        const int c = (i * lanes + lane) * kUnit + j;
                        dg[i][j] += others[w][c][0];
                        db[i][j] += others[w][c][1];
                    }
        }
    }
    if (!writes) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * lanes + sub) * kUnit;
        if (c >= a.C) continue;
        if (gridDim.x > 1) {
            float* row = a.partial + static_cast<long long>(blockIdx.x) * 2 * width + c;
            store_n<F32, 8>(row, dg[i]);
            store_n<F32, 8>(row + width, db[i]);
            continue;
        }
        for (int j = 0; j < kUnit && c + j < a.C; ++j) {
            if (a.dgamma) store_typed(a.dgamma, a.param_type, c + j, dg[i][j]);
            if (a.dbeta) store_typed(a.dbeta, a.param_type, c + j, db[i][j]);
        }
    }
}

// Rows past the registers: the row's sums in one walk, its results in a second; dgamma and dbeta in k_norm_bwd_cols_long.
template <typename T, typename S, bool JOIN, bool SUM>
__global__ __launch_bounds__(1024) void k_norm_bwd_long(NormBwdArgs a) {
    typedef typename std::conditional<JOIN, S, T>::type H;
    __shared__ float slots[2][kSums][16];
    int turn = 0;
    const int units = (a.C + kUnit - 1) / kUnit;
    DropKey key = {0, 0, 0, 0};
    if constexpr (JOIN)
        if (a.drop.threshold) key = drop_key(a.drop);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float mean = a.mean[row], rstd = a.rstd[row];
        float gg[kUnit], xhat[kUnit], s[2] = {0.f, 0.f};
        for (int walk = 0; walk < 2; ++walk) {
            const float m1 = s[0] * a.inv_c, m2 = s[1] * a.inv_c;
            for (int u = threadIdx.x; u < units; u += blockDim.x) {
                const int count = unit_count<2>(a.C, u);
                const long long c = static_cast<long long>(u) * kUnit;
                load_unit<H, 2>(static_cast<const typename H::store*>(a.h) + row * a.h_ld + c, count, xhat);
                unsigned bits = 0;
                if constexpr (SUM) {
                    const Raw<T> x = load_raw<T, 2>(static_cast<const typename T::store*>(a.x) + row * a.x_ld + c, true, count);
                    bits = sum_again<T, 2>(a, key, row, u, count, x, xhat);
                }
                load_unit<T, 2>(static_cast<const typename T::store*>(a.dy) + row * a.dy_ld + c, count, gg);
                float ga[kUnit];
                load_typed<2>(a.gamma, a.param_type, c, count, 1.f, ga);
#pragma unroll
                for (int j = 0; j < kUnit; ++j) {
                    xhat[j] = (xhat[j] - mean) * rstd;
                    gg[j] *= ga[j];
                }
                clear_far(xhat, count, mean, rstd);
                if (walk == 0) {
#pragma unroll
                    for (int j = 0; j < kUnit; ++j) {
                        s[0] += gg[j];
                        s[1] += gg[j] * xhat[j];
                    }
                } else {
                    Raw<S> dh = {};
                    if (JOIN && a.dh) dh = load_raw<S, 2>(static_cast<const typename S::store*>(a.dh) + row * a.dh_ld + c, true, count);
                    store_grads<T, S, JOIN, 2, SUM>(a, key, row, u, count, gg, xhat, dh, bits, rstd, m1, m2);
                }
            }
            if (walk == 0) row_sums<1024>(s, 64, slots, turn);
        }
    }
}

// dgamma, dbeta of one unit of columns over the strip blockIdx.y of the rows, one partial row per strip
template <typename T, typename H, bool SUM>
__global__ __launch_bounds__(256) void k_norm_bwd_cols_long(NormBwdArgs a) {
    const int unit = blockIdx.x * 256 + threadIdx.x, count = unit_count<2>(a.C, unit);
    if (count == 0) return;
    const int width = (a.C + kUnit - 1) / kUnit * kUnit;
    const long long c = static_cast<long long>(unit) * kUnit;
    float dg[kUnit] = {}, db[kUnit] = {}, h[kUnit], g[kUnit];
    DropKey key = {0, 0, 0, 0};
    if constexpr (SUM)
        if (a.drop.threshold) key = drop_key(a.drop);
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        load_unit<H, 2>(static_cast<const typename H::store*>(a.h) + row * a.h_ld + c, count, h);
        if constexpr (SUM) {
            const Raw<T> x = load_raw<T, 2>(static_cast<const typename T::store*>(a.x) + row * a.x_ld + c, true, count);
            sum_again<T, 2>(a, key, row, unit, count, x, h);
        }
        load_unit<T, 2>(static_cast<const typename T::store*>(a.dy) + row * a.dy_ld + c, count, g);
        const float mean = a.mean[row], rstd = a.rstd[row];
#pragma unroll
        for (int j = 0; j < kUnit; ++j) {
            dg[j] += g[j] * ((h[j] - mean) * rstd);
            db[j] += g[j];
        }
    }
    float* out = a.partial + static_cast<long long>(blockIdx.y) * 2 * width + c;
    store_n<F32, 8>(out, dg);
    store_n<F32, 8>(out + width, db);
}

}  // namespace

// ---- host side ---------------------------------------------------------------------------------------------------------------
inline int row_ops_cus() {
    static const int n_cu = [] {
        int dev = 0, n = 0;
        if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        return n;
    }();
    return n_cu;
}

// How a row's units are dealt: NV units per lane; threads > 0: a workgroup of that many shares the row; 0: 1 << lane_bits lanes of a
// wavefront do, in workgroups of 256; nv 0: long rows (1024 threads).
struct NormShape {
    int nv, threads, lane_bits;
    int per_block() const { return threads || !nv ? 1 : 256 >> lane_bits; }          // rows of one pass of a workgroup
    int block() const { return threads ? threads : nv ? 256 : 1024; }
};
inline NormShape norm_shape(int C) {
    const int units = (C + kUnit - 1) / kUnit;
    if (units <= 128) {
        int bits = 0;
        while (bits < 6 && (1 << bits) < units) ++bits;
        return {units <= 64 ? 1 : 2, 0, bits};
    }
    if (units <= 256) return {1, 256, 0};
    if (units <= 512) return {2, 256, 0};
    if (units <= 1024) return {2, 512, 0};
    return {0, 0, 0};
}
// at most `most` workgroups, each with as many passes as the others or one less
inline int even_blocks(int64_t passes, int64_t most) {
    const int64_t rounds = (passes + most - 1) / most;
    return static_cast<int>((passes + rounds - 1) / rounds);
}
// Workgroups per CU.  More of them than it takes to keep memory busy cost: the streams' pages are spread wider (forward, 64 fp32
// columns: 44 us with 2, 48 with 8 for 480,000 rows), and every workgroup of the backward pass leaves a partial row (4096 bf16
// columns, 8192 rows: 44 us with 1, 55 with 4).  Forward: 512 lanes with 32 bytes or 1024 with 16 (4096 bf16 columns: 36 us with
// 1 workgroup, 24 with 4; 101 fp32, joined: 57 with 2, 60 with 4); half as many again for ragged 16-bit rows of one unit a lane, which
// are bound by their arithmetic (30 million bf16 values, us with 4, 6, 8 workgroups, alone and joined: 9 columns 44 41 49, 95 81 92;
// 35: 44 39 48, 99 86 94; 133: 48 40 46, 113 99 101; 301: 45 38 43, 105 94 97; 501: 31 27 32, 69 61 67; rows of a workgroup, 1101: 49 40 36,
// 94 83 84; 2001: 32 27 29, 60 58 63; fewer than 4 are slower throughout).  Backward, whose next row is on its
// way already: 16 KB of each tensor in flight where wavefronts hold the rows (bf16, 64 columns: 73 us with 1, 39 with 4, 44 with 8), 8 KB
// where workgroups do.
inline int norm_fwd_per_cu(const NormShape& s, int C, int unit_bytes) {
    const int n = 16384 / unit_bytes / s.block();
    return n < 2 ? 2 : C % kUnit && s.nv == 1 && unit_bytes == 16 ? n + n / 2 : n;
}
inline int norm_bwd_per_cu(const NormShape& s, int C, int unit_bytes) {
    const int n = (C % kUnit && s.threads ? 2 : 1) * (s.threads ? 8192 : 16384) / (s.block() * s.nv * unit_bytes);
    return n < 1 ? 1 : n;
}
// workgroups of the backward pass = partial rows of dgamma / dbeta; unit_bytes: of the wider of the tensors (the largest for a workspace)
inline int norm_bwd_blocks(int64_t rows, int C, int unit_bytes) {
    const NormShape s = norm_shape(C);
    if (s.nv == 0) {                                                         // strips of rows of the columns' kernel
        const int64_t most = row_ops_cus() * 4 / ((C + 256 * kUnit - 1) / (256 * kUnit));
        return static_cast<int>(rows < 8 ? rows : most < 8 ? 8 : rows < most ? rows : most);
    }
    const int64_t passes = (rows + s.per_block() - 1) / s.per_block();
    if (passes <= 8) return 1;                                               // one workgroup writes the results itself
    return even_blocks(passes, static_cast<int64_t>(row_ops_cus()) * norm_bwd_per_cu(s, C, unit_bytes));
}
inline int64_t norm_bwd_workspace_floats(int64_t rows, int C) {
    const int blocks = norm_bwd_blocks(rows, C, 16);
    if (blocks == 1 && norm_shape(C).nv) return 0;
    return static_cast<int64_t>(blocks) * 2 * ((C + kUnit - 1) / kUnit * kUnit);
}

void norm_finish(const NormBwdArgs& a, int blocks, hipStream_t stream);          // layer_norm.hip

namespace {

template <typename T, typename S, bool JOIN, int RAGGED, typename Run>
void norm_fwd_pick(const NormShape& s, Run run) {
    if (s.threads == 0)
        s.nv == 1 ? run(k_norm_fwd<T, S, JOIN, 1, 0, RAGGED ? 1 : 0>) : run(k_norm_fwd<T, S, JOIN, 2, 0, RAGGED>);
    else if (s.threads == 256)
        s.nv == 1 ? run(k_norm_fwd<T, S, JOIN, 1, 256, RAGGED>) : run(k_norm_fwd<T, S, JOIN, 2, 256, RAGGED>);
    else
        run(k_norm_fwd<T, S, JOIN, 2, 512, RAGGED>);
}
template <typename T, typename S, bool JOIN>
void norm_fwd_launch(NormFwdArgs a, hipStream_t stream) {
    const NormShape s = norm_shape(a.C);
    a.lane_bits = s.lane_bits;
    const int64_t passes = (static_cast<int64_t>(a.rows) + s.per_block() - 1) / s.per_block();
    const int per_cu = norm_fwd_per_cu(s, a.C, kUnit * sizeof(typename S::store));
    const dim3 grid(even_blocks(passes, static_cast<int64_t>(row_ops_cus()) * per_cu)), block(s.block());
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); };
    if (s.nv == 0)
        run(k_norm_fwd_long<T, S, JOIN>);
    else if (a.C < kUnit)
        run(k_norm_fwd<T, S, JOIN, 1, 0, 3>);
    else
        a.C % kUnit ? norm_fwd_pick<T, S, JOIN, 2>(s, run) : norm_fwd_pick<T, S, JOIN, 0>(s, run);
}

template <typename T, typename S, bool JOIN, bool SUM, int RAGGED, typename Run>
void norm_bwd_pick(const NormShape& s, Run run) {
    if (s.threads == 0)
        s.nv == 1 ? run(k_norm_bwd<T, S, JOIN, 1, 0, RAGGED ? 1 : 0, SUM>) : run(k_norm_bwd<T, S, JOIN, 2, 0, RAGGED, SUM>);
    else if (s.threads == 256)
        s.nv == 1 ? run(k_norm_bwd<T, S, JOIN, 1, 256, RAGGED, SUM>) : run(k_norm_bwd<T, S, JOIN, 2, 256, RAGGED, SUM>);
    else
        run(k_norm_bwd<T, S, JOIN, 2, 512, RAGGED, SUM>);
}
template <typename T, typename S, bool JOIN, bool SUM = false>
void norm_bwd_launch(NormBwdArgs a, hipStream_t stream) {
    typedef typename std::conditional<JOIN, S, T>::type H;
    const NormShape s = norm_shape(a.C);
    a.lane_bits = s.lane_bits;
    const bool sums = a.dgamma || a.dbeta;
    const int blocks = norm_bwd_blocks(a.rows, a.C, kUnit * sizeof(typename S::store));
    if (!sums) a.partial = nullptr;
    if (s.nv == 0) {
        const int units = (a.C + kUnit - 1) / kUnit, most = 2 * row_ops_cus();
        hipLaunchKernelGGL((k_norm_bwd_long<T, S, JOIN, SUM>), dim3(a.rows < most ? a.rows : most), dim3(1024), 0, stream, a);
        if (!sums) return;
        hipLaunchKernelGGL((k_norm_bwd_cols_long<T, H, SUM>), dim3(ceil_div(units, 256), blocks), dim3(256), 0, stream, a);
        norm_finish(a, blocks, stream);
        return;
    }
    const dim3 grid(blocks), block(s.block());
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); };
    if (a.C < kUnit)
        run(k_norm_bwd<T, S, JOIN, 1, 0, 3, SUM>);
    else
        a.C % kUnit ? norm_bwd_pick<T, S, JOIN, SUM, 2>(s, run) : norm_bwd_pick<T, S, JOIN, SUM, 0>(s, run);
    if (sums && blocks > 1) norm_finish(a, blocks, stream);
}

}  // namespace
}  // namespace fiery
