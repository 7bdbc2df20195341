// Dropout from a counter-based generator, forward and backward, with a fused residual sum: y = [residual +] (kept ? scale x : 0).
// The mask (row_ops.h) is a function of (seed, call, row, column): nothing of it is stored, the backward pass is the same
// kernel on the gradient without a residual.  Masks per element, per channel of an image (nn.Dropout2d) or per image (the
// trunk's drop-connect) differ only in the row and column that number them.
//
// Memory-bound: x [and the residual] read once, y written once.  The generator costs 20 wide integer multiplications per unit
// of eight columns, beside 16 or 32 bytes in and out.  Units are dealt to lanes flat over (row, unit), so narrow rows fill
// their wavefronts; the split of the flat index is one multiplication.
//
// Measured (one MI355X; a large copy reaches 5.35 TB/s): 16,384 x 4096 bf16 48 us = 5.6 TB/s; 480,000 x 64 fp32 per channel with a
// residual 69 us = 5.4 TB/s, its backward pass 43 us = 5.7 TB/s; 90,720 x 56 fp32 per image 12 us = 5.2 TB/s.
#include "row_ops.h"

namespace fiery {
namespace {

template <typename I, typename O, bool RES, int RAGGED>
__global__ __launch_bounds__(256) void k_dropout(DropoutArgs a) {
    DropKey key = {0, 0, 0, 0};
    if (a.drop.threshold) key = drop_key(a.drop);
    drop_note(a.drop);
    for (unsigned long long q = static_cast<unsigned long long>(blockIdx.x) * 256 + threadIdx.x; q < a.total; q += static_cast<unsigned long long>(gridDim.x) * 256) {
        const unsigned at = div_by(static_cast<unsigned>(q), a.units), row = a.first + at, unit = static_cast<unsigned>(q) - at * a.units.d;
        const long long c = static_cast<long long>(unit) * kUnit;
        const int count = RAGGED ? unit_count<RAGGED>(a.C, unit) : kUnit;
        float v[kUnit];
        load_unit<I, RAGGED>(static_cast<const typename I::store*>(a.x) + row * a.x_ld + c, count, v);
        if constexpr (RES) {
            float r[kUnit];
            load_unit<O, RAGGED>(static_cast<const typename O::store*>(a.residual) + row * a.res_ld + c, count, r);
            drop_unit(a.drop, key, row, unit, v);
#pragma unroll
            for (int j = 0; j < kUnit; ++j) v[j] += r[j];
        } else {
            drop_unit(a.drop, key, row, unit, v);
        }
        store_unit<O, RAGGED>(static_cast<typename O::store*>(a.y) + row * a.y_ld + c, count, v);
    }
}

template <typename I, typename O>
void dropout_launch(const DropoutArgs& a, hipStream_t stream) {
    const dim3 grid(ceil_div(a.total, 256)), block(256);
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, stream, a); };
    if (a.C < kUnit)
        a.residual ? run(k_dropout<I, O, true, 3>) : run(k_dropout<I, O, false, 3>);
    else if (a.C % kUnit)
        a.residual ? run(k_dropout<I, O, true, 1>) : run(k_dropout<I, O, false, 1>);
    else
        a.residual ? run(k_dropout<I, O, true, 0>) : run(k_dropout<I, O, false, 0>);
}

}  // namespace

// (as many launches as keep the flat index below 2^31: a launch's rows start at `first`, which the mask counts too)
void dropout_rows(DropoutArgs a, int64_t rows, int x_type, int y_type, hipStream_t stream) {
    const int64_t units = (static_cast<int64_t>(a.C) + kUnit - 1) / kUnit, most = ((1ll << 31) - 1) / units;
    a.units = fast_div(static_cast<unsigned>(units));
    for (int64_t first = 0; first < rows; first += most) {
        a.first = static_cast<unsigned>(first);
        a.total = static_cast<unsigned>((rows - first < most ? rows - first : most) * units);
        if (first > 0) a.drop.rng_used = nullptr;
        if (x_type == FIERY_TYPE_F32 && y_type == FIERY_TYPE_F32)
            dropout_launch<F32, F32>(a, stream);
        else if (x_type == FIERY_TYPE_BF16 && y_type == FIERY_TYPE_BF16)
            dropout_launch<BF16, BF16>(a, stream);
        else if (x_type == FIERY_TYPE_F16 && y_type == FIERY_TYPE_F16)
            dropout_launch<F16, F16>(a, stream);
        else if (x_type == FIERY_TYPE_BF16)
            dropout_launch<BF16, F32>(a, stream);
        else if (x_type == FIERY_TYPE_F16)
            dropout_launch<F16, F32>(a, stream);
        else if (y_type == FIERY_TYPE_BF16)
            dropout_launch<F32, BF16>(a, stream);
        else
            dropout_launch<F32, F16>(a, stream);
    }
}

}  // namespace fiery

using namespace fiery;

extern "C" int fiery_dropout(const void* x, int64_t x_ld, int x_type, const void* residual, int64_t res_ld, int64_t rows, int C, int threshold,
                             const int64_t* rng, int64_t call, int64_t rows_per_mask, int one_column, int64_t* rng_used, void* y, int64_t y_ld, int y_type,
                             fiery_stream_t stream) {
    FIERY_REQUIRE(x && y, "dropout: null pointer");
    FIERY_REQUIRE(rows > 0 && C > 0 && rows < (1ll << 31), "dropout: bad shape");
    const int64_t units = (static_cast<int64_t>(C) + kUnit - 1) / kUnit;
    FIERY_REQUIRE(rows * units < (1ll << 31), "dropout: over 2^31 units of eight columns in one call");
    FIERY_REQUIRE(row_type(x_type) && row_type(y_type), "dropout: unknown element type");
    FIERY_REQUIRE(x_type == y_type || x_type == FIERY_TYPE_F32 || y_type == FIERY_TYPE_F32, "dropout: bf16 and fp16 do not mix");
    FIERY_REQUIRE(x_ld >= 0 && (!residual || res_ld >= 0) && y_ld >= C, "dropout: bad row stride");
    DropoutArgs a = {};
    const char* bad = drop_args(a.drop, rng, rng_used, call, threshold, rows_per_mask, one_column);
    FIERY_REQUIRE(!bad, "dropout: %s", bad);
    a.x = x;
    a.residual = residual;
    a.y = y;
    a.x_ld = x_ld;
    a.res_ld = res_ld;
    a.y_ld = y_ld;
    a.C = C;
    dropout_rows(a, rows, x_type, y_type, as_stream(stream));
    return check_launch("dropout");
}
