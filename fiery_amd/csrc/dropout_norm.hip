// Residual + dropout + layer norm in one pass each way: entry points.  The kernels: layer_norm_kernel.h (JOIN).
#include "layer_norm_kernel.h"

namespace fiery {
namespace {

// The stream (residual, h and their gradients) is of the rows' type or fp32.
template <typename Launch>
void by_types(int x_type, int stream_type, Launch launch) {
    if (x_type == FIERY_TYPE_F32)
        launch(F32(), F32());
    else if (x_type == FIERY_TYPE_BF16)
        stream_type == FIERY_TYPE_F32 ? launch(BF16(), F32()) : launch(BF16(), BF16());
    else
        stream_type == FIERY_TYPE_F32 ? launch(F16(), F32()) : launch(F16(), F16());
}

const char* join_check(int64_t rows, int C, int x_type, int stream_type, int param_type, bool params) {
    if (rows <= 0 || rows >= (1ll << 31) || C <= 0 || C > (1 << 30)) return "bad shape";
    if (!row_type(x_type)) return "unknown element type";
    if (stream_type != FIERY_TYPE_F32 && stream_type != x_type) return "the residual is fp32 or of the rows' type";
    if (params && param_type != FIERY_TYPE_F32 && param_type != x_type) return "parameters are fp32 or of the rows' type";
    return nullptr;
}

int join_fwd(const void* x, int64_t x_ld, int x_type, const void* residual, int64_t res_ld, int stream_type, int64_t rows, int C, const void* gamma,
             const void* beta, int param_type, float eps, int threshold, const int64_t* rng, int64_t call, int64_t rows_per_mask, int one_column,
             int64_t* rng_used, void* y, int64_t y_ld, void* h, int64_t h_ld, float* mean, float* rstd, bool of_sum, fiery_stream_t stream) {
    FIERY_REQUIRE(x && residual && y && h && !mean == !rstd, "dropout_add_layer_norm_fwd: null pointer");
    NormFwdArgs a = {};
    const char* bad = join_check(rows, C, x_type, stream_type, param_type, gamma || beta);
    if (!bad) bad = drop_args(a.drop, rng, rng_used, call, threshold, rows_per_mask, one_column);
    FIERY_REQUIRE(!bad, "dropout_add_layer_norm_fwd: %s", bad);
    FIERY_REQUIRE(x_ld >= 0 && res_ld >= 0 && y_ld >= C && h_ld >= C, "dropout_add_layer_norm_fwd: bad row stride");
    a.x = x;
    a.residual = residual;
    a.gamma = gamma;
    a.beta = beta;
    a.y = y;
    a.h = h;
    a.mean = mean;
    a.rstd = rstd;
    a.x_ld = x_ld;
    a.res_ld = res_ld;
    a.y_ld = y_ld;
    a.h_ld = h_ld;
    a.rows = static_cast<int>(rows);
    a.C = C;
    a.param_type = param_type;
    a.eps = eps;
    a.of_sum = of_sum;
    a.inv_c = 1.f / static_cast<float>(C);
    by_types(x_type, stream_type, [&](auto t, auto s) { norm_fwd_launch<decltype(t), decltype(s), true>(a, as_stream(stream)); });
    return check_launch("dropout_add_layer_norm_fwd");
}

// x null: h is read as it is stored; otherwise it is made again from x and the residual
int join_bwd(const void* dy, int64_t dy_ld, const void* dh, int64_t dh_ld, const void* x, int64_t x_ld, const void* h, int64_t h_ld, int x_type, int stream_type,
             int64_t rows, int C, const void* gamma, int param_type, const float* mean, const float* rstd, int threshold, const int64_t* rng_used,
             int64_t rows_per_mask, int one_column, void* dx, int64_t dx_ld, void* dresidual, int64_t dres_ld, void* dgamma, void* dbeta, float* workspace,
             int64_t workspace_floats, fiery_stream_t stream) {
    const bool h_alone = !dy;                                              // only h went on: dx is the dropout of dh, dresidual is dh itself
    FIERY_REQUIRE(h_alone ? dh && dx && !dresidual && !dgamma && !dbeta : h && mean && rstd && (dx || dresidual || dgamma || dbeta),
                  "dropout_add_layer_norm_bwd: null pointer");
    NormBwdArgs a = {};
    const char* bad = join_check(rows, C, x_type, stream_type, param_type, gamma || dgamma || dbeta);
    if (!bad) bad = drop_args(a.drop, rng_used, nullptr, 0, threshold, rows_per_mask, one_column);
    FIERY_REQUIRE(!bad, "dropout_add_layer_norm_bwd: %s", bad);
    FIERY_REQUIRE(dy_ld >= 0 && h_ld >= 0 && x_ld >= 0 && (!dh || dh_ld >= 0) && (!dx || dx_ld >= C) && (!dresidual || dres_ld >= C),
                  "dropout_add_layer_norm_bwd: bad row stride");
    if (h_alone) {
        DropoutArgs d = {};
        d.x = dh;
        d.y = dx;
        d.x_ld = dh_ld;
        d.y_ld = dx_ld;
        d.C = C;
        d.drop = a.drop;
        dropout_rows(d, rows, stream_type, x_type, as_stream(stream));
        return check_launch("dropout_add_layer_norm_bwd");
    }
    if ((dgamma || dbeta) && norm_bwd_workspace_floats(rows, C) > 0) {
        FIERY_REQUIRE(workspace, "dropout_add_layer_norm_bwd: null workspace");
        if (workspace_floats < norm_bwd_workspace_floats(rows, C)) return fail(FIERY_ENOMEM, "dropout_add_layer_norm_bwd: workspace too small");
    }
    a.dy = dy;
    a.dh = dh;
    a.h = h;
    a.x = x;
    a.gamma = gamma;
    a.mean = mean;
    a.rstd = rstd;
    a.dx = dx;
    a.dres = dresidual;
    a.partial = workspace;
    a.dgamma = dgamma;
    a.dbeta = dbeta;
    a.dy_ld = dy_ld;
    a.dh_ld = dh_ld;
    a.h_ld = h_ld;
    a.x_ld = x_ld;
    a.dx_ld = dx_ld;
    a.dres_ld = dres_ld;
    a.rows = static_cast<int>(rows);
    a.C = C;
    a.param_type = param_type;
    a.inv_c = 1.f / static_cast<float>(C);
    if (!x)
        by_types(x_type, stream_type, [&](auto t, auto s) { norm_bwd_launch<decltype(t), decltype(s), true>(a, as_stream(stream)); });
    else if (x_type == FIERY_TYPE_BF16)
        norm_bwd_launch<BF16, BF16, true, true>(a, as_stream(stream));
    else
        norm_bwd_launch<F16, F16, true, true>(a, as_stream(stream));
    return check_launch("dropout_add_layer_norm_bwd");
}

}  // namespace
}  // namespace fiery

using namespace fiery;

extern "C" int fiery_dropout_add_layer_norm_fwd(const void* x, int64_t x_ld, int x_type, const void* residual, int64_t res_ld, int stream_type, int64_t rows,
                                                int C, const void* gamma, const void* beta, int param_type, float eps, int threshold, const int64_t* rng,
                                                int64_t call, int64_t rows_per_mask, int one_column, int64_t* rng_used, void* y, int64_t y_ld, void* h,
                                                int64_t h_ld, float* mean, float* rstd, fiery_stream_t stream) {
    return join_fwd(x, x_ld, x_type, residual, res_ld, stream_type, rows, C, gamma, beta, param_type, eps, threshold, rng, call, rows_per_mask, one_column,
                    rng_used, y, y_ld, h, h_ld, mean, rstd, false, stream);
}

extern "C" int fiery_dropout_add_layer_norm_fwd_unrounded(const void* x, int64_t x_ld, int x_type, const void* residual, int64_t res_ld, int stream_type, int64_t rows,
                                                          int C, const void* gamma, const void* beta, int param_type, float eps, int threshold, const int64_t* rng,
                                                          int64_t call, int64_t rows_per_mask, int one_column, int64_t* rng_used, void* y, int64_t y_ld, void* h,
                                                          int64_t h_ld, float* mean, float* rstd, fiery_stream_t stream) {
    return join_fwd(x, x_ld, x_type, residual, res_ld, stream_type, rows, C, gamma, beta, param_type, eps, threshold, rng, call, rows_per_mask, one_column,
                    rng_used, y, y_ld, h, h_ld, mean, rstd, true, stream);
}

extern "C" int fiery_dropout_add_layer_norm_bwd(const void* dy, int64_t dy_ld, const void* dh, int64_t dh_ld, const void* h, int64_t h_ld, int x_type,
                                                int stream_type, int64_t rows, int C, const void* gamma, int param_type, const float* mean,
                                                const float* rstd, int threshold, const int64_t* rng_used, int64_t rows_per_mask, int one_column,
                                                void* dx, int64_t dx_ld, void* dresidual, int64_t dres_ld, void* dgamma, void* dbeta, float* workspace,
                                                int64_t workspace_floats, fiery_stream_t stream) {
    return join_bwd(dy, dy_ld, dh, dh_ld, nullptr, 0, h, h_ld, x_type, stream_type, rows, C, gamma, param_type, mean, rstd, threshold, rng_used, rows_per_mask,
                    one_column, dx, dx_ld, dresidual, dres_ld, dgamma, dbeta, workspace, workspace_floats, stream);
}

extern "C" int fiery_dropout_add_layer_norm_bwd_unrounded(const void* dy, int64_t dy_ld, const void* dh, int64_t dh_ld, const void* x, int64_t x_ld,
                                                          const void* residual, int64_t res_ld, int type, int64_t rows, int C, const void* gamma,
                                                          int param_type, const float* mean, const float* rstd, int threshold,
                                                          const int64_t* rng_used, int64_t rows_per_mask, int one_column, void* dx, int64_t dx_ld,
                                                          void* dresidual, int64_t dres_ld, void* dgamma, void* dbeta, float* workspace,
                                                          int64_t workspace_floats, fiery_stream_t stream) {
    FIERY_REQUIRE(x, "dropout_add_layer_norm_bwd_unrounded: null pointer");
    FIERY_REQUIRE(type != FIERY_TYPE_F32, "dropout_add_layer_norm_bwd_unrounded: a stream of 16 bits (an fp32 h is not rounded)");
    return join_bwd(dy, dy_ld, dh, dh_ld, x, x_ld, residual, res_ld, type, type, rows, C, gamma, param_type, mean, rstd, threshold, rng_used, rows_per_mask,
                    one_column, dx, dx_ld, dresidual, dres_ld, dgamma, dbeta, workspace, workspace_floats, stream);
}
