// Layer norm alone: entry points, and the sum of the partial dgamma / dbeta rows.  The kernels: layer_norm_kernel.h.
#include "layer_norm_kernel.h"

namespace fiery {
namespace {

// dgamma / dbeta = the sum of the workgroups' partial rows, 16 columns at a time per workgroup: lane group r adds rows r, r + 64, ... in
// double, then the 64 sums are added pairwise.  A fixed order: the same inputs give the same bits.
__global__ __launch_bounds__(1024) void k_norm_finish(const float* __restrict__ partial, int blocks, int C, int width, void* dgamma, void* dbeta, int type) {
    __shared__ double lds[64][16];
    const int col = threadIdx.x & 15, r = threadIdx.x >> 4;
    void* out = blockIdx.y ? dbeta : dgamma;
    for (long long first = static_cast<long long>(blockIdx.x) * 16; first < C; first += static_cast<long long>(gridDim.x) * 16) {
        const long long c = first + col;
        double s = 0.0;
        if (c < C) {
            const float* p = partial + static_cast<long long>(blockIdx.y) * width + c;
#pragma unroll 8
            for (int b = r; b < blocks; b += 64) s += p[static_cast<long long>(b) * 2 * width];
        }
        lds[r][col] = s;
        for (int m = 32; m > 0; m >>= 1) {
            __syncthreads();
            if (r < m) lds[r][col] += lds[r + m][col];
        }
        if (r == 0 && c < C && out) store_typed(out, type, c, static_cast<float>(lds[0][col]));
        __syncthreads();                                                   // (the next columns' sums go where these were read)
    }
}

const char* norm_check(int64_t rows, int C, int x_type, int param_type, bool params) {
    if (rows <= 0 || rows >= (1ll << 31) || C <= 0 || C > (1 << 30)) return "bad shape";
    if (!row_type(x_type)) return "unknown element type";
    if (params && param_type != FIERY_TYPE_F32 && param_type != x_type) return "parameters are fp32 or of the rows' type";
    return nullptr;
}

}  // namespace

void norm_finish(const NormBwdArgs& a, int blocks, hipStream_t stream) {
    const int width = (a.C + kUnit - 1) / kUnit * kUnit;
    const int groups = ceil_div(a.C, 16), most = 8 * row_ops_cus();        // (a launch has fewer than 2^32 work-items: 2^26 columns would pass that)
    hipLaunchKernelGGL(k_norm_finish, dim3(groups < most ? groups : most, 2), dim3(1024), 0, stream, a.partial, blocks, a.C, width, a.dgamma, a.dbeta, a.param_type);
}

}  // namespace fiery

using namespace fiery;

extern "C" int fiery_layer_norm_fwd(const void* x, int64_t x_ld, int x_type, int64_t rows, int C, const void* gamma, const void* beta, int param_type,
                                    float eps, void* y, int64_t y_ld, float* mean, float* rstd, fiery_stream_t stream) {
    FIERY_REQUIRE(x && y && !mean == !rstd, "layer_norm_fwd: null pointer");
    const char* bad = norm_check(rows, C, x_type, param_type, gamma || beta);
    FIERY_REQUIRE(!bad, "layer_norm_fwd: %s", bad);
    FIERY_REQUIRE(x_ld >= 0 && y_ld >= C, "layer_norm_fwd: bad row stride");
    NormFwdArgs a = {};
    a.x = x;
    a.gamma = gamma;
    a.beta = beta;
    a.y = y;
    a.mean = mean;
    a.rstd = rstd;
    a.x_ld = x_ld;
    a.y_ld = y_ld;
    a.rows = static_cast<int>(rows);
    a.C = C;
    a.param_type = param_type;
    a.eps = eps;
    a.inv_c = 1.f / static_cast<float>(C);
    if (x_type == FIERY_TYPE_F32)
        norm_fwd_launch<F32, F32, false>(a, as_stream(stream));
    else if (x_type == FIERY_TYPE_BF16)
        norm_fwd_launch<BF16, BF16, false>(a, as_stream(stream));
    else
        norm_fwd_launch<F16, F16, false>(a, as_stream(stream));
    return check_launch("layer_norm_fwd");
}

extern "C" int64_t fiery_layer_norm_bwd_workspace_floats(int64_t rows, int C) {
    return rows > 0 && rows < (1ll << 31) && C > 0 && C <= (1 << 30) ? norm_bwd_workspace_floats(rows, C) : 0;
}

extern "C" int fiery_layer_norm_bwd(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, int x_type, int64_t rows, int C, const void* gamma,
                                    int param_type, const float* mean, const float* rstd, void* dx, int64_t dx_ld, void* dgamma, void* dbeta,
                                    float* workspace, int64_t workspace_floats, fiery_stream_t stream) {
    FIERY_REQUIRE(dy && x && mean && rstd && (dx || dgamma || dbeta), "layer_norm_bwd: null pointer");
    const char* bad = norm_check(rows, C, x_type, param_type, gamma || dgamma || dbeta);
    FIERY_REQUIRE(!bad, "layer_norm_bwd: %s", bad);
    FIERY_REQUIRE(x_ld >= 0 && dy_ld >= 0 && (!dx || dx_ld >= C), "layer_norm_bwd: bad row stride");
    if ((dgamma || dbeta) && norm_bwd_workspace_floats(rows, C) > 0) {
        FIERY_REQUIRE(workspace, "layer_norm_bwd: null workspace");
        if (workspace_floats < norm_bwd_workspace_floats(rows, C)) return fail(FIERY_ENOMEM, "layer_norm_bwd: workspace too small");
    }
    NormBwdArgs a = {};
    a.dy = dy;
    a.h = x;
    a.gamma = gamma;
    a.mean = mean;
    a.rstd = rstd;
    a.dx = dx;
    a.partial = workspace;
    a.dgamma = dgamma;
    a.dbeta = dbeta;
    a.dy_ld = dy_ld;
    a.h_ld = x_ld;
    a.dx_ld = dx_ld;
    a.rows = static_cast<int>(rows);
    a.C = C;
    a.param_type = param_type;
    a.inv_c = 1.f / static_cast<float>(C);
    if (x_type == FIERY_TYPE_F32)
        norm_bwd_launch<F32, F32, false>(a, as_stream(stream));
    else if (x_type == FIERY_TYPE_BF16)
        norm_bwd_launch<BF16, BF16, false>(a, as_stream(stream));
    else
        norm_bwd_launch<F16, F16, false>(a, as_stream(stream));
    return check_launch("layer_norm_bwd");
}
