// Layer norm and RMS norm over the last axis, forward and backward, with the residual sum and dropout that stand before
// them in a transformer's sub-layer:
//     v = [residual +] dropout(x)                     (x alone: a plain norm; residual alone: a sum that was kept)
//     layer: xh = (v - mean v) * r,  r = (mean (v - mean v)^2 + eps)^-1/2        RMS: xh = v * r,  r = (mean v^2 + eps)^-1/2
//     y = xh * w + b
// Backward, g = dy * w:
//     dv = r * (g - mean g - xh * mean(g xh)) [+ dsum]       (RMS: without mean g)
//     dresidual = dv,  dx = kept ? dv / (1 - p) : 0,  dw = sum over rows of dy * xh,  db = sum over rows of dy
// Everything is fp32 between load and store; v is never rounded in between.  Bound by memory: a forward pass reads x (and the
// residual) and writes y (and the sum), a backward pass reads dy, x (and residual, or the sum instead of both) and writes dv.
#include <algorithm>

#include "norm_rows.h"

namespace tvae {
namespace {

// dw, and db where blockIdx.y = 1 or there is no dw: the partial sums added in a fixed order, in fp64; COLS columns by
// 1024 / COLS chunk lanes
template <typename W, int COLS>
__global__ __launch_bounds__(1024) void norm_param_final_kernel(const float* part, int chunks, int d, int first, W* dw, W* db) {
    constexpr int LANES = 1024 / COLS, UNROLL = COLS == 64 ? 8 : 4;
    __shared__ double sm[LANES][COLS + 1];
    const bool second = blockIdx.y || !dw;
    W* out = second ? db : dw;
    const float* p = part + (second ? (long long)chunks * d : 0);
    const int cx = threadIdx.x % COLS, ry = threadIdx.x / COLS;
    const long long col = (long long)(first + blockIdx.x) * COLS + cx;
    double s = 0.0;
    if (col < d) {
#pragma unroll UNROLL
        for (int k = ry; k < chunks; k += LANES) s += (double)p[(long long)k * d + col];
    }
    sm[ry][cx] = s;
    __syncthreads();
    if (LANES > 16) {                            // sixteen lanes a column take four each
        if (ry < 16) sm[ry][cx] = (s + sm[ry + LANES / 4][cx]) + (sm[ry + LANES / 2][cx] + sm[ry + 3 * LANES / 4][cx]);
        __syncthreads();
    }
    if (ry == 0 && col < d) {
        s = 0.0;
#pragma unroll
        for (int k = 0; k < 16; ++k) s += sm[k][cx];
        out[col] = from_f32<W>((float)s);
    }
}

int norm_dispatch(const NormCall& c, int dtype, int r_dtype, bool bwd, hipStream_t s) {
    if (dtype == TVAE_F32) return norm_launch_f32(c, bwd, s);
    return dtype == TVAE_BF16 ? norm_launch_bf16(c, r_dtype, bwd, s) : norm_launch_f16(c, r_dtype, bwd, s);
}

template <typename W, int COLS>
int norm_params_launch(const NormCall& c, hipStream_t s) {
    W *dw = static_cast<W*>(c.dw), *db = static_cast<W*>(c.db);
    const int blocks = (c.d + COLS - 1) / COLS;
    constexpr int MOST = 1 << 21;               // a launch has less than 2^32 threads
    for (int first = 0; first < blocks; first += MOST) {
        const int n = blocks - first < MOST ? blocks - first : MOST;
        hipLaunchKernelGGL((norm_param_final_kernel<W, COLS>), dim3((unsigned)n, dw && db ? 2 : 1), dim3(1024), 0, s, c.part, c.chunks, c.d, first, dw, db);
        TVAE_CHECK_HIP(hipGetLastError());
    }
    return TVAE_OK;
}
// Long rows: 64 columns a workgroup, 256 bytes of every partial sum.  Short ones would leave most of the card idle then.
template <typename W>
int norm_params(const NormCall& c, hipStream_t s) {
    return c.d >= 8192 ? norm_params_launch<W, 64>(c, s) : norm_params_launch<W, 16>(c, s);
}

// what both directions check and fill in
int norm_call(const char* what, int kind, const void* x, int64_t x_so, int64_t x_si, const void* residual, int64_t res_so,
              int64_t res_si, int64_t grp, double p, const int64_t* rng, uint64_t seed, uint64_t offset, int64_t rows, int64_t d,
              int dtype, int w_dtype, int r_dtype, NormCall* c) {
    TVAE_REQUIRE(kind == TVAE_NORM_LAYER || kind == TVAE_NORM_RMS, "%s: unknown norm %d", what, kind);
    TVAE_REQUIRE(norm_dtype_ok(dtype), "%s: unknown dtype %d", what, dtype);
    TVAE_REQUIRE(w_dtype == dtype || w_dtype == TVAE_F32, "%s: weights are of x's type or fp32, got %d", what, w_dtype);
    TVAE_REQUIRE(r_dtype == dtype || r_dtype == TVAE_F32, "%s: the residual is of x's type or fp32, got %d", what, r_dtype);
    TVAE_REQUIRE(x || residual, "%s: null pointer argument", what);
    TVAE_REQUIRE(rows > 0 && d > 0 && rows < (1ll << 31) && d < (1ll << 31), "%s: bad shape rows=%lld d=%lld", what, (long long)rows, (long long)d);
    TVAE_REQUIRE(grp > 0 && rows % grp == 0, "%s: %lld rows are not groups of %lld", what, (long long)rows, (long long)grp);
    TVAE_REQUIRE(dropout_args(p, rng, seed, offset, &c->drop), "%s: p = %g is not a probability", what, p);
    c->x = x; c->residual = residual;
    c->x_rows = RowsOf{x_so, x_si}; c->res_rows = RowsOf{res_so, res_si};
    c->grp = (int)grp; c->d = (int)d; c->inv_d = 1.f / (float)d; c->groups = (int)((d + 7) / 8); c->rows = rows;
    c->w_f32 = w_dtype == TVAE_F32; c->rms = kind == TVAE_NORM_RMS;
    return TVAE_OK;
}

}  // namespace
}  // namespace tvae

using namespace tvae;

extern "C" int tvae_norm_fwd(int kind, const void* x, int64_t x_so, int64_t x_si, const void* residual, int64_t res_so, int64_t res_si,
                             int64_t grp, const void* weight, const void* bias, double eps, double p, const int64_t* rng, uint64_t seed,
                             uint64_t offset, void* y, void* sum, float* mean, float* rstd, int64_t rows, int64_t d, int dtype,
                             int w_dtype, int r_dtype, void* stream) {
    NormCall c{};
    TVAE_PROPAGATE(norm_call("norm_fwd", kind, x, x_so, x_si, residual, res_so, res_si, grp, p, rng, seed, offset, rows, d, dtype, w_dtype, r_dtype, &c));
    TVAE_REQUIRE(y, "norm_fwd: null pointer argument");
    TVAE_REQUIRE(eps >= 0.0 && eps < 1e30, "norm_fwd: eps = %g is not a finite number >= 0", eps);
    TVAE_REQUIRE(c.rms ? !mean : (!rstd) == (!mean), "norm_fwd: mean and rstd are both given or neither (RMS norm: rstd alone)");
    TVAE_REQUIRE(!(c.rms && bias), "norm_fwd: RMS norm has no bias");
    c.weight = weight; c.bias = bias; c.eps = (float)eps;
    c.y = y; c.sum = sum; c.mean = mean; c.rstd = rstd;
    return norm_dispatch(c, dtype, r_dtype, false, static_cast<hipStream_t>(stream));
}

extern "C" int64_t tvae_norm_bwd_workspace_bytes(int64_t rows, int64_t d) {
    if (rows <= 0 || d <= 0 || rows >= (1ll << 31) || d >= (1ll << 31)) return -1;
    if (bwd_small(rows, d)) return 0;
    return 2 * std::max(bwd_chunks(rows, d, false), bwd_chunks(rows, d, true)) * d * 4;
}

extern "C" int tvae_norm_bwd(int kind, const void* dy, int64_t dy_so, int64_t dy_si, const void* dsum, int64_t ds_so, int64_t ds_si,
                             const void* x, int64_t x_so, int64_t x_si, const void* residual, int64_t res_so, int64_t res_si, int64_t grp,
                             const void* weight, const float* mean, const float* rstd, double p, const int64_t* rng, uint64_t seed,
                             uint64_t offset, void* dx, void* dresidual, void* dweight, void* dbias, int64_t rows, int64_t d, int dtype,
                             int w_dtype, int r_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    NormCall c{};
    TVAE_PROPAGATE(norm_call("norm_bwd", kind, x, x_so, x_si, residual, res_so, res_si, grp, p, rng, seed, offset, rows, d, dtype, w_dtype, r_dtype, &c));
    TVAE_REQUIRE(dy && rstd, "norm_bwd: null pointer argument");
    TVAE_REQUIRE(c.rms ? !mean && !dbias : mean != nullptr, "norm_bwd: layer norm needs mean, RMS norm has neither mean nor bias");
    if (!(dx || dresidual || dweight || dbias)) return TVAE_OK;
    if ((dweight || dbias) && !bwd_small(rows, d))
        TVAE_REQUIRE(workspace && workspace_bytes >= tvae_norm_bwd_workspace_bytes(rows, d), "norm_bwd: workspace of %lld bytes, %lld needed",
                     (long long)workspace_bytes, (long long)tvae_norm_bwd_workspace_bytes(rows, d));
    c.weight = weight; c.mean = const_cast<float*>(mean); c.rstd = const_cast<float*>(rstd);
    c.dy = dy; c.dsum = dsum; c.dy_rows = RowsOf{dy_so, dy_si}; c.ds_rows = RowsOf{ds_so, ds_si};
    c.dx = dx; c.dres = dresidual; c.dw = dweight; c.db = dbias; c.part = static_cast<float*>(workspace);
    c.chunks = (int)bwd_chunks(rows, d, r_dtype != TVAE_F32);
    hipStream_t s = static_cast<hipStream_t>(stream);
    TVAE_PROPAGATE(norm_dispatch(c, dtype, r_dtype, true, s));
    if (!(dweight || dbias) || bwd_small(rows, d)) return TVAE_OK;
    return w_dtype == TVAE_F32 ? norm_params<float>(c, s) : w_dtype == TVAE_BF16 ? norm_params<bf16>(c, s) : norm_params<f16>(c, s);
}
