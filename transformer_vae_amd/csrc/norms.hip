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
#include "norm_common.h"

namespace tvae {
namespace {

struct NormCall {
    const void* x; const void* residual;            // at least one; T and R
    RowsOf x_rows, res_rows;
    int grp, d, groups;                             // groups = ceil(d / 8)
    long long rows;
    DropoutArgs drop;
    const void* weight; const void* bias;           // null: 1 and 0
    int w_f32, rms;                                 // weights are fp32 (else T); RMS norm
    float eps;
    float* mean; float* rstd;                       // forward: null in inference.  Backward: given (mean null for RMS)
    void* y; void* sum;                             // forward outputs (T; R, nullable)
    const void* dy; const void* dsum;               // backward: cotangents (T, nullable: 0; R, nullable: 0)
    RowsOf dy_rows, ds_rows;
    void* dx; void* dres;                           // nullable (T; R)
    float* part; int chunks;                        // [2][chunks][d] partial sums of dw and db
    int chunk_rows;
    void* dw; void* db;                             // nullable
};

// sum over the 256 threads of a workgroup, the same bits in every thread
__device__ __forceinline__ float block_sum(float v, float* sm) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

template <typename T>
__device__ __forceinline__ void load8_param(const void* p, int f32, int col, int nv, float fill, float v[8]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fill;
    } else if (f32) {
        load8(static_cast<const float*>(p) + col, nv, v);
    } else {
        load8(static_cast<const T*>(p) + col, nv, v);
    }
}

// the eight values of v that start at column 8 g; columns beyond d are 0
template <typename T, typename R>
__device__ __forceinline__ void value8(const NormCall& c, const Philox& ph, long long row, int g, float v[8]) {
    const int nv = c.d - 8 * g;
    if (c.x) {
        load8(static_cast<const T*>(c.x) + row_offset(c.x_rows, c.grp, row) + 8 * g, nv, v);
        if (c.drop.threshold) drop8(ph, c.drop, (uint32_t)g, (uint32_t)row, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
    if (c.residual) {
        float r[8];
        load8(static_cast<const R*>(c.residual) + row_offset(c.res_rows, c.grp, row) + 8 * g, nv, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
    }
}

// ---- rows of any length: one workgroup per row, the row is read again for every pass over it ----------------------------
template <typename T, typename R>
__global__ __launch_bounds__(256) void norm_fwd_wide_kernel(NormCall c) {
    __shared__ float sm[4];
    const Philox ph(c.drop);
    for (long long row = blockIdx.x; row < c.rows; row += gridDim.x) {
        float mu = 0.f, m2 = 0.f, q = 0.f;
        if (!c.rms) {
            float s = 0.f;
            for (int g = threadIdx.x; g < c.groups; g += 256) {
                float v[8];
                value8<T, R>(c, ph, row, g, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) s += v[e];
            }
            mu = block_sum(s, sm) / (float)c.d;
        }
        // squares about the fp32 mean, with the sum of the deviations beside them: their mean is what rounding left in mu,
        // and taking it out of both keeps rows of equal values at 0 under the smallest eps
        float t1 = 0.f;
        for (int g = threadIdx.x; g < c.groups; g += 256) {
            float v[8];
            value8<T, R>(c, ph, row, g, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float t = 8 * g + e < c.d ? v[e] - mu : 0.f;
                t1 += t;
                q = fmaf(t, t, q);
            }
        }
        q = block_sum(q, sm) / (float)c.d;
        if (!c.rms) {
            m2 = block_sum(t1, sm) / (float)c.d;
            q -= m2 * m2;
            if (q < 0.f) q = 0.f;
        }
        const float rs = rsqrtf(q + c.eps);
        for (int g = threadIdx.x; g < c.groups; g += 256) {
            float v[8], w[8], b[8];
            const int nv = c.d - 8 * g;
            value8<T, R>(c, ph, row, g, v);
            if (c.sum) store8(static_cast<R*>(c.sum) + row * c.d + 8 * g, nv, v);
            load8_param<T>(c.weight, c.w_f32, 8 * g, nv, 1.f, w);
            load8_param<T>(c.bias, c.w_f32, 8 * g, nv, 0.f, b);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(((v[e] - mu) - m2) * rs, w[e], b[e]);
            store8(static_cast<T*>(c.y) + row * c.d + 8 * g, nv, v);
        }
        if (threadIdx.x == 0 && c.rstd) {
            c.rstd[row] = rs;
            if (c.mean) c.mean[row] = mu + m2;
        }
    }
}

template <typename T, typename R>
__global__ __launch_bounds__(256) void norm_bwd_wide_kernel(NormCall c) {
    __shared__ float sm[4];
    const Philox ph(c.drop);
    for (long long row = blockIdx.x; row < c.rows; row += gridDim.x) {
        const float mu = c.mean ? c.mean[row] : 0.f, rs = c.rstd[row];
        const T* dy = static_cast<const T*>(c.dy) + row_offset(c.dy_rows, c.grp, row);
        float s1 = 0.f, s2 = 0.f;
        for (int g = threadIdx.x; g < c.groups; g += 256) {
            float v[8], w[8], u[8];
            const int nv = c.d - 8 * g;
            value8<T, R>(c, ph, row, g, v);
            load8(dy + 8 * g, nv, u);
            load8_param<T>(c.weight, c.w_f32, 8 * g, nv, 1.f, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float gw = u[e] * w[e];
                s1 += gw;
                s2 = fmaf(gw, (v[e] - mu) * rs, s2);
            }
        }
        s2 = block_sum(s2, sm) / (float)c.d;
        s1 = c.rms ? 0.f : block_sum(s1, sm) / (float)c.d;
        for (int g = threadIdx.x; g < c.groups; g += 256) {
            float v[8], w[8], u[8];
            const int nv = c.d - 8 * g;
            value8<T, R>(c, ph, row, g, v);
            load8(dy + 8 * g, nv, u);
            load8_param<T>(c.weight, c.w_f32, 8 * g, nv, 1.f, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = rs * ((u[e] * w[e] - s1) - (v[e] - mu) * rs * s2);
            if (c.dsum) {
                load8(static_cast<const R*>(c.dsum) + row_offset(c.ds_rows, c.grp, row) + 8 * g, nv, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += u[e];
            }
            if (c.dres) store8(static_cast<R*>(c.dres) + row * c.d + 8 * g, nv, v);
            if (c.dx) {
                if (c.drop.threshold) drop8(ph, c.drop, (uint32_t)g, (uint32_t)row, v);
                store8(static_cast<T*>(c.dx) + row * c.d + 8 * g, nv, v);
            }
        }
    }
}

// partial sums of dw and db over chunk_rows rows: 64 groups of columns by 4 row lanes a workgroup
template <typename T, typename R>
__global__ __launch_bounds__(256) void norm_param_wide_kernel(NormCall c) {
    __shared__ float sm[3][64][17];
    const Philox ph(c.drop);
    const int gl = threadIdx.x & 63, ry = threadIdx.x >> 6;
    const int g = blockIdx.x * 64 + gl;
    const long long r0 = (long long)blockIdx.y * c.chunk_rows, r1 = min(c.rows, r0 + c.chunk_rows);
    float aw[8] = {}, ab[8] = {};
    if (g < c.groups) {
        for (long long row = r0 + ry; row < r1; row += 4) {
            float v[8], u[8];
            const float mu = c.mean ? c.mean[row] : 0.f, rs = c.rstd[row];
            value8<T, R>(c, ph, row, g, v);
            load8(static_cast<const T*>(c.dy) + row_offset(c.dy_rows, c.grp, row) + 8 * g, c.d - 8 * g, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                aw[e] = fmaf(u[e], (v[e] - mu) * rs, aw[e]);
                ab[e] += u[e];
            }
        }
    }
    if (ry > 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) { sm[ry - 1][gl][e] = aw[e]; sm[ry - 1][gl][8 + e] = ab[e]; }
    }
    __syncthreads();
    if (ry == 0 && g < c.groups) {
        for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) { aw[e] += sm[k][gl][e]; ab[e] += sm[k][gl][8 + e]; }
        float* pw = c.part + (long long)blockIdx.y * c.d + 8 * g;
        store8(pw, c.d - 8 * g, aw);
        store8(pw + (long long)c.chunks * c.d, c.d - 8 * g, ab);
    }
}

// dw (blockIdx.y = 0) and db (1): the partial sums added in a fixed order, in fp64; 64 columns by 16 chunk lanes
template <typename W>
__global__ __launch_bounds__(1024) void norm_param_final_kernel(const float* part, int chunks, int d, W* dw, W* db) {
    __shared__ double sm[16][64];
    W* out = blockIdx.y ? db : dw;
    if (!out) return;
    const float* p = part + (long long)blockIdx.y * chunks * d;
    const int cx = threadIdx.x & 63, ry = threadIdx.x >> 6;
    const long long col = (long long)blockIdx.x * 64 + cx;
    double s = 0.0;
    if (col < d)
        for (int k = ry; k < chunks; k += 16) s += (double)p[(long long)k * d + col];
    sm[ry][cx] = s;
    __syncthreads();
    if (ry == 0 && col < d) {
        for (int k = 1; k < 16; ++k) s += sm[k][cx];
        out[col] = from_f32<W>((float)s);
    }
}

constexpr int64_t WIDE_CHUNK_ROWS = 64;     // at least; more where that would make over 1024 chunks
inline int64_t wide_chunk_rows(int64_t rows) {
    const int64_t r = (rows + 1023) / 1024;
    return r > WIDE_CHUNK_ROWS ? r : WIDE_CHUNK_ROWS;
}

template <typename T, typename R>
int norm_fwd_launch(const NormCall& c, hipStream_t s) {
    const unsigned blocks = (unsigned)(c.rows < 65536 ? c.rows : 65536);
    hipLaunchKernelGGL((norm_fwd_wide_kernel<T, R>), dim3(blocks), dim3(256), 0, s, c);
    TVAE_CHECK_HIP(hipGetLastError());
    return TVAE_OK;
}

template <typename T, typename R>
int norm_bwd_launch(NormCall c, hipStream_t s) {
    const unsigned blocks = (unsigned)(c.rows < 65536 ? c.rows : 65536);
    if (c.dx || c.dres) {
        hipLaunchKernelGGL((norm_bwd_wide_kernel<T, R>), dim3(blocks), dim3(256), 0, s, c);
        TVAE_CHECK_HIP(hipGetLastError());
    }
    if (c.dw || c.db) {
        c.chunk_rows = (int)wide_chunk_rows(c.rows);
        c.chunks = (int)((c.rows + c.chunk_rows - 1) / c.chunk_rows);
        hipLaunchKernelGGL((norm_param_wide_kernel<T, R>), dim3((unsigned)((c.groups + 63) / 64), (unsigned)c.chunks), dim3(256), 0, s, c);
        TVAE_CHECK_HIP(hipGetLastError());
        const dim3 grid((unsigned)((c.d + 63) / 64), 2);
        if (c.w_f32)
            hipLaunchKernelGGL((norm_param_final_kernel<float>), grid, dim3(1024), 0, s, c.part, c.chunks, c.d, (float*)c.dw, (float*)c.db);
        else
            hipLaunchKernelGGL((norm_param_final_kernel<T>), grid, dim3(1024), 0, s, c.part, c.chunks, c.d, (T*)c.dw, (T*)c.db);
        TVAE_CHECK_HIP(hipGetLastError());
    }
    return TVAE_OK;
}

template <typename F>
int with_types(int dtype, int r_dtype, F&& f) {
    if (dtype == TVAE_F32) return f(float{}, float{});
    if (dtype == TVAE_BF16) return r_dtype == TVAE_F32 ? f(bf16{}, float{}) : f(bf16{}, bf16{});
    return r_dtype == TVAE_F32 ? f(f16{}, float{}) : f(f16{}, f16{});
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
    c->grp = (int)grp; c->d = (int)d; c->groups = (int)((d + 7) / 8); c->rows = rows;
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
    return with_types(dtype, r_dtype, [&](auto t, auto r) { return norm_fwd_launch<decltype(t), decltype(r)>(c, static_cast<hipStream_t>(stream)); });
}

extern "C" int64_t tvae_norm_bwd_workspace_bytes(int64_t rows, int64_t d) {
    if (rows <= 0 || d <= 0 || rows >= (1ll << 31) || d >= (1ll << 31)) return -1;
    const int64_t cr = wide_chunk_rows(rows);
    return 2 * ((rows + cr - 1) / cr) * d * 4;
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
    if (dweight || dbias)
        TVAE_REQUIRE(workspace && workspace_bytes >= tvae_norm_bwd_workspace_bytes(rows, d), "norm_bwd: workspace of %lld bytes, %lld needed",
                     (long long)workspace_bytes, (long long)tvae_norm_bwd_workspace_bytes(rows, d));
    c.weight = weight; c.mean = const_cast<float*>(mean); c.rstd = const_cast<float*>(rstd);
    c.dy = dy; c.dsum = dsum; c.dy_rows = RowsOf{dy_so, dy_si}; c.ds_rows = RowsOf{ds_so, ds_si};
    c.dx = dx; c.dres = dresidual; c.dw = dweight; c.db = dbias; c.part = static_cast<float*>(workspace);
    return with_types(dtype, r_dtype, [&](auto t, auto r) { return norm_bwd_launch<decltype(t), decltype(r)>(c, static_cast<hipStream_t>(stream)); });
}
