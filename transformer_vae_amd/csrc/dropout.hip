// Dropout, alone or added to a residual, with keep decisions that are evaluated and never stored (norm_common.h):
//     out = [residual +] (kept ? in / (1 - p) : 0)
// The backward pass is the same call on the cotangent.  Bound by memory: in + out (+ residual) bytes a pass.
#include <cmath>

#include "norm_common.h"

namespace tvae {

bool dropout_args(double p, const int64_t* rng, uint64_t seed, uint64_t offset, DropoutArgs* out) {
    if (!(p >= 0.0 && p <= 1.0)) return false;
    out->rng = rng; out->seed = seed; out->offset = offset;
    out->threshold = (uint32_t)std::nearbyint(p * 65536.0);
    out->scale = out->threshold >= 65536u ? 0.f : (float)(65536.0 / (65536.0 - (double)out->threshold));
    return true;
}

namespace {

struct DropoutCall {
    const void* in; const void* residual; void* out;
    RowsOf in_rows, res_rows;
    int grp, d, groups;
    long long rows;
    DropoutArgs drop;
};

// one thread per group of eight columns
template <typename A, typename O>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutCall c) {
    const Philox ph(c.drop);
    const long long total = c.rows * c.groups;
    for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
        const long long row = t / c.groups;
        const int g = (int)(t - row * c.groups), col = 8 * g, nv = c.d - col;
        float v[8];
        load8(static_cast<const A*>(c.in) + row_offset(c.in_rows, c.grp, row), col, nv, v);
        if (c.drop.threshold) drop8(ph, c.drop, (uint32_t)g, (uint32_t)row, v);
        if (c.residual) {
            float r[8];
            load8(static_cast<const O*>(c.residual) + row_offset(c.res_rows, c.grp, row), col, nv, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
        }
        store8(static_cast<O*>(c.out) + row * c.d, col, nv, v);
    }
}

template <typename A, typename O>
int dropout_launch(const DropoutCall& c, hipStream_t s) {
    const long long total = c.rows * c.groups;
    const long long blocks = (total + 255) / 256;
    hipLaunchKernelGGL((dropout_kernel<A, O>), dim3((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20))), dim3(256), 0, s, c);
    TVAE_CHECK_HIP(hipGetLastError());
    return TVAE_OK;
}

}  // namespace
}  // namespace tvae

using namespace tvae;

extern "C" int tvae_dropout(const void* in, int64_t in_so, int64_t in_si, const void* residual, int64_t res_so, int64_t res_si,
                            int64_t grp, void* out, int64_t rows, int64_t d, double p, const int64_t* rng, uint64_t seed,
                            uint64_t offset, int in_dtype, int out_dtype, void* stream) {
    TVAE_REQUIRE(norm_dtype_ok(in_dtype) && norm_dtype_ok(out_dtype), "dropout: unknown dtype %d / %d", in_dtype, out_dtype);
    TVAE_REQUIRE(in_dtype == out_dtype || in_dtype == TVAE_F32 || out_dtype == TVAE_F32,
                 "dropout: input and output are of one type, or one of them is fp32");
    TVAE_REQUIRE(in && out, "dropout: null pointer argument");
    TVAE_REQUIRE(rows > 0 && d > 0 && rows < (1ll << 31) && d < (1ll << 31), "dropout: bad shape rows=%lld d=%lld", (long long)rows, (long long)d);
    TVAE_REQUIRE(grp > 0 && rows % grp == 0, "dropout: %lld rows are not groups of %lld", (long long)rows, (long long)grp);
    DropoutCall c{};
    TVAE_REQUIRE(dropout_args(p, rng, seed, offset, &c.drop), "dropout: p = %g is not a probability", p);
    c.in = in; c.residual = residual; c.out = out;
    c.in_rows = RowsOf{in_so, in_si}; c.res_rows = RowsOf{res_so, res_si};
    c.grp = (int)grp; c.d = (int)d; c.groups = (int)((d + 7) / 8); c.rows = rows;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (in_dtype == TVAE_F32)
        return out_dtype == TVAE_F32 ? dropout_launch<float, float>(c, s) : out_dtype == TVAE_BF16 ? dropout_launch<float, bf16>(c, s)
                                                                                                 : dropout_launch<float, f16>(c, s);
    if (in_dtype == TVAE_BF16) return out_dtype == TVAE_BF16 ? dropout_launch<bf16, bf16>(c, s) : dropout_launch<bf16, float>(c, s);
    return out_dtype == TVAE_F16 ? dropout_launch<f16, f16>(c, s) : dropout_launch<f16, float>(c, s);
}
