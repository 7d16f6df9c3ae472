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
    int grp, d, groups;                         // groups = ceil(d / 8)
    long long rows, first;                      // first: the launch's first workgroup
    unsigned long long inv64; unsigned inv32;   // floor((2^64 - 1) / groups), floor((2^32 - 1) / groups)
    DropoutArgs drop;
};

// A workgroup takes 256 * GROUPS neighbouring groups, in the order of rows; every thread has its loads in flight before it
// evaluates the generator.  The row of a group is a multiplication by the reciprocal of a row's groups, whose quotient is
// at most one too small.
template <typename A, typename O, bool NT, int GROUPS>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutCall c) {
    const Philox ph(c.drop);
    const unsigned long long t0 = (unsigned long long)(c.first + blockIdx.x) * (256 * GROUPS);
    unsigned long long row0 = __umul64hi(t0, c.inv64);
    unsigned g0 = (unsigned)(t0 - row0 * (unsigned)c.groups);
    if (g0 >= (unsigned)c.groups) { ++row0; g0 -= (unsigned)c.groups; }
    Raw8<A> in[GROUPS];
    Raw8<O> res[GROUPS];
    long long row[GROUPS];
    unsigned g[GROUPS];
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        const unsigned u = g0 + threadIdx.x + 256 * k;
        unsigned q = __umulhi(u, c.inv32);
        unsigned r = u - q * (unsigned)c.groups;
        if (r >= (unsigned)c.groups) { ++q; r -= (unsigned)c.groups; }
        row[k] = (long long)row0 + q;
        g[k] = r;
        if (row[k] < c.rows) {
            const int nv = c.d - 8 * (int)r;
            const Cols at{8 * r, 8 * r + 4};
            in[k] = load_cols<A, false, NT>(static_cast<const A*>(c.in) + row_offset(c.in_rows, c.grp, row[k]), at, nv, 0);
            if (c.residual) res[k] = load_cols<O, false, NT>(static_cast<const O*>(c.residual) + row_offset(c.res_rows, c.grp, row[k]), at, nv, 0);
        }
    }
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        if (row[k] >= c.rows) continue;
        float v[8];
        unpack8(in[k], v);
        if (c.drop.threshold) drop8(ph, c.drop, g[k], (uint32_t)row[k], v);
        if (c.residual) {
            float r[8];
            unpack8(res[k], r);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
        }
        store_cols<false, NT>(static_cast<O*>(c.out) + row[k] * c.d, Cols{8 * g[k], 8 * g[k] + 4}, c.d - 8 * (int)g[k], 0, v);
    }
}

template <typename A, typename O, bool NT, int GROUPS>
int dropout_launch(DropoutCall c, hipStream_t s) {
    const long long blocks = (c.rows * c.groups + 256 * GROUPS - 1) / (256 * GROUPS);
    constexpr long long MOST = 1ll << 23;       // a launch has less than 2^32 threads
    TVAE_REQUIRE(blocks < (1ll << 31), "dropout: too many elements");
    for (c.first = 0; c.first < blocks; c.first += MOST) {
        const long long left = blocks - c.first;
        hipLaunchKernelGGL((dropout_kernel<A, O, NT, GROUPS>), dim3((unsigned)(left < MOST ? left : MOST)), dim3(256), 0, s, c);
        TVAE_CHECK_HIP(hipGetLastError());
    }
    return TVAE_OK;
}
// Long streams go past the caches.  Four groups a thread pay where they keep enough narrow loads in flight for that (bf16,
// 245760 x 1024: 166 us with four, 169 with two, 175 with one) and cost where workgroups are few or a thread's loads are
// 32 bytes anyway (f16 + residual, 30690 x 77: 11.4 / 7.6 / 5.7 us; fp32, 65536 x 1024: 99 / 98 / 94 us).
template <typename A, typename O>
int dropout_rows(const DropoutCall& c, hipStream_t s) {
    if (c.rows * c.d * (long long)sizeof(A) < (32ll << 20)) return dropout_launch<A, O, false, 1>(c, s);
    return dropout_launch<A, O, true, sizeof(A) == 2 && sizeof(O) == 2 ? 4 : 1>(c, s);
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
    c.inv64 = ~0ull / (unsigned)c.groups; c.inv32 = ~0u / (unsigned)c.groups;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (in_dtype == TVAE_F32)
        return out_dtype == TVAE_F32 ? dropout_rows<float, float>(c, s) : out_dtype == TVAE_BF16 ? dropout_rows<float, bf16>(c, s)
                                                                                                 : dropout_rows<float, f16>(c, s);
    if (in_dtype == TVAE_BF16) return out_dtype == TVAE_BF16 ? dropout_rows<bf16, bf16>(c, s) : dropout_rows<bf16, float>(c, s);
    return out_dtype == TVAE_F16 ? dropout_rows<f16, f16>(c, s) : dropout_rows<f16, float>(c, s);
}
