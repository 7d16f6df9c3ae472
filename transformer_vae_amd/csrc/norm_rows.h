// The kernels of norms.hip, as templates: norms_f32.hip, norms_bf16.hip and norms_f16.hip compile them for x of their type.
#pragma once
#include "norm_common.h"

namespace tvae {

struct NormCall {
    const void* x; const void* residual;            // at least one; T and R
    RowsOf x_rows, res_rows;
    int grp, d, groups;                             // groups = ceil(d / 8)
    long long rows;
    DropoutArgs drop;
    const void* weight; const void* bias;           // null: 1 and 0
    int w_f32, rms;                                 // weights are fp32 (else T); RMS norm
    float eps, inv_d;                               // inv_d = 1 / d
    float* mean; float* rstd;                       // forward: null in inference.  Backward: given (mean null for RMS)
    void* y; void* sum;                             // forward outputs (T; R, nullable)
    const void* dy; const void* dsum;               // backward: cotangents (T, nullable: 0; R, nullable: 0)
    RowsOf dy_rows, ds_rows;
    void* dx; void* dres;                           // nullable (T; R)
    float* part; int chunks;                        // [2][chunks][d] partial sums of dw and db
    int chunk_rows;
    void* dw; void* db;                             // nullable
};

// one translation unit each
int norm_launch_f32(const NormCall& c, bool bwd, hipStream_t s);
int norm_launch_bf16(const NormCall& c, int r_dtype, bool bwd, hipStream_t s);
int norm_launch_f16(const NormCall& c, int r_dtype, bool bwd, hipStream_t s);

namespace {

// sum over the 256 threads of a workgroup, the same bits in every thread
template <typename V>
__device__ __forceinline__ V block_sum(V v, V* sm) {
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
        load8(static_cast<const float*>(p), col, nv, v);
    } else {
        load8(static_cast<const T*>(p), col, nv, v);
    }
}

// the eight values of v that start at column 8 g; columns beyond d are 0
template <typename T, typename R>
__device__ __forceinline__ void value8(const NormCall& c, const Philox& ph, long long row, int g, float v[8]) {
    const int nv = c.d - 8 * g;
    if (c.x) {
        load8(static_cast<const T*>(c.x) + row_offset(c.x_rows, c.grp, row), 8 * g, nv, v);
        if (c.drop.threshold) drop8(ph, c.drop, (uint32_t)g, (uint32_t)row, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
    if (c.residual) {
        float r[8];
        load8(static_cast<const R*>(c.residual) + row_offset(c.res_rows, c.grp, row), 8 * g, nv, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
    }
}

// ---- rows that fit the registers of TPR threads, V packs of eight columns each -----------------------------------------
// Each of the inputs is read once: the row stays in registers between the sums and the output.  Short rows take 8 .. 64 lanes
// of a wave, so that several of them share one; longer ones take whole waves and add their sums through LDS.  The weights
// are loaded once a workgroup, which then walks over rows.

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// sum over aligned groups of LANES lanes, the same bits in each of them: exchanges inside rows of 16 lanes, then between
// rows, all in the vector ALU
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    v = dpp_add<0xB1>(v);                        // lane ^ 1
    v = dpp_add<0x4E>(v);                        // lane ^ 2
    v = dpp_add<0x141>(v);                       // the other four of eight
    if constexpr (LANES >= 16) v = dpp_add<0x140>(v);
    if constexpr (LANES >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (LANES >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// Four packs a thread: the sums for dw and db live in LDS, every thread's in places of its own, and the next row's loads do not
// fly beside the current row's work in a backward pass whose registers they would not fit (FUSED, fp32).
constexpr bool sums_in_lds(int v) { return v >= 4; }
template <typename T, int V, int FORM> constexpr bool bwd_ahead() { return V < 4 || (!(FORM & 1) && sizeof(T) == 2); }

// sum over the lanes of a wave that hold the same columns: those TPR apart
template <int TPR>
__device__ __forceinline__ float same_columns_sum(float v) {
    if constexpr (TPR <= 8) v = dpp_add<0x128>(v);       // the other eight of sixteen
    if constexpr (TPR <= 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (TPR <= 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

template <int TPR>
struct RowThreads {
    static constexpr int BLOCK = TPR > 256 ? TPR : 256;
    static constexpr int ROWS = BLOCK / TPR;             // rows a workgroup works on at a time
    static constexpr int WAVES = TPR > 64 ? TPR / 64 : 1;  // waves of a row
    static constexpr int WPE = 2;                        // waves a SIMD that the registers are held to
};
// sums of N values over the TPR threads of a row.  `sm` is one of two buffers that take turns, [BLOCK / 64][N]: a wave may
// write the next sum while another still reads this one, and there is a barrier between this and the one after
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* sm) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum<(TPR < 64 ? TPR : 64)>(v[i]);
    if constexpr (TPR > 64) {
        constexpr int W = RowThreads<TPR>::WAVES;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) sm[wave * N + i] = v[i];
        }
        __syncthreads();
        const float* mine = sm + (wave / W) * W * N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t = mine[i];
#pragma unroll
            for (int k = 1; k < W; ++k) t += mine[k * N + i];
            v[i] = t;
        }
    }
}

// What a kernel is compiled for.  PLAIN: x alone, without dropout, dx alone.  FUSED: everything the call can ask for.  The ragged
// ones take d that is no multiple of 8 (their handling of the cut pack, compiled into all, cost the others 3 to 15 %); TINY
// is FUSED for rows of less than eight elements, which are loaded piece by piece.
enum NormForm { PLAIN = 0, FUSED = 1, RAGGED_PLAIN = 2, RAGGED_FUSED = 3, TINY = 7 };
constexpr bool is_fused(int form) { return form & 1; }
constexpr bool is_ragged(int form) { return form & 2; }

// the columns of a thread's pack k of eight, and how many of them are in the row
template <int TPR, bool SPLIT, int FORM>
struct RowCols {
    uint32_t l, d;
    __device__ __forceinline__ Cols at(int k) const {
        if constexpr (SPLIT) return Cols{4 * (l + 2 * TPR * k), 4 * (l + 2 * TPR * k + TPR)};
        else return Cols{8 * (l + TPR * k), 8 * (l + TPR * k) + 4};
    }
    __device__ __forceinline__ int left(uint32_t col) const { return (int)(d - col); }
};

// the last n elements of 16 bytes (of 8: the half that starts at dword h) to their start, zeros behind them
__device__ __forceinline__ u32x4 last_first16(u32x4 q, int n) {          // eight 16-bit elements
    const int a = 8 - n;
    if (a & 1) q = u32x4{q[0] >> 16 | q[1] << 16, q[1] >> 16 | q[2] << 16, q[2] >> 16 | q[3] << 16, q[3] >> 16};
    if (a & 2) q = u32x4{q[1], q[2], q[3], 0};
    if (a & 4) q = u32x4{q[2], q[3], 0, 0};
    return q;
}
__device__ __forceinline__ u32x4 last_first_half(u32x4 q, int h, int n) { // four 16-bit elements
    const uint64_t v = ((uint64_t)q[h + 1] << 32 | q[h]) >> (16 * (4 - n));
    q[h] = (uint32_t)v;
    q[h + 1] = (uint32_t)(v >> 32);
    return q;
}
__device__ __forceinline__ u32x4 last_first32(u32x4 q, int n) {          // four fp32 elements
    const int a = 4 - n;
    if (a & 1) q = u32x4{q[1], q[2], q[3], 0};
    if (a & 2) q = u32x4{q[2], q[3], 0, 0};
    return q;
}

// What one row's loads bring: those of a workgroup's next row fly while it works on this one.  Every access is whole: one that the
// row's end cuts, or that lies beyond it, takes the row's last elements, and use() puts them in place.
template <typename T, int TPR, int V, bool SPLIT, int FORM, bool NT>
struct RowLoad {
    static constexpr int N = SPLIT ? 4 : 8;              // elements of an access
    Raw8<T> g[V];
    using C = RowCols<TPR, SPLIT, FORM>;
    __device__ __forceinline__ void get(const void* p, const RowsOf& rows, int grp, long long row, const C& cols) {
        const T* q = static_cast<const T*>(p) + row_offset(rows, grp, row);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const Cols c = cols.at(k);
            if constexpr (FORM == TINY) g[k] = load_cols<T, SPLIT, NT>(q, c, cols.left(c.col), cols.left(c.second));
            else g[k] = load_cols<T, SPLIT, NT>(q, Cols{min(c.col, cols.d - N), min(c.second, cols.d - N)}, 8, 8);
        }
    }
    __device__ __forceinline__ void use(int k, const C& cols, float v[8]) const {
        Raw8<T> r = g[k];
        if constexpr (FORM != TINY) {
            const Cols c = cols.at(k);
            const int n[2] = {cols.left(c.col), cols.left(c.second)};
            if constexpr (sizeof(T) == 2 && !SPLIT) {
                if (is_ragged(FORM) && n[0] > 0 && n[0] < 8) r.q[0] = last_first16(r.q[0], n[0]);
#pragma unroll
                for (int e = 0; e < 4; ++e) r.q[0][e] = n[0] > 0 ? r.q[0][e] : 0u;
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if constexpr (sizeof(T) == 2) {
                        if (is_ragged(FORM) && n[i] > 0 && n[i] < 4) r.q[0] = last_first_half(r.q[0], 2 * i, n[i]);
#pragma unroll
                        for (int e = 0; e < 2; ++e) r.q[0][2 * i + e] = n[i] > 0 ? r.q[0][2 * i + e] : 0u;
                    } else {
                        if (is_ragged(FORM) && n[i] > 0 && n[i] < 4) r.q[i] = last_first32(r.q[i], n[i]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) r.q[i][e] = n[i] > 0 ? r.q[i][e] : 0u;
                    }
                }
            }
        }
        unpack8(r, v);
    }
};
template <typename T, int TPR, bool SPLIT, int FORM, bool NT>
__device__ __forceinline__ void store_pack(void* base, long long row, int k, const RowCols<TPR, SPLIT, FORM>& cols, const float v[8]) {
    T* p = static_cast<T*>(base) + row * cols.d;
    const Cols c = cols.at(k);
    if constexpr (is_ragged(FORM)) store_cols<SPLIT, NT>(p, c, cols.left(c.col), cols.left(c.second), v);
    else if constexpr (SPLIT) store_cols<true, NT>(p, c, c.col < cols.d ? 4 : 0, c.second < cols.d ? 4 : 0, v);
    else if (c.col < cols.d) store_cols<false, NT>(p, c, 8, 4, v);
}
// weights: `fill` where there are none, 0 beyond the row
template <typename T, int TPR, bool SPLIT, int FORM>
__device__ __forceinline__ void load_params(const void* p, int f32, int k, const RowCols<TPR, SPLIT, FORM>& cols, float fill, float v[8]) {
    const Cols c = cols.at(k);
    if (!p) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fill;
    } else if (sizeof(T) == 4 || f32) {
        unpack8(load_cols<float, SPLIT, false>(static_cast<const float*>(p), c, cols.left(c.col), cols.left(c.second)), v);
    } else {
        unpack8(load_cols<T, SPLIT, false>(static_cast<const T*>(p), c, cols.left(c.col), cols.left(c.second)), v);
    }
}
// keep decisions of a pack.  SPLIT: its quads are halves of two groups, whose other halves the neighbouring lane holds; each of the
// two evaluates one of the groups and hands the other half over.
template <int TPR, bool SPLIT, int FORM>
__device__ __forceinline__ uint32_t keep_pack(const Philox& ph, const DropoutArgs& a, int k, const RowCols<TPR, SPLIT, FORM>& cols, uint32_t row) {
    if constexpr (!SPLIT) return keep8(ph, a, (uint32_t)(cols.l + TPR * k), row);
    const int odd = cols.l & 1;
    const uint32_t own = keep8(ph, a, (uint32_t)((cols.l >> 1) + TPR * k + (odd ? TPR / 2 : 0)), row);
    const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)own, 0xB1, 0xf, 0xf, true);     // lane ^ 1
    return odd ? (other >> 4) | (own & 0xf0u) : (own & 0xfu) | (other & 0xfu) << 4;
}

template <int TPR>
__device__ __forceinline__ int row_slot() {
    if constexpr (TPR >= 64) return __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);     // one row a wave: scalar addresses
    return threadIdx.x / TPR;
}

template <typename T, typename R, int TPR, int V, int FORM, bool NT>
__global__ __launch_bounds__(RowThreads<TPR>::BLOCK, RowThreads<TPR>::WPE) void norm_fwd_kernel(NormCall c) {
    using L = RowThreads<TPR>;
    constexpr bool SPLIT = sizeof(R) == 4;
    __shared__ float sm[2][L::BLOCK / 64 * 2];
    const Philox ph(c.drop);
    const int sub = row_slot<TPR>();
    const uint32_t l = threadIdx.x % TPR;
    const RowCols<TPR, SPLIT, FORM> cols{l, (uint32_t)c.d};
    const long long step = (long long)gridDim.x * L::ROWS;
    long long row = (long long)blockIdx.x * L::ROWS + sub;
    RowLoad<T, TPR, V, SPLIT, FORM, NT> nx{};
    RowLoad<R, TPR, V, SPLIT, FORM, NT> nr{};
    auto fetch = [&](long long at) {
        if (at >= c.rows) return;
        if (!is_fused(FORM) || c.x) nx.get(c.x, c.x_rows, c.grp, at, cols);
        if (is_fused(FORM) && c.residual) nr.get(c.residual, c.res_rows, c.grp, at, cols);
    };
    fetch(row);
    float w[V][8], b[V][8];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        load_params<T>(c.weight, c.w_f32, k, cols, 1.f, w[k]);
        load_params<T>(c.bias, c.w_f32, k, cols, 0.f, b[k]);
    }
    int turn = 0;
    for (long long base = (long long)blockIdx.x * L::ROWS; base < c.rows; base += step, row += step) {
        float v[V][8];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            nx.use(k, cols, v[k]);
            if constexpr (is_fused(FORM)) {
                if (c.x && c.drop.threshold) drop8(keep_pack(ph, c.drop, k, cols, (uint32_t)row), c.drop.scale, v[k]);
                if (c.residual) {
                    float r[8];
                    nr.use(k, cols, r);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[k][e] += r[e];
                }
            }
        }
        fetch(row + step);
        const bool live = row < c.rows;
        if constexpr (is_fused(FORM)) {
            if (c.sum && live) {
#pragma unroll
                for (int k = 0; k < V; ++k) store_pack<R, TPR, SPLIT, FORM, NT>(c.sum, row, k, cols, v[k]);
            }
        }
        float mu = 0.f;
        if (!c.rms) {
            float s[1] = {0.f};
#pragma unroll
            for (int k = 0; k < V; ++k)
                s[0] += ((v[k][0] + v[k][1]) + (v[k][2] + v[k][3])) + ((v[k][4] + v[k][5]) + (v[k][6] + v[k][7]));
            row_sums<TPR, 1>(s, sm[turn]);
            turn ^= 1;
            mu = s[0] * c.inv_d;
        }
        // squares about the fp32 mean, with the sum of the deviations beside them: their mean is what rounding left in mu,
        // and taking it out of both keeps rows of equal values at 0 under the smallest eps
        float q[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const Cols at = cols.at(k);
            if constexpr (is_ragged(FORM)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k][e] -= (e < 4 ? at.col : at.second) + (e & 3) < cols.d ? mu : 0.f;
            } else {
                const float m[2] = {at.col < cols.d ? mu : 0.f, at.second < cols.d ? mu : 0.f};
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k][e] -= m[e >> 2];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                q[0] = fmaf(v[k][e], v[k][e], q[0]);
                q[1] += v[k][e];
            }
        }
        row_sums<TPR, 2>(q, sm[turn]);
        turn ^= 1;
        const float m2 = c.rms ? 0.f : q[1] * c.inv_d;
        float var = q[0] * c.inv_d - m2 * m2;
        if (var < 0.f) var = 0.f;
        const float rs = rsqrtf(var + c.eps);
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < V; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] = fmaf((v[k][e] - m2) * rs, w[k][e], b[k][e]);
            store_pack<T, TPR, SPLIT, FORM, NT>(c.y, row, k, cols, v[k]);
        }
        if (l == 0 && c.rstd) {
            c.rstd[row] = rs;
            if (c.mean) c.mean[row] = mu + m2;
        }
    }
}

// The sums for dw and db grow in registers while the workgroup walks over rows; at the end the rows that a workgroup works on
// at a time add theirs in a fixed order, across lanes and then through LDS, and one partial sum a workgroup goes out.
template <typename T, typename R, int TPR, int V, int FORM, bool NT>
__global__ __launch_bounds__(RowThreads<TPR>::BLOCK, RowThreads<TPR>::WPE) void norm_bwd_kernel(NormCall c) {
    using L = RowThreads<TPR>;
    constexpr bool SPLIT = sizeof(R) == 4, AHEAD = bwd_ahead<T, V, FORM>();
    __shared__ float sm[2][L::BLOCK / 64 * 2];
    extern __shared__ float sums[];                  // [2][V][8][TPR] where the registers do not hold them
    const Philox ph(c.drop);
    const int sub = row_slot<TPR>();
    const uint32_t l = threadIdx.x % TPR;
    const RowCols<TPR, SPLIT, FORM> cols{l, (uint32_t)c.d};
    const long long step = (long long)gridDim.x * L::ROWS;
    long long row = (long long)blockIdx.x * L::ROWS + sub;
    RowLoad<T, TPR, V, SPLIT, FORM, NT> ny{}, nx{};
    RowLoad<R, TPR, V, SPLIT, FORM, NT> nr{};
    float nmu = 0.f, nrs = 0.f;
    auto fetch = [&](long long at) {
        if (at >= c.rows) return;
        ny.get(c.dy, c.dy_rows, c.grp, at, cols);
        if (!is_fused(FORM) || c.x) nx.get(c.x, c.x_rows, c.grp, at, cols);
        if (is_fused(FORM) && c.residual) nr.get(c.residual, c.res_rows, c.grp, at, cols);
        nrs = c.rstd[at];
        if (c.mean) nmu = c.mean[at];
    };
    if (AHEAD) fetch(row);
    float w[V][8], aw[V][8], ab[V][8];
    auto slot = [&](int which, int k, int e) -> float& { return sums[((which * V + k) * 8 + e) * TPR + l]; };
#pragma unroll
    for (int k = 0; k < V; ++k) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            aw[k][e] = 0.f; ab[k][e] = 0.f;
            if (sums_in_lds(V)) { slot(0, k, e) = 0.f; slot(1, k, e) = 0.f; }
        }
        load_params<T>(c.weight, c.w_f32, k, cols, 1.f, w[k]);
    }
    int turn = 0;
    for (long long base = (long long)blockIdx.x * L::ROWS; base < c.rows; base += step, row += step) {
        const bool live = row < c.rows;
        if (!AHEAD) fetch(row);
        const float mu = nmu, rs = nrs;
        float u[V][8], v[V][8];
        uint32_t kept[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            nx.use(k, cols, v[k]);
            if constexpr (is_fused(FORM)) {
                kept[k] = 0;
                if (c.drop.threshold) {
                    kept[k] = keep_pack(ph, c.drop, k, cols, (uint32_t)row);
                    if (c.x) drop8(kept[k], c.drop.scale, v[k]);
                }
                if (c.residual) {
                    float r[8];
                    nr.use(k, cols, r);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[k][e] += r[e];
                }
            }
            ny.use(k, cols, u[k]);
        }
        RowLoad<R, TPR, V, SPLIT, FORM, NT> ds{};        // before the next row's: loads arrive in order
        if constexpr (is_fused(FORM)) {
            if (c.dsum && live) ds.get(c.dsum, c.ds_rows, c.grp, row, cols);
        }
        if (AHEAD) fetch(row + step);
        float s[2] = {0.f, 0.f};
        if (live) {
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[k][e] = (v[k][e] - mu) * rs;
                    if (!sums_in_lds(V)) {
                        aw[k][e] = fmaf(u[k][e], v[k][e], aw[k][e]);
                        ab[k][e] += u[k][e];
                    } else {
                        slot(0, k, e) = fmaf(u[k][e], v[k][e], slot(0, k, e));
                        slot(1, k, e) += u[k][e];
                    }
                    u[k][e] *= w[k][e];
                    s[0] += u[k][e];
                    s[1] = fmaf(u[k][e], v[k][e], s[1]);
                }
        }
        row_sums<TPR, 2>(s, sm[turn]);
        turn ^= 1;
        if (!live || !(c.dx || (is_fused(FORM) && c.dres))) continue;
        const float s1 = c.rms ? 0.f : s[0] * c.inv_d, s2 = s[1] * c.inv_d;
#pragma unroll
        for (int k = 0; k < V; ++k) {
#pragma unroll
            for (int e = 0; e < 8; ++e) u[k][e] = rs * ((u[k][e] - s1) - v[k][e] * s2);
            if constexpr (is_fused(FORM)) {
                if (c.dsum) {
                    float t[8];
                    ds.use(k, cols, t);
#pragma unroll
                    for (int e = 0; e < 8; ++e) u[k][e] += t[e];
                }
                if (c.dres) store_pack<R, TPR, SPLIT, FORM, NT>(c.dres, row, k, cols, u[k]);
                if (!c.dx) continue;
                if (c.drop.threshold) drop8(kept[k], c.drop.scale, u[k]);
            }
            store_pack<T, TPR, SPLIT, FORM, NT>(c.dx, row, k, cols, u[k]);
        }
    }
    if (!c.dw && !c.db) return;
    constexpr int SLOTS = TPR > 64 ? L::ROWS : 4;        // what is left to add once a wave's rows are one
    const int slot_at = TPR > 64 ? sub : (int)(threadIdx.x >> 6);
    if constexpr (SLOTS > 1) {
        __shared__ float acc[SLOTS - 1][TPR][9];         // nine: eight neighbouring words a lane would meet in eight banks
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                if (!(which ? c.db : c.dw)) continue;
                float (&a)[8] = which ? ab[k] : aw[k];
#pragma unroll
                for (int e = 0; e < 8; ++e) a[e] = same_columns_sum<TPR>(a[e]);
                __syncthreads();
                if (slot_at && (threadIdx.x & 63) < TPR) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[slot_at - 1][l][e] = a[e];
                }
                __syncthreads();
                if (!slot_at) {
#pragma unroll
                    for (int o = 0; o < SLOTS - 1; ++o)
#pragma unroll
                        for (int e = 0; e < 8; ++e) a[e] += acc[o][l][e];
                }
            }
    }
    if (sub) return;                                     // (the first row's threads hold the sums)
#pragma unroll
    for (int k = 0; k < V; ++k) {
        if (sums_in_lds(V)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) { aw[k][e] = slot(0, k, e); ab[k][e] = slot(1, k, e); }
        }
        if (c.dw) store_pack<float, TPR, SPLIT, FORM, false>(c.part, blockIdx.x, k, cols, aw[k]);
        if (c.db) store_pack<float, TPR, SPLIT, FORM, false>(c.part + (long long)c.chunks * c.d, blockIdx.x, k, cols, ab[k]);
    }
}

// ---- a few hundred rows: dx, dw and db in one launch ------------------------------------------------------------------------
// The first workgroups take a row a wave and write dx, the others take 16 columns each and write their dw and db: two packs by 128 row
// lanes, whose sums meet in LDS in a fixed order.  Both read the inputs, which the caches hold at these sizes; what it saves is
// the second kernel behind the first and the partial sums between them (fp32, one launch against two: 40 x 512 2.9 / 7.5 us,
// 350 x 768 4.3 / 7.0, 512 x 2048 7.6 / 9.9; with dropout and residual 512 x 768 8.9 / 9.5: the row lanes' serial loops catch up).
constexpr int SMALL_ROWS = 512, SMALL_D = 2048;
inline bool bwd_small(int64_t rows, int64_t d) { return rows <= SMALL_ROWS && d <= SMALL_D; }

template <typename T, typename R>
__global__ __launch_bounds__(256) void norm_bwd_small_kernel(NormCall c, int row_blocks) {
    const Philox ph(c.drop);
    if ((int)blockIdx.x < row_blocks) {
        constexpr int PACKS = SMALL_D / 8 / 64;
        const int lane = threadIdx.x & 63;
        const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
        if (row >= c.rows) return;
        const float mu = c.mean ? c.mean[row] : 0.f, rs = c.rstd[row];
        const T* dy = static_cast<const T*>(c.dy) + row_offset(c.dy_rows, c.grp, row);
        float u[PACKS][8], v[PACKS][8], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
            const int g = lane + 64 * k, nv = c.d - 8 * g;
            if (g >= c.groups) continue;
            float w[8];
            load8(dy, 8 * g, nv, u[k]);
            load8_param<T>(c.weight, c.w_f32, 8 * g, nv, 1.f, w);
            value8<T, R>(c, ph, row, g, v[k]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[k][e] = (v[k][e] - mu) * rs;
                u[k][e] *= w[e];
                s1 += u[k][e];
                s2 = fmaf(u[k][e], v[k][e], s2);
            }
        }
        s1 = c.rms ? 0.f : lanes_sum<64>(s1) * c.inv_d;
        s2 = lanes_sum<64>(s2) * c.inv_d;
#pragma unroll
        for (int k = 0; k < PACKS; ++k) {
            const int g = lane + 64 * k, nv = c.d - 8 * g;
            if (g >= c.groups) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) u[k][e] = rs * ((u[k][e] - s1) - v[k][e] * s2);
            if (c.dsum) {
                float t[8];
                load8(static_cast<const R*>(c.dsum) + row_offset(c.ds_rows, c.grp, row), 8 * g, nv, t);
#pragma unroll
                for (int e = 0; e < 8; ++e) u[k][e] += t[e];
            }
            if (c.dres) store8(static_cast<R*>(c.dres) + row * c.d, 8 * g, nv, u[k]);
            if (c.dx) {
                if (c.drop.threshold) drop8(ph, c.drop, (uint32_t)g, (uint32_t)row, u[k]);
                store8(static_cast<T*>(c.dx) + row * c.d, 8 * g, nv, u[k]);
            }
        }
        return;
    }
    __shared__ float sums[2][128][18];           // 18: lanes that write eight neighbours meet few others in a bank
    const int pack = threadIdx.x & 1, lane = threadIdx.x >> 1;
    const int g = ((int)blockIdx.x - row_blocks) * 2 + pack;
    float aw[8] = {}, ab[8] = {};
    if (g < c.groups) {
        for (long long row = lane; row < c.rows; row += 128) {
            float u[8], v[8];
            const float mu = c.mean ? c.mean[row] : 0.f, rs = c.rstd[row];
            load8(static_cast<const T*>(c.dy) + row_offset(c.dy_rows, c.grp, row), 8 * g, c.d - 8 * g, u);
            value8<T, R>(c, ph, row, g, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                aw[e] = fmaf(u[e], (v[e] - mu) * rs, aw[e]);
                ab[e] += u[e];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) { sums[0][lane][8 * pack + e] = aw[e]; sums[1][lane][8 * pack + e] = ab[e]; }
    __syncthreads();
    const int which = threadIdx.x >> 7, part = threadIdx.x >> 4 & 7, col = threadIdx.x & 15;     // eight threads a column
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += sums[which][16 * part + k][col];
    __syncthreads();
    sums[which][part][col] = t;
    __syncthreads();
    void* out = which ? c.db : c.dw;
    const int at = ((int)blockIdx.x - row_blocks) * 16 + col;
    if (part || at >= c.d || !out) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) t += sums[which][k][col];
    if (sizeof(T) == 4 || c.w_f32) static_cast<float*>(out)[at] = t;
    else static_cast<T*>(out)[at] = from_f32<T>(t);
}

// ---- longer rows: one workgroup per row, the row is read again for every pass over it ----------------------------
// Eight neighbours are added in fp32, all further ones in fp64: a thread adds d / 2048 of them one after another, where fp32 would
// lose up to as many roundings (2000000 equal values: their RMS norm was 2.2e-5 of itself off).  Two fp64 additions for eight
// elements cost nothing beside the loads (2048 x 40000 bf16 forward 116 us either way, with its backward pass 364).
__device__ __forceinline__ float sum8(const float v[8]) { return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])); }
__device__ __forceinline__ float dot8(const float a[8], const float b[8]) {
    return (fmaf(a[1], b[1], a[0] * b[0]) + fmaf(a[3], b[3], a[2] * b[2])) + (fmaf(a[5], b[5], a[4] * b[4]) + fmaf(a[7], b[7], a[6] * b[6]));
}

template <typename T, typename R>
__global__ __launch_bounds__(256) void norm_fwd_wide_kernel(NormCall c) {
    __shared__ double sm[4];
    const Philox ph(c.drop);
    for (long long row = blockIdx.x; row < c.rows; row += gridDim.x) {
        float mu = 0.f, m2 = 0.f;
        if (!c.rms) {
            // A first guess of the mean from 2048 elements at 32 places of the row (these rows are longer).  It is off by next to
            // nothing for most rows, so sums about it lose nothing and the row is read twice, not three times.
            float v[8];
            value8<T, R>(c, ph, row, (int)((long long)(threadIdx.x >> 3) * c.groups / 32) + (threadIdx.x & 7), v);
            mu = (float)block_sum((double)sum8(v), sm) * (1.f / 2048.f);
        }
        double t1 = 0.0, q = 0.0;
        const auto sums = [&] {
            t1 = q = 0.0;
            for (int g = threadIdx.x; g < c.groups; g += 256) {
                float v[8];
                value8<T, R>(c, ph, row, g, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = 8 * g + e < c.d ? v[e] - mu : 0.f;
                t1 += (double)sum8(v);
                q += (double)dot8(v, v);
            }
            q = block_sum(q, sm) / (double)c.d;
            if (c.rms) return;
            t1 = block_sum(t1, sm) / (double)c.d;
            q -= t1 * t1;
            if (q < 0.0) q = 0.0;
        };
        sums();
        // Where those places are unlike the rest the guess can be off by sqrt(d / 2048) standard deviations, and every difference to
        // it carries a rounding of that much.  Beyond one standard deviation the sums are taken again, about the mean that they
        // gave (2000000 elements, the first 64 of each 32nd a thousand above the others' unit spread: half of the results
        // were over 4e-5 of themselves off, 5e-8 now).  All threads have the same sums.
        if (!c.rms && t1 * t1 > q) {
            mu += (float)t1;
            sums();
        }
        if (!c.rms) m2 = (float)t1;
        const float rs = rsqrtf((float)q + c.eps);
        for (int g = threadIdx.x; g < c.groups; g += 256) {
            float v[8], w[8], b[8];
            const int nv = c.d - 8 * g;
            value8<T, R>(c, ph, row, g, v);
            if (c.sum) store8(static_cast<R*>(c.sum) + row * c.d, 8 * g, nv, v);
            load8_param<T>(c.weight, c.w_f32, 8 * g, nv, 1.f, w);
            load8_param<T>(c.bias, c.w_f32, 8 * g, nv, 0.f, b);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(((v[e] - mu) - m2) * rs, w[e], b[e]);
            store8(static_cast<T*>(c.y) + row * c.d, 8 * g, nv, v);
        }
        if (threadIdx.x == 0 && c.rstd) {
            c.rstd[row] = rs;
            if (c.mean) c.mean[row] = mu + m2;
        }
    }
}

template <typename T, typename R>
__global__ __launch_bounds__(256) void norm_bwd_wide_kernel(NormCall c) {
    __shared__ double sm[4];
    const Philox ph(c.drop);
    for (long long row = blockIdx.x; row < c.rows; row += gridDim.x) {
        const float mu = c.mean ? c.mean[row] : 0.f, rs = c.rstd[row];
        const T* dy = static_cast<const T*>(c.dy) + row_offset(c.dy_rows, c.grp, row);
        double t1 = 0.0, t2 = 0.0;
        for (int g = threadIdx.x; g < c.groups; g += 256) {
            float v[8], w[8], u[8];
            const int nv = c.d - 8 * g;
            value8<T, R>(c, ph, row, g, v);
            load8(dy, 8 * g, nv, u);
            load8_param<T>(c.weight, c.w_f32, 8 * g, nv, 1.f, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                u[e] *= w[e];
                v[e] = (v[e] - mu) * rs;
            }
            t1 += (double)sum8(u);
            t2 += (double)dot8(u, v);
        }
        const float s2 = (float)(block_sum(t2, sm) / (double)c.d);
        const float s1 = c.rms ? 0.f : (float)(block_sum(t1, sm) / (double)c.d);
        for (int g = threadIdx.x; g < c.groups; g += 256) {
            float v[8], w[8], u[8];
            const int nv = c.d - 8 * g;
            value8<T, R>(c, ph, row, g, v);
            load8(dy, 8 * g, nv, u);
            load8_param<T>(c.weight, c.w_f32, 8 * g, nv, 1.f, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = rs * ((u[e] * w[e] - s1) - (v[e] - mu) * rs * s2);
            if (c.dsum) {
                load8(static_cast<const R*>(c.dsum) + row_offset(c.ds_rows, c.grp, row), 8 * g, nv, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += u[e];
            }
            if (c.dres) store8(static_cast<R*>(c.dres) + row * c.d, 8 * g, nv, v);
            if (c.dx) {
                if (c.drop.threshold) drop8(ph, c.drop, (uint32_t)g, (uint32_t)row, v);
                store8(static_cast<T*>(c.dx) + row * c.d, 8 * g, nv, v);
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
            load8(static_cast<const T*>(c.dy) + row_offset(c.dy_rows, c.grp, row), 8 * g, c.d - 8 * g, u);
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
        float* pw = c.part + (long long)blockIdx.y * c.d;
        store8(pw, 8 * g, c.d - 8 * g, aw);
        store8(pw + (long long)c.chunks * c.d, 8 * g, c.d - 8 * g, ab);
    }
}

// ---- which kernel, and how many workgroups ----------------------------------------------------------------------------
constexpr int NORM_CUS = 256;

// threads a row and packs of eight a thread; tpr 0: longer than any of these
struct RowPlan { int tpr, v; };
// The shape with the least room that holds the row: idle threads cost what their loads would have brought.  The last list: where x and
// the residual are of 16 bits (bf16 with dropout and residual, 60000 x 1280: forward 85 us with 64 x 3, 124 with 128 x 2, backward 156
// and 193); three packs of fp32 do not fit the registers of a fused backward pass.  They are there for the widths that were measured
// (768, 1280, 5120).  Not measured: three packs of 16, 128 and 512 threads (bf16, 16384 x 3000: forward 45.5 us with 256 x 2, its bytes
// alone 32), and three of fp32 without a fused backward pass (60000 x 768 and x 1280 take 2 to 9 % more than their bytes as they are).
#define NORM_SHAPES(X) X(8, 1) X(16, 1) X(32, 1) X(32, 2) X(64, 2) X(128, 2) X(256, 2) X(512, 2) X(512, 4)
#define NORM_TINY_SHAPES(X) X(8, 1)
#define NORM_NARROW_SHAPES(X) X(32, 3) X(64, 3) X(256, 3)
inline RowPlan row_plan(int64_t d, bool narrow) {
    const int64_t packs = (d + 7) / 8;
    RowPlan p{0, 0};
#define X(TPR, V) if (packs <= TPR * V && (!p.tpr || TPR * V < p.tpr * p.v)) p = RowPlan{TPR, V};
    NORM_SHAPES(X)
    if (narrow) { NORM_NARROW_SHAPES(X) }
#undef X
    return p;
}
inline NormForm norm_form(const NormCall& c) {
    if (c.d < 8) return TINY;
    const bool fused = !c.x || c.residual || c.drop.threshold || c.sum || c.dsum || c.dres;
    if (c.d % 8) return fused ? RAGGED_FUSED : RAGGED_PLAIN;
    return fused ? FUSED : PLAIN;
}
inline int plan_rows(const RowPlan& p) { return p.tpr >= 256 ? 1 : 256 / p.tpr; }
// Workgroups in flight, a CU: 512 threads of loads of two packs or more keep the memory busy, and the fewer streams there are, the
// better the order in which it sees them (bf16, 245760 x 1024: forward 173 us with 512 workgroups of 256, 184 with 768, 190 with
// 1024; backward 253 / 275 / 290).  Single packs need twice as many (fp32, 1000000 x 24: forward 61 us with two, 46 with four).
inline int64_t plan_blocks(const RowPlan& p) { return (p.tpr > 256 ? 1 : p.v == 1 ? 4 : 2) * NORM_CUS; }
// Streams of 32 MB on go past the caches (bf16, 245760 x 1024, backward: 280 -> 261 us); shorter ones may still be there when
// the next kernel reads them (fp32, 5120 x 768, backward: 14.4 us with the caches, 16.5 past them).
inline bool norm_streams(const NormCall& c, int64_t esize) { return c.rows * c.d * esize >= (32ll << 20); }

constexpr int64_t WIDE_CHUNK_ROWS = 64;          // rows a partial sum, at least; more where that would make over 1024 of them
inline int64_t wide_chunk_rows(int64_t rows) {
    const int64_t r = (rows + 1023) / 1024;
    return r > WIDE_CHUNK_ROWS ? r : WIDE_CHUNK_ROWS;
}
// partial sums of a backward pass: workgroups of the row kernel, or chunks of rows
inline int64_t bwd_chunks(int64_t rows, int64_t d, bool narrow) {
    const RowPlan p = row_plan(d, narrow);
    if (!p.tpr) { const int64_t r = wide_chunk_rows(rows); return (rows + r - 1) / r; }
    const int64_t turns = (rows + plan_rows(p) - 1) / plan_rows(p), most = plan_blocks(p);
    const int64_t want = (turns + 3) / 4;        // at least four turns a workgroup, while that leaves enough of them
    const int64_t n = want < NORM_CUS ? (turns < NORM_CUS ? turns : NORM_CUS) : want;
    return n < most ? n : most;
}

template <typename T, typename R, int TPR, int V, int FORM, bool NT>
int norm_rows_launch(const NormCall& c, bool bwd, int64_t blocks, hipStream_t s) {
    using L = RowThreads<TPR>;
    size_t lds = 0;
    if constexpr (sums_in_lds(V)) {
        if (bwd) {
            lds = sizeof(float) * 2 * V * 8 * TPR;
            static PerDeviceOnce once;
            TVAE_CHECK_HIP(per_device_once(once, [] {
                return hipFuncSetAttribute(reinterpret_cast<const void*>(&norm_bwd_kernel<T, R, TPR, V, FORM, NT>),
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(float) * 2 * V * 8 * TPR));
            }));
        }
    }
    if (bwd) hipLaunchKernelGGL((norm_bwd_kernel<T, R, TPR, V, FORM, NT>), dim3((unsigned)blocks), dim3(L::BLOCK), lds, s, c);
    else hipLaunchKernelGGL((norm_fwd_kernel<T, R, TPR, V, FORM, NT>), dim3((unsigned)blocks), dim3(L::BLOCK), 0, s, c);
    TVAE_CHECK_HIP(hipGetLastError());
    return TVAE_OK;
}
template <typename T, typename R, int FORM, bool NT>
int norm_rows(const RowPlan& p, const NormCall& c, bool bwd, int64_t blocks, hipStream_t s) {
#define X(TPR, V) if (p.tpr == TPR && p.v == V) return norm_rows_launch<T, R, TPR, V, FORM, NT>(c, bwd, blocks, s);
    if constexpr (FORM == TINY) { NORM_TINY_SHAPES(X) } else { NORM_SHAPES(X) }
    if constexpr (FORM != TINY && sizeof(R) == 2) { NORM_NARROW_SHAPES(X) }
#undef X
    return fail(TVAE_ERR_ARG, "norm: no kernel for %d threads a row", p.tpr);
}
template <typename T, typename R>
int norm_rows_form(const RowPlan& p, const NormCall& c, bool bwd, int64_t blocks, hipStream_t s) {
    const NormForm form = norm_form(c);
    const bool nt = norm_streams(c, sizeof(T));
    switch (form) {
        case TINY: return norm_rows<T, R, TINY, false>(p, c, bwd, blocks, s);
        case RAGGED_FUSED: return norm_rows<T, R, RAGGED_FUSED, false>(p, c, bwd, blocks, s);
        case FUSED: return nt ? norm_rows<T, R, FUSED, true>(p, c, bwd, blocks, s) : norm_rows<T, R, FUSED, false>(p, c, bwd, blocks, s);
        default: break;
    }
    // nothing of the residual's type takes part
    if constexpr (sizeof(T) != sizeof(R)) return norm_rows_form<T, T>(p, c, bwd, blocks, s);
    else if (form == RAGGED_PLAIN) return norm_rows<T, T, RAGGED_PLAIN, false>(p, c, bwd, blocks, s);
    else return nt ? norm_rows<T, T, PLAIN, true>(p, c, bwd, blocks, s) : norm_rows<T, T, PLAIN, false>(p, c, bwd, blocks, s);
}

// forward, or the backward pass up to the partial sums (c.chunks = bwd_chunks)
template <typename T, typename R>
int norm_launch(NormCall c, bool bwd, hipStream_t s) {
    if (bwd && (c.dw || c.db) && bwd_small(c.rows, c.d)) {
        const int row_blocks = c.dx || c.dres ? (int)((c.rows + 3) / 4) : 0;
        hipLaunchKernelGGL((norm_bwd_small_kernel<T, R>), dim3((unsigned)(row_blocks + (c.groups + 1) / 2)), dim3(256), 0, s, c, row_blocks);
        TVAE_CHECK_HIP(hipGetLastError());
        return TVAE_OK;
    }
    const RowPlan p = row_plan(c.d, sizeof(R) == 2);
    if (p.tpr) {
        const int64_t turns = (c.rows + plan_rows(p) - 1) / plan_rows(p), most = plan_blocks(p);
        return norm_rows_form<T, R>(p, c, bwd, bwd ? c.chunks : turns < most ? turns : most, s);
    }
    const unsigned blocks = (unsigned)(c.rows < 65536 ? c.rows : 65536);
    if (!bwd) {
        hipLaunchKernelGGL((norm_fwd_wide_kernel<T, R>), dim3(blocks), dim3(256), 0, s, c);
        TVAE_CHECK_HIP(hipGetLastError());
        return TVAE_OK;
    }
    if (c.dx || c.dres) {
        hipLaunchKernelGGL((norm_bwd_wide_kernel<T, R>), dim3(blocks), dim3(256), 0, s, c);
        TVAE_CHECK_HIP(hipGetLastError());
    }
    if (c.dw || c.db) {
        c.chunk_rows = (int)wide_chunk_rows(c.rows);
        hipLaunchKernelGGL((norm_param_wide_kernel<T, R>), dim3((unsigned)((c.groups + 63) / 64), (unsigned)c.chunks), dim3(256), 0, s, c);
        TVAE_CHECK_HIP(hipGetLastError());
    }
    return TVAE_OK;
}

}  // namespace
}  // namespace tvae
