// Row access, dropout's keep decisions and launch arguments shared by norms.hip and dropout.hip.
#pragma once
#include "tvae_common.h"

namespace tvae {

typedef _Float16 f16;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// rows start wherever their stride puts them: the 16-byte accesses below promise the alignment of a 16-bit element only
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

// ---- elements <-> fp32 ----------------------------------------------------------------------------------------------------
// NT: past the caches, for streams too long to be found there again
template <bool NT>
__device__ __forceinline__ u32x4 load16(const u32x4_a2* p) {
    if constexpr (NT) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool NT>
__device__ __forceinline__ void put16(u32x4_a2* p, u32x4 v) {
    if constexpr (NT) __builtin_nontemporal_store(v, p);
    else *p = v;
}
// eight elements in their type's own bits, which is what a load in flight keeps in registers
template <typename T> struct Raw8 { u32x4 q[sizeof(T) / 2]; };

// The first nv of four (fp32) or eight (16 bits) elements at p in 16 bytes; the others are 0.  The end of a row that is no whole
// pack comes in pieces of four, two and one element: at most three accesses.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
typedef uint32_t u32_a2 __attribute__((aligned(2)));
template <bool NT>
__device__ __forceinline__ u32x4 load_raw(const float* p, int nv) {
    if (nv >= 4) return load16<NT>(reinterpret_cast<const u32x4_a2*>(p));
    u32x4 q = {0, 0, 0, 0};
    if (nv <= 0) return q;
    if (nv & 2) {
        const u32x2 a = *reinterpret_cast<const u32x2_a2*>(p);
        q[0] = a[0]; q[1] = a[1];
    }
    if (nv & 1) {
        const uint32_t a = reinterpret_cast<const uint32_t*>(p)[nv & 2];
        if (nv & 2) q[2] = a;
        else q[0] = a;
    }
    return q;
}
template <bool NT, typename T>
__device__ __forceinline__ u32x4 load_raw(const T* p, int nv) {
    if (nv >= 8) return load16<NT>(reinterpret_cast<const u32x4_a2*>(p));
    u32x4 q = {0, 0, 0, 0};
    if (nv <= 0) return q;
    if (nv & 4) {
        const u32x2 a = *reinterpret_cast<const u32x2_a2*>(p);
        q[0] = a[0]; q[1] = a[1];
    }
    if (nv & 2) {
        const uint32_t a = *reinterpret_cast<const u32_a2*>(p + (nv & 4));
        if (nv & 4) q[2] = a;
        else q[0] = a;
    }
    if (nv & 1) {
        const uint32_t a = reinterpret_cast<const uint16_t*>(p)[nv & 6];
        const int at = nv >> 1;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (at == e) q[e] = a;
    }
    return q;
}
// the first nv of four 16-bit elements in 8 bytes
template <bool NT, typename T>
__device__ __forceinline__ u32x2 load_half(const T* p, int nv) {
    if (nv >= 4) {
        const u32x2_a2* q = reinterpret_cast<const u32x2_a2*>(p);
        if constexpr (NT) return __builtin_nontemporal_load(q);
        else return *q;
    }
    const u32x4 q = load_raw<false>(p, nv);
    return u32x2{q[0], q[1]};
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float v[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r.q[e >> 2][e & 3]);
}
__device__ __forceinline__ void unpack8(const Raw8<bf16>& r, float v[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(r.q[0][e] << 16); v[2 * e + 1] = __uint_as_float(r.q[0][e] & 0xffff0000u); }
}
__device__ __forceinline__ void unpack8(const Raw8<f16>& r, float v[8]) {
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t w = r.q[0][e];       // a copy: the builtin takes a vector element for the vector's first
        const f16x2 h = __builtin_bit_cast(f16x2, w);
        v[2 * e] = (float)h[0]; v[2 * e + 1] = (float)h[1];
    }
}
__device__ __forceinline__ u32x4 pack4(const float v[4]) {
    return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
__device__ __forceinline__ u32x4 pack8(const float v[8], bf16) {
    u32x4 a;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        a[e] = (uint32_t)__bfloat16_as_ushort(__float2bfloat16(v[2 * e])) | ((uint32_t)__bfloat16_as_ushort(__float2bfloat16(v[2 * e + 1])) << 16);
    return a;
}
__device__ __forceinline__ u32x4 pack8(const float v[8], f16) {
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
    u32x4 a;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const f16x2 h = {(f16)v[2 * e], (f16)v[2 * e + 1]};
        a[e] = __builtin_bit_cast(uint32_t, h);
    }
    return a;
}

// ---- eight elements of a row: which ones, and moving them ----------------------------------------------------------------
// Columns of one lane's eight: col .. col + 3 and second .. second + 3.  Where rows of fp32 take part (SPLIT) the two quads lie
// apart, so that neighbouring lanes take neighbouring 16 bytes of them in each access (and 8 of 16-bit rows); else they are
// neighbours.
struct Cols { uint32_t col, second; };            // unsigned: one 32-bit offset from a scalar row address

template <typename T, bool SPLIT, bool NT>
__device__ __forceinline__ Raw8<T> load_cols(const T* p, const Cols& c, int n_col, int n_second) {
    Raw8<T> r;
    if constexpr (sizeof(T) == 2 && SPLIT) {
        const u32x2 a = load_half<NT>(p + c.col, n_col), b = load_half<NT>(p + c.second, n_second);
        r.q[0] = u32x4{a[0], a[1], b[0], b[1]};
    } else if constexpr (sizeof(T) == 2) {
        r.q[0] = load_raw<NT>(p + c.col, n_col);
    } else {
        // neighbouring quads: each line comes with two accesses, so it has to stay for the second
        r.q[0] = load_raw<NT && SPLIT>(p + c.col, n_col);
        r.q[1] = load_raw<NT && SPLIT>(p + c.second, SPLIT ? n_second : n_col - 4);
    }
    return r;
}
__device__ __forceinline__ void store_part(float* p, int nv, u32x4 q) {         // nv < 4
    if (nv <= 0) return;
    if (nv & 2) *reinterpret_cast<u32x2_a2*>(p) = u32x2{q[0], q[1]};
    if (nv & 1) reinterpret_cast<uint32_t*>(p)[nv & 2] = nv & 2 ? q[2] : q[0];
}
template <typename T>
__device__ __forceinline__ void store_part(T* p, int nv, u32x4 q) {             // nv < 8
    if (nv <= 0) return;
    if (nv & 4) *reinterpret_cast<u32x2_a2*>(p) = u32x2{q[0], q[1]};
    if (nv & 2) *reinterpret_cast<u32_a2*>(p + (nv & 4)) = nv & 4 ? q[2] : q[0];
    if (nv & 1) {
        const int at = nv >> 1;
        const uint32_t a = at & 2 ? (at & 1 ? q[3] : q[2]) : (at & 1 ? q[1] : q[0]);
        reinterpret_cast<uint16_t*>(p)[nv & 6] = (uint16_t)a;
    }
}
// n_col, n_second: elements of the row from col and second on (neighbouring quads: n_col says both)
template <bool SPLIT, bool NT>
__device__ __forceinline__ void store_cols(float* p, const Cols& c, int n_col, int n_second, const float v[8]) {
    const int n[2] = {n_col, SPLIT ? n_second : n_col - 4};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float* q = p + (i ? c.second : c.col);
        if (n[i] >= 4) put16<NT && SPLIT>(reinterpret_cast<u32x4_a2*>(q), pack4(v + 4 * i));
        else store_part(q, n[i], pack4(v + 4 * i));
    }
}
template <bool SPLIT, bool NT, typename T>
__device__ __forceinline__ void store_cols(T* p, const Cols& c, int n_col, int n_second, const float v[8]) {
    if constexpr (SPLIT) {
        const u32x4 q = pack8(v, T{});
        const int n[2] = {n_col, n_second};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            T* at = p + (i ? c.second : c.col);
            const u32x2 h = {q[2 * i], q[2 * i + 1]};
            if (n[i] < 4) store_part(at, n[i], u32x4{h[0], h[1], 0, 0});
            else if constexpr (NT) __builtin_nontemporal_store(h, reinterpret_cast<u32x2_a2*>(at));
            else *reinterpret_cast<u32x2_a2*>(at) = h;
        }
    } else if (n_col >= 8) put16<NT>(reinterpret_cast<u32x4_a2*>(p + c.col), pack8(v, T{}));
    else store_part(p + c.col, n_col, pack8(v, T{}));
}
// eight neighbours from column col on, nv of them in the row
template <typename T>
__device__ __forceinline__ void load8(const T* p, int col, int nv, float v[8]) {
    unpack8(load_cols<T, false, false>(p, Cols{(uint32_t)col, (uint32_t)col + 4}, nv, nv - 4), v);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int col, int nv, const float v[8]) {
    store_cols<false, false>(p, Cols{(uint32_t)col, (uint32_t)col + 4}, nv, nv - 4, v);
}

// ---- rows of a tensor whose leading axes have at most two strides: element (i, c) at (i / grp) * so + (i % grp) * si + c -----
struct RowsOf { long long so, si; };
__device__ __forceinline__ long long row_offset(const RowsOf& s, int grp, long long row) {
    if (grp == 1) return row * s.so;
    const unsigned r = (unsigned)row, q = r / (unsigned)grp;      // rows < 2^31
    return (long long)q * s.so + (long long)(r - q * (unsigned)grp) * s.si;
}

// ---- dropout's keep decisions ------------------------------------------------------------------------------------------
// A pure function of (seed, offset, row, column): nothing is stored, the backward pass evaluates it again, and it does not
// depend on strides, on the launch or on which operator asks.  Philox4x32 with ten rounds (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011): key = seed, counter = (column / 8, row, offset low, offset high);
// the four words are eight 16-bit draws for eight neighbouring columns, low half first.  One evaluation thus serves eight
// elements, half the integer work of 32-bit draws; p is in force as the nearest multiple of 2^-16, and the scale is that
// value's own, so the result is unbiased for it.
struct DropoutArgs {
    const int64_t* rng;         // device {seed, offset}, read by the kernel; null: the two words below
    uint64_t seed, offset;
    uint32_t threshold;         // round(65536 p): an element is dropped where its draw is below it; 0 = no dropout
    float scale;                // 65536 / (65536 - threshold); 0 where everything is dropped
};
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }
struct Philox {
    uint32_t k0, k1, c2, c3;
    __device__ __forceinline__ explicit Philox(const DropoutArgs& a) {
        const uint64_t s = a.rng ? (uint64_t)a.rng[0] : a.seed, o = a.rng ? (uint64_t)a.rng[1] : a.offset;
        k0 = (uint32_t)s; k1 = (uint32_t)(s >> 32);
        c2 = (uint32_t)o; c3 = (uint32_t)(o >> 32);
    }
    __device__ __forceinline__ u32x4 words(uint32_t group, uint32_t row) const {
        uint32_t a = group, b = row, c = c2, d = c3, x = k0, y = k1;
#pragma unroll
        for (int r = 0; r < 10; ++r) {
            const uint64_t p = (uint64_t)a * 0xD2511F53u, q = (uint64_t)c * 0xCD9E8D57u;
            a = xor3((uint32_t)(q >> 32), b, x); b = (uint32_t)q;
            c = xor3((uint32_t)(p >> 32), d, y); d = (uint32_t)p;
            x += 0x9E3779B9u; y += 0xBB67AE85u;
        }
        return u32x4{a, b, c, d};
    }
};
// bit e: element e of the group is kept
__device__ __forceinline__ uint32_t keep8(const Philox& ph, const DropoutArgs& a, uint32_t group, uint32_t row) {
    const u32x4 w = ph.words(group, row);
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t u = (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
        bits |= u < a.threshold ? 0u : 1u << e;
    }
    return bits;
}
// v[e] <- kept ? v[e] * scale : 0.  A dropped infinity or NaN becomes 0: the element is replaced, not multiplied.
__device__ __forceinline__ void drop8(uint32_t kept, float scale, float v[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = kept >> e & 1 ? v[e] * scale : 0.f;
}
__device__ __forceinline__ void drop8(const Philox& ph, const DropoutArgs& a, uint32_t group, uint32_t row, float v[8]) {
    const u32x4 w = ph.words(group, row);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t u = (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu;
        v[e] = u < a.threshold ? 0.f : v[e] * a.scale;
    }
}

// threshold and scale of a drop probability; false: p is outside [0, 1] or not a number
bool dropout_args(double p, const int64_t* rng, uint64_t seed, uint64_t offset, DropoutArgs* out);

inline bool norm_dtype_ok(int t) { return t == TVAE_F32 || t == TVAE_BF16 || t == TVAE_F16; }

}  // namespace tvae
