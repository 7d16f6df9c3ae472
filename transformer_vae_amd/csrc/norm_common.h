// Row access, dropout's keep decisions and launch arguments shared by norms.hip and dropout.hip.
#pragma once
#include "tvae_common.h"

namespace tvae {

typedef _Float16 f16;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// rows start wherever their stride puts them, so the 16-byte accesses below promise the element's own alignment only
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

// ---- eight neighbouring elements <-> fp32 ----------------------------------------------------------------------------
__device__ __forceinline__ void load8_full(const float* p, float v[8]) {
    const u32x4 a = *reinterpret_cast<const u32x4_a4*>(p), b = *reinterpret_cast<const u32x4_a4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = __uint_as_float(a[e]); v[4 + e] = __uint_as_float(b[e]); }
}
__device__ __forceinline__ void load8_full(const bf16* p, float v[8]) {
    const u32x4 a = *reinterpret_cast<const u32x4_a2*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(a[e] << 16); v[2 * e + 1] = __uint_as_float(a[e] & 0xffff0000u); }
}
__device__ __forceinline__ void load8_full(const f16* p, float v[8]) {
    const u32x4 a = *reinterpret_cast<const u32x4_a2*>(p);
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t w = a[e];        // a copy: the builtin takes a vector element for the vector's first
        const f16x2 h = __builtin_bit_cast(f16x2, w);
        v[2 * e] = (float)h[0]; v[2 * e + 1] = (float)h[1];
    }
}
// the first nv (1..8) of eight; the others read as 0
template <typename T>
__device__ __forceinline__ void load8(const T* p, int nv, float v[8]) {
    if (nv >= 8) {
        load8_full(p, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < nv ? to_f32(p[e]) : 0.f;
    }
}
__device__ __forceinline__ void store8_full(float* p, const float v[8]) {
    u32x4 a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) { a[e] = __float_as_uint(v[e]); b[e] = __float_as_uint(v[4 + e]); }
    *reinterpret_cast<u32x4_a4*>(p) = a;
    *reinterpret_cast<u32x4_a4*>(p + 4) = b;
}
__device__ __forceinline__ void store8_full(bf16* p, const float v[8]) {
    u32x4 a;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        a[e] = (uint32_t)__bfloat16_as_ushort(__float2bfloat16(v[2 * e])) | ((uint32_t)__bfloat16_as_ushort(__float2bfloat16(v[2 * e + 1])) << 16);
    *reinterpret_cast<u32x4_a2*>(p) = a;
}
__device__ __forceinline__ void store8_full(f16* p, const float v[8]) {
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
    u32x4 a;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const f16x2 h = {(f16)v[2 * e], (f16)v[2 * e + 1]};
        a[e] = __builtin_bit_cast(uint32_t, h);
    }
    *reinterpret_cast<u32x4_a2*>(p) = a;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int nv, const float v[8]) {
    if (nv >= 8) {
        store8_full(p, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < nv) p[e] = from_f32<T>(v[e]);
    }
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
            a = (uint32_t)(q >> 32) ^ b ^ x; b = (uint32_t)q;
            c = (uint32_t)(p >> 32) ^ d ^ y; d = (uint32_t)p;
            x += 0x9E3779B9u; y += 0xBB67AE85u;
        }
        return u32x4{a, b, c, d};
    }
};
// v[e] <- kept ? v[e] * scale : 0.  A dropped infinity or NaN becomes 0: the element is replaced, not multiplied.
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
