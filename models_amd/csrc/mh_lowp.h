// Element types of the kernels that take fp32, bf16 or fp16 data: loads to fp32, and roundings (to nearest, ties to even) from it.
#pragma once
#include "mh_common.h"

// Host: whether nx rows of wx bytes at x, lx bytes apart, and nd rows of wd bytes at d, ld apart, share a byte.  Rows that are equally far apart may lie
// between each other (columns of one wider buffer); others count as sharing where their ranges do.
static inline bool lp_shared(const void* x, int64_t lx, int64_t wx, int64_t nx, const void* d, int64_t ld, int64_t wd, int64_t nd) {
    if (nx <= 0 || nd <= 0 || wx <= 0 || wd <= 0) return false;
    const int64_t by = (int64_t)(reinterpret_cast<uintptr_t>(d) - reinterpret_cast<uintptr_t>(x));
    if (lx != ld || (nx == 1 && nd == 1)) return by < (nx - 1) * lx + wx && -by < (nd - 1) * ld + wd;
    const int64_t q = by >= 0 ? by / lx : -((-by + lx - 1) / lx), r = by - q * lx;  // row j of d begins r bytes into row j + q of x
    return (r < wx && q < nx && -q < nd) || (r + wd > lx && q + 1 < nx && -(q + 1) < nd);
}

struct lp_bf16 {
    uint16_t u;
};
struct lp_f16 {
    _Float16 h;
};

__device__ __forceinline__ float lp_float(float v) { return v; }
__device__ __forceinline__ float lp_float(lp_bf16 v) { return __uint_as_float((uint32_t)v.u << 16); }
__device__ __forceinline__ float lp_float(lp_f16 v) { return (float)v.h; }

// two values as one word, the first in the low half
__device__ __forceinline__ uint32_t lp_pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((mh_f32x2_t{a, b}), mh_bf16x2_t));
}
typedef _Float16 lp_f16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t lp_pack_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((mh_f32x2_t{a, b}), lp_f16x2_t));
}

// Sixteen bytes that may lie at any element's address: rows of odd length start where they start, and the hardware's unaligned mode (the
// default of the ROCm ABI) loads them in one instruction; a wavefront then touches one line more than an aligned one.
struct __attribute__((packed, aligned(4))) lp_u4_at4 {
    uint32_t x, y, z, w;
};
struct __attribute__((packed, aligned(2))) lp_u4_at2 {
    uint32_t x, y, z, w;
};
template <typename T>
struct lp_vec {
    typedef lp_u4_at2 at;
    static constexpr int N = 8;
};
template <>
struct lp_vec<float> {
    typedef lp_u4_at4 at;
    static constexpr int N = 4;
};

__device__ __forceinline__ uint4 lp_load16(const float* p) {
    const lp_u4_at4 v = *reinterpret_cast<const lp_u4_at4*>(p);
    return make_uint4(v.x, v.y, v.z, v.w);
}
template <typename T>
__device__ __forceinline__ uint4 lp_load16(const T* p) {
    const lp_u4_at2 v = *reinterpret_cast<const lp_u4_at2*>(p);
    return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void lp_unpack(const uint4& w, float (&v)[4], const float*) {
    v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void lp_unpack(const uint4& w, float (&v)[8], const lp_bf16*) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(a[i] << 16);
        v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void lp_unpack(const uint4& w, float (&v)[8], const lp_f16*) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const lp_f16x2_t h = __builtin_bit_cast(lp_f16x2_t, a[i]);
        v[2 * i] = (float)h[0];
        v[2 * i + 1] = (float)h[1];
    }
}
__device__ __forceinline__ void lp_load8(const float* p, float (&v)[8]) {
    float a[4], b[4];
    lp_unpack(lp_load16(p), a, p);
    lp_unpack(lp_load16(p + 4), b, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
}
template <typename T>
__device__ __forceinline__ void lp_load8(const T* p, float (&v)[8]) {
    lp_unpack(lp_load16(p), v, p);
}

// four entries
typedef uint32_t lp_u2_at2 __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ void lp_load4(const float* p, float (&v)[4]) { lp_unpack(lp_load16(p), v, p); }
template <typename T>
__device__ __forceinline__ void lp_load4(const T* p, float (&v)[4]) {
    const lp_u2_at2 w = *reinterpret_cast<const lp_u2_at2*>(p);
    float u[8];
    lp_unpack(make_uint4(w.x, w.y, 0, 0), u, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = u[i];
}

// the sixteen bytes of lp_vec<T>::N rounded values
__device__ __forceinline__ void lp_store16(float* p, const float (&v)[4]) {
    lp_u4_at4 w = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    *reinterpret_cast<lp_u4_at4*>(p) = w;
}
__device__ __forceinline__ void lp_store16(lp_bf16* p, const float (&v)[8]) {
    lp_u4_at2 w = {lp_pack_bf16(v[0], v[1]), lp_pack_bf16(v[2], v[3]), lp_pack_bf16(v[4], v[5]), lp_pack_bf16(v[6], v[7])};
    *reinterpret_cast<lp_u4_at2*>(p) = w;
}
__device__ __forceinline__ void lp_store16(lp_f16* p, const float (&v)[8]) {
    lp_u4_at2 w = {lp_pack_f16(v[0], v[1]), lp_pack_f16(v[2], v[3]), lp_pack_f16(v[4], v[5]), lp_pack_f16(v[6], v[7])};
    *reinterpret_cast<lp_u4_at2*>(p) = w;
}
__device__ __forceinline__ void lp_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void lp_store(lp_bf16* p, float v) { p->u = (uint16_t)lp_pack_bf16(v, 0.f); }
__device__ __forceinline__ void lp_store(lp_f16* p, float v) { p->h = (_Float16)v; }
