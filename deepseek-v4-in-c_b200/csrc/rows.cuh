// rows.cuh - typed rows in 8-element groups, and rotary angles: what rope.cu,
// kvq.cu and logits.cu share.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "tree.h"

namespace dsv4b {

__host__ __device__ constexpr int row_dt_size(int dt) { return dt == DSV4B_F32 ? 4 : 2; }

// One element of a typed array (F32, BF16 or F16) as float.
template <int DT>
__device__ __forceinline__ float ld_row1(const void *p, size_t i)
{
    if constexpr (DT == DSV4B_F32) return __ldcg(reinterpret_cast<const float *>(p) + i);
    const unsigned short u = __ldcg(reinterpret_cast<const unsigned short *>(p) + i);
    if constexpr (DT == DSV4B_BF16) return __uint_as_float((uint32_t)u << 16);
    return __half2float(__ushort_as_half(u));
}

template <int DT>
__device__ __forceinline__ void st_row1(void *p, size_t i, float v)
{
    if constexpr (DT == DSV4B_F32) reinterpret_cast<float *>(p)[i] = v;
    else if constexpr (DT == DSV4B_BF16) reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half *>(p)[i] = __float2half_rn(v);
}

// Elements i .. i + 8: 16-byte accesses where VEC (the caller has checked
// the alignment), else element by element. raw8 keeps the loaded words so
// that several groups can be in flight before any is converted.
template <int DT>
struct Raw8 {
    uint4 w[DT == DSV4B_F32 ? 2 : 1];
};

template <int DT, bool VEC>
__device__ __forceinline__ Raw8<DT> ld_raw8(const void *p, size_t i)
{
    Raw8<DT> r;
    if constexpr (VEC) {
        const uint4 *q = reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(p) + i * row_dt_size(DT));
#pragma unroll
        for (int k = 0; k < (DT == DSV4B_F32 ? 2 : 1); k++) r.w[k] = __ldcg(q + k);
    } else if constexpr (DT == DSV4B_F32) {
        const unsigned *q = reinterpret_cast<const unsigned *>(p) + i;
        r.w[0] = make_uint4(__ldcg(q), __ldcg(q + 1), __ldcg(q + 2), __ldcg(q + 3));
        r.w[1] = make_uint4(__ldcg(q + 4), __ldcg(q + 5), __ldcg(q + 6), __ldcg(q + 7));
    } else {
        const unsigned short *q = reinterpret_cast<const unsigned short *>(p) + i;
        unsigned u[4];
#pragma unroll
        for (int k = 0; k < 4; k++) u[k] = (unsigned)__ldcg(q + 2 * k) | ((unsigned)__ldcg(q + 2 * k + 1) << 16);
        r.w[0] = make_uint4(u[0], u[1], u[2], u[3]);
    }
    return r;
}

template <int DT>
__device__ __forceinline__ void widen8(const Raw8<DT> &r, float (&v)[8])
{
    const unsigned u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
    if constexpr (DT == DSV4B_F32) {
        const unsigned t[4] = {r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[k] = __uint_as_float(u[k]);
            v[4 + k] = __uint_as_float(t[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            float2 f;
            if constexpr (DT == DSV4B_BF16) f = bf16x2(u[k]);
            else f = __half22float2(*reinterpret_cast<const __half2 *>(&u[k]));
            v[2 * k] = f.x;
            v[2 * k + 1] = f.y;
        }
    }
}

// Two floats as one word of two DT values, rounded to nearest even.
template <int DT>
__device__ __forceinline__ unsigned pack2(float a, float b)
{
    if constexpr (DT == DSV4B_BF16) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const unsigned *>(&t);
    } else {
        const __half2 t = __floats2half2_rn(a, b);
        return *reinterpret_cast<const unsigned *>(&t);
    }
}

template <int DT, bool VEC>
__device__ __forceinline__ void st_row8(void *p, size_t i, const float (&v)[8])
{
    if constexpr (!VEC) {
#pragma unroll
        for (int k = 0; k < 8; k++) st_row1<DT>(p, i + k, v[k]);
    } else {
        uint4 *q = reinterpret_cast<uint4 *>(reinterpret_cast<char *>(p) + i * row_dt_size(DT));
        if constexpr (DT == DSV4B_F32) {
            q[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            q[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
        } else {
            q[0] = make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7]));
        }
    }
}

// Cosine and sine of pos * freq. The product and its reduction to [-pi/4,
// pi/4] are in double (pi/2 as a double and its remainder: for |angle| < 2^31
// the reduction adds less than 1e-15 to the product's own rounding, which is
// 2^-53 of the angle: 2^-33 at 2^20 radians), and so are the Taylor sums,
// cut at r^13 / 13! and r^12 / 12!, which leaves less than 2^-40: the one
// rounding that counts is the float's. Twelve independent-by-halves fused
// steps, where the general double functions take 5 us of an 8 us rotation.
__device__ __forceinline__ float2 rope_angle(int pos, double freq)
{
    const double th = (double)pos * freq;
    const double n = rint(th * 0.63661977236758134);
    double r = fma(-n, 1.5707963267948966, th);
    r = fma(-n, 6.123233995736766e-17, r);
    const double z = r * r;
    double s = fma(z, 1.0 / 6227020800.0, -1.0 / 39916800.0);
    double c = fma(z, 1.0 / 479001600.0, -1.0 / 3628800.0);
    s = fma(z, s, 1.0 / 362880.0);
    c = fma(z, c, 1.0 / 40320.0);
    s = fma(z, s, -1.0 / 5040.0);
    c = fma(z, c, -1.0 / 720.0);
    s = fma(z, s, 1.0 / 120.0);
    c = fma(z, c, 1.0 / 24.0);
    s = fma(z, s, -1.0 / 6.0);
    c = fma(z, c, -0.5);
    const float fs = (float)fma(r * z, s, r), fc = (float)fma(z, c, 1.0);
    const int q = (int)__double2ll_rn(n) & 3;      // quarter turns
    const float x = q & 1 ? fs : fc, y = q & 1 ? fc : fs;
    return make_float2((q + 1) & 2 ? -x : x, q & 2 ? -y : y);
}

// (a, b) turned by the angle of cs = (cos, sin), each product rounded.
__device__ __forceinline__ void turn(float &a, float &b, float2 cs)
{
    const float x = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
    b = __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x));
    a = x;
}

// Runs F<type constant> for a checked row type.
#define DSV4B_ROW_DT(dt, NAME, ...)                     \
    do {                                                \
        if ((dt) == DSV4B_F32) {                        \
            constexpr int NAME = DSV4B_F32;             \
            __VA_ARGS__;                                \
        } else if ((dt) == DSV4B_BF16) {                \
            constexpr int NAME = DSV4B_BF16;            \
            __VA_ARGS__;                                \
        } else {                                        \
            constexpr int NAME = DSV4B_F16;             \
            __VA_ARGS__;                                \
        }                                               \
    } while (0)

}  // namespace dsv4b
