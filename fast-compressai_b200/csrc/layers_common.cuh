// layers_common.cuh -- element types, activations and 8-bit blocks shared by
// the pointwise layers (linear_tc.cu, rowwise.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <float.h>
#include <stdint.h>

#include "../../include/fcai_layers.h"
#include "fcai_common.h"

namespace ly {

// ---- element types ----------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&v);
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) {
    return __half22float2(*reinterpret_cast<__half2 *>(&w));
}

// ---- activations --------------------------------------------------------------
__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 values in a register pair: sm_100 computes both with one
// instruction, which halves the arithmetic of the epilogues and elementwise
// kernels (they are otherwise bound by instruction issue with GELU).
struct F2 {
    uint64_t r;
};
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v.r) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ float2 split(F2 v) {
    float2 o;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(v.r));
    return o;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v.r) : "l"(a.r), "l"(b.r), "l"(c.r));
    return v;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v.r) : "l"(a.r), "l"(b.r));
    return v;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v.r) : "l"(a.r), "l"(b.r));
    return v;
}

// Eight consecutive elements from / to a 16-byte aligned address (f32: two
// 16-byte accesses).
template <typename T> struct Vec8 {
    static __device__ __forceinline__ void load(const T *p, float (&v)[8]) {
        const uint4 q = __ldg(reinterpret_cast<const uint4 *>(p));
        unpack(q, v);
    }
    static __device__ __forceinline__ void unpack(const uint4 &q, float (&v)[8]) {
        const float2 a = unpack2(q.x, T()), b = unpack2(q.y, T()), c = unpack2(q.z, T()), d = unpack2(q.w, T());
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
    }
    static __device__ __forceinline__ void store(T *p, const float (&v)[8]) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()),
                                                   pack2(v[4], v[5], T()), pack2(v[6], v[7], T()));
    }
};
template <> struct Vec8<float> {
    static __device__ __forceinline__ void load(const float *p, float (&v)[8]) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(p));
        const float4 b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    static __device__ __forceinline__ void store(float *p, const float (&v)[8]) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
};

// Eight values as pairs.
struct V8 {
    F2 p[4];
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = f2(v[2 * i], v[2 * i + 1]);
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = split(p[i]);
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
};
__device__ __forceinline__ float hsum(F2 v) {
    const float2 f = split(v);
    return f.x + f.y;
}

// The normal distribution's upper tail Q(t) = erfc(t / sqrt 2) / 2, t >= 0, as
// e * R(u) with e = exp(-t^2 / 2), u = 1 / (1 + 0.24 t) and R a polynomial
// without constant term, the form of Hastings' approximations (Approximations
// for Digital Computers, 1955).  The coefficients are a fit of this project's
// own: iteratively reweighted least squares of R against Q e^(t^2/2) on
// t in [0, 40], largest relative error 7.6e-7 evaluated in fp32.  `e` comes
// back for the density.
// One reciprocal serves the pair (1 / a = b / (a b)): the special function
// unit, not the arithmetic, bounds GELU.  The last bits of a value then depend on
// the other one, so pairs of two rows (kApart) take a reciprocal each: a row's
// results are the same whatever stands beside it.  t <= 30, where Q is zero in fp32.
template <bool kApart>
__device__ __forceinline__ F2 normal_tail2(F2 t, F2 &e) {
    const float2 a = split(mul2(mul2(t, f2(-0.72134752f)), t));  // log2(e) / 2
    const float2 d = split(fma2(f2(0.24f), t, f2(1.f)));
    e = f2(ex2_approx(a.x), ex2_approx(a.y));
    const F2 u = kApart ? f2(rcp_approx(d.x), rcp_approx(d.y)) : mul2(f2(d.y, d.x), f2(rcp_approx(d.x * d.y)));
    F2 r = fma2(u, f2(-0.0529928472f), f2(0.152797519f));
    r = fma2(u, r, f2(-0.0657069748f));
    r = fma2(u, r, f2(0.118390834f));
    r = fma2(u, r, f2(0.0633970503f));
    r = fma2(u, r, f2(0.0928386496f));
    r = fma2(u, r, f2(0.0955221622f));
    r = fma2(u, r, f2(0.0957537928f));
    return mul2(e, mul2(u, r));
}
// min(|x|, 30), 30 for a NaN: the pair's shared reciprocal must not carry one
// value's NaN into the other.
__device__ __forceinline__ F2 tail_arg(float2 x) { return f2(fminf(fabsf(x.x), 30.f), fminf(fabsf(x.y), 30.f)); }
__device__ __forceinline__ float relu_nan(float x) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(0.f));
    return y;
}
__device__ __forceinline__ float clamp_nan(float x) {  // to +-30; a NaN stays
    float y;
    asm("{\n\t.reg .f32 t;\n\tmin.NaN.f32 t, %1, %2;\n\tmax.NaN.f32 %0, t, %3;\n\t}" : "=f"(y) : "f"(x), "f"(30.f), "f"(-30.f));
    return y;
}
__device__ __forceinline__ float finite(float x) {  // to +-FLT_MAX: the smaller magnitude, with x's sign
    float y;
    asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(FLT_MAX));
    return y;
}
// x Phi(x) = max(x, 0) - |x| Q(|x|)
template <bool kApart>
__device__ __forceinline__ F2 gelu2(F2 v) {
    const float2 x = split(v);
    F2 e;
    const F2 t = tail_arg(x);
    return fma2(mul2(t, f2(-1.f)), normal_tail2<kApart>(t, e), f2(relu_nan(x.x), relu_nan(x.y)));
}
// its derivative, Phi(x) + x phi(x)
__device__ __forceinline__ F2 gelu_grad2(F2 v) {
    const float2 x = split(v);
    F2 e;
    const F2 q = normal_tail2<false>(tail_arg(x), e);
    const float2 lo = split(q), hi = split(fma2(q, f2(-1.f), f2(1.f)));
    const F2 cdf = f2(x.x < 0.f ? lo.x : hi.x, x.y < 0.f ? lo.y : hi.y);
    return fma2(mul2(f2(clamp_nan(x.x), clamp_nan(x.y)), e), f2(0.398942280f), cdf);
}
// Exponential and reciprocal flush to zero: SiLU and its derivative are 0 below
// x = -87.3, where they are less than 1.2e-36, for one special function each.
__device__ __forceinline__ F2 sigmoid2(F2 x) {
    const float2 a = split(mul2(x, f2(-1.44269504f)));
    const float2 d = split(add2(f2(ex2_approx(a.x), ex2_approx(a.y)), f2(1.f)));
    return f2(rcp_approx(d.x), rcp_approx(d.y));
}

// v = act(v) of kN pairs; `kind` is the same for the whole kernel.  kApart: the
// values of a pair belong to different rows.
template <int kN, bool kApart = false>
__device__ __forceinline__ void act_n(int kind, F2 (&v)[kN]) {
    if (kind == FCAI_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const float2 x = split(v[i]);
            v[i] = f2(x.x < 0.f ? 0.f : x.x, x.y < 0.f ? 0.f : x.y);  // a NaN stays
        }
    } else if (kind == FCAI_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = gelu2<kApart>(v[i]);
    } else if (kind == FCAI_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = mul2(v[i], sigmoid2(v[i]));
    }
}
// g *= act'(x)
template <int kN>
__device__ __forceinline__ void act_grad_n(int kind, const F2 (&x)[kN], F2 (&g)[kN]) {
    if (kind == FCAI_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            // a choice, not a product: an infinite gradient does not meet a zero, and a NaN x passes the gradient on
            const float2 xx = split(x[i]), gg = split(g[i]);
            g[i] = f2(xx.x <= 0.f ? 0.f : gg.x, xx.y <= 0.f ? 0.f : gg.y);
        }
    } else if (kind == FCAI_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < kN; ++i) g[i] = mul2(g[i], gelu_grad2(x[i]));
    } else if (kind == FCAI_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const F2 s = sigmoid2(x[i]);
            // x as a finite number: where it is infinite, s or 1 - s is zero and the limit is wanted, not a NaN.
            // A NaN comes through s.  16-bit types reach infinities from values of 65520 on.
            const float2 xx = split(x[i]);
            const F2 xf = f2(finite(xx.x), finite(xx.y));
            g[i] = mul2(g[i], mul2(s, fma2(xf, fma2(s, f2(-1.f), f2(1.f)), f2(1.f))));
        }
    }
}
__device__ __forceinline__ float act_1(int kind, float x) {
    F2 v[1] = {f2(x, 0.f)};
    act_n(kind, v);
    return split(v[0]).x;
}

// ---- 8-bit blocks ---------------------------------------------------------------
// The scale of a block from its largest magnitude (given NaN or infinity when
// the block holds one), and the reciprocal its values are multiplied by.
template <bool kE4m3>
__device__ __forceinline__ float block_scale(float amax) {
    constexpr float kInvTop = kE4m3 ? 1.f / 448.f : 1.f / 127.f;
    const float s = fmaxf(__fmul_rn(amax, kInvTop), FLT_MIN);
    return amax <= FLT_MAX ? s : __int_as_float(0x7FC00000);
}
// max that keeps a NaN of either side.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// Codes of four values times inv.  The products are rounded before they become
// codes, as the definition says.  int8 without conversion instructions, which run at an
// eighth of the rate: adding 1.5 * 2^23 leaves the integer, ties to even, in
// the low bits; |x * inv| <= 127 (1 + 2^-22), so no code leaves its range, and
// a NaN block's codes, whatever they are, read back as NaN.
template <bool kE4m3>
__device__ __forceinline__ uint32_t encode4(F2 a, F2 b, float inv) {
    if (kE4m3) {
        a = mul2(a, f2(inv));
        b = mul2(b, f2(inv));
        const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(split(a), __NV_SATFINITE, __NV_E4M3);
        const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(split(b), __NV_SATFINITE, __NV_E4M3);
        return (uint32_t)lo | ((uint32_t)hi << 16);
    }
    // The sum is written as a product with 1: a packed product and sum can come
    // out as one fused operation, which would round once.
    const float2 x = split(fma2(mul2(a, f2(inv)), f2(1.f), f2(12582912.f)));
    const float2 y = split(fma2(mul2(b, f2(inv)), f2(1.f), f2(12582912.f)));
    const uint32_t lo = __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}
template <bool kE4m3>
__device__ __forceinline__ uint2 encode8(const V8 &v, float inv) {
    return make_uint2(encode4<kE4m3>(v.p[0], v.p[1], inv), encode4<kE4m3>(v.p[2], v.p[3], inv));
}
// Four codes times scale.  int8: the byte with its sign flipped becomes the low
// bits of 2^23, and 2^23 + 128 is taken off again.
template <bool kE4m3>
__device__ __forceinline__ void decode4(uint32_t w, float scale, F2 &a, F2 &b) {
    if (kE4m3) {
        const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3);
        const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
        const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&lo));
        const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
        a = f2(x.x, x.y), b = f2(y.x, y.y);
    } else {
        w ^= 0x80808080u;
        auto at = [&](uint32_t sel) { return __uint_as_float(__byte_perm(w, 0x4B000000u, sel)); };
        a = add2(f2(at(0x7440), at(0x7441)), f2(-8388736.f));
        b = add2(f2(at(0x7442), at(0x7443)), f2(-8388736.f));
    }
    a = mul2(a, f2(scale));
    b = mul2(b, f2(scale));
}

inline int dtype_size(int dtype) { return dtype == FCAI_DTYPE_F32 ? 4 : 2; }
inline bool aligned16(const void *p, int64_t ld, int dtype) {
    return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * dtype_size(dtype))) & 15) == 0;
}

}  // namespace ly
