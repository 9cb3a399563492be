// Quantisation of a group of values to 8 or 4 bits, and its inverse.
//
//   s = max(fl32(a * fl32(1 / qmax)), 2^-126), a = max |x_k|;   q_k = nearest(x_k / s), halves to even.
//
// The codes are exact: x_k and s are taken as they are, and the quotient is
// never rounded to the wrong side of a border between two codes.
//
//   FP32 rows. q0 = rint(x * r), r = 1/s to 2^-22, is off by at most one, and
//   x - q0 s = fma(-q0, s, x) is exact (a multiple of ulp(s)/2 below 0.51 s),
//   so comparing twice its magnitude with s settles it.
//
//   FP16 rows. x / s = (qmax x / a)(1 + d) with |d| < 2^-22, and qmax x / a
//   is a quotient of whole numbers (11-bit significands): it is a half, or at
//   least 2^-19 (relative) away from one. So x * r, r = 1/s to 2^-22, is on
//   the right side but where qmax x / a is a half exactly. Then the sign of
//   s - a / qmax decides, which fma(s, qmax, -a) gives exactly: scaling r by
//   1 -+ 2^-21 moves those products to the side they belong to and no other
//   one across a border. Where s = a / qmax exactly (8 of 1024 significands
//   at 8 bits), the quotient can be a half, and one correction step, t +
//   fma(-t, s, x) * r, returns it correctly rounded. It was checked for all
//   pairs of significands, and costs a multiply and an add per value instead
//   of a division; the rare groups (that case, and groups that are not finite)
//   take a slower path together with their warp.
#pragma once

#include <cstdint>
#include <cuda_fp16.h>

#include "sm100.cuh"

namespace dnb {

constexpr float kTinyScale = 1.17549435e-38f;  // 2^-126
constexpr float kRint = 12582912.f;            // 1.5 * 2^23: adding it rounds to a whole number, held in the low bits

// One group's scale and what the codes are made with.
struct GroupScale {
    float s;    // NaN for a group that holds a NaN or an infinity
    float r;    // 1 / s, biased (FP16)
    bool rare;  // the codes need codes8_rare
};

__device__ __forceinline__ float reciprocal(float x) {  // to 1 ulp
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Magnitude bits of 8 packed fp16 values / of fp32 values: the unsigned
// maximum orders finite < infinity < NaN.
__device__ __forceinline__ uint32_t umax16x2(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }

template <typename T>
struct QuantOf;

template <>
struct QuantOf<__half> {
    static constexpr bool kF32 = false;
    struct Vec {  // 8 values
        uint4 v;
    };
    __device__ static __forceinline__ Vec zero() { return Vec{make_uint4(0, 0, 0, 0)}; }
    __device__ static __forceinline__ Vec load(const __half* p) { return Vec{__ldg(reinterpret_cast<const uint4*>(p))}; }
    __device__ static __forceinline__ Vec load_some(const __half* p, int n) {  // the first n of 8, any alignment
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) w[i >> 1] |= static_cast<uint32_t>(__half_as_ushort(p[i])) << ((i & 1) * 16);
        return Vec{make_uint4(w[0], w[1], w[2], w[3])};
    }
    __device__ static __forceinline__ Vec load_local(const __half (&h)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = static_cast<uint32_t>(__half_as_ushort(h[2 * i])) | static_cast<uint32_t>(__half_as_ushort(h[2 * i + 1])) << 16;
        return Vec{make_uint4(w[0], w[1], w[2], w[3])};
    }
    __device__ static __forceinline__ Vec only(Vec x, int lo, int hi) {  // elements outside [lo, hi) as zeros
        uint32_t w[4] = {x.v.x, x.v.y, x.v.z, x.v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] &= (2 * i >= lo && 2 * i < hi ? 0xffffu : 0u) | (2 * i + 1 >= lo && 2 * i + 1 < hi ? 0xffff0000u : 0u);
        return Vec{make_uint4(w[0], w[1], w[2], w[3])};
    }
    __device__ static __forceinline__ uint32_t mag(const Vec& x) {
        const uint32_t m = 0x7fff7fffu;
        const uint32_t a = umax16x2(umax16x2(x.v.x & m, x.v.y & m), umax16x2(x.v.z & m, x.v.w & m));
        return max(a >> 16, a & 0xffffu);
    }
    __device__ static __forceinline__ uint32_t mag1(__half x) { return __half_as_ushort(x) & 0x7fffu; }
    __device__ static __forceinline__ float mag_value(uint32_t bits) {
        return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
    }
    __device__ static __forceinline__ void unpack(const Vec& x, float (&f)[8]) { h8_to_f(x.v, f); }
};

template <>
struct QuantOf<float> {
    static constexpr bool kF32 = true;
    struct Vec {
        float4 a, b;
    };
    __device__ static __forceinline__ Vec zero() {
        return Vec{make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    }
    __device__ static __forceinline__ Vec load(const float* p) {
        return Vec{__ldg(reinterpret_cast<const float4*>(p)), __ldg(reinterpret_cast<const float4*>(p) + 1)};
    }
    __device__ static __forceinline__ Vec load_local(const float (&f)[8]) {
        return Vec{make_float4(f[0], f[1], f[2], f[3]), make_float4(f[4], f[5], f[6], f[7])};
    }
    __device__ static __forceinline__ Vec only(const Vec& x, int lo, int hi) {
        float f[8];
        unpack(x, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i >= lo && i < hi ? f[i] : 0.f;
        return Vec{make_float4(f[0], f[1], f[2], f[3]), make_float4(f[4], f[5], f[6], f[7])};
    }
    __device__ static __forceinline__ Vec load_some(const float* p, int n) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < n ? p[i] : 0.f;
        return Vec{make_float4(f[0], f[1], f[2], f[3]), make_float4(f[4], f[5], f[6], f[7])};
    }
    __device__ static __forceinline__ void unpack(const Vec& x, float (&f)[8]) {
        f[0] = x.a.x, f[1] = x.a.y, f[2] = x.a.z, f[3] = x.a.w;
        f[4] = x.b.x, f[5] = x.b.y, f[6] = x.b.z, f[7] = x.b.w;
    }
    __device__ static __forceinline__ uint32_t mag(const Vec& x) {
        float f[8];
        unpack(x, f);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
        return m;
    }
    __device__ static __forceinline__ uint32_t mag1(float x) { return __float_as_uint(x) & 0x7fffffffu; }
    __device__ static __forceinline__ float mag_value(uint32_t bits) { return __uint_as_float(bits); }
};

template <typename T>
__device__ __forceinline__ GroupScale group_scale(uint32_t mag, float qmax) {
    const float a = QuantOf<T>::mag_value(mag);
    GroupScale g;
    g.s = fmaxf(__fmul_rn(a, qmax == 127.f ? 1.f / 127.f : 1.f / 7.f), kTinyScale);
    g.r = reciprocal(g.s);
    if (QuantOf<T>::kF32) {
        g.rare = !(a <= 3.402823466e38f);
    } else {
        const float d = fmaf(g.s, qmax, -a);  // exact sign of s - a / qmax
        g.r *= d > 0.f ? 1.f - 4.76837158e-7f : 1.f + 4.76837158e-7f;
        g.rare = !(d > 0.f || d < 0.f);  // exact, or not finite
    }
    if (!(a <= 3.402823466e38f)) g.s = __uint_as_float(0x7fc00000u);
    return g;
}

// The low byte of each of 8 words.
__device__ __forceinline__ uint2 low_bytes(const uint32_t (&u)[8]) {
    uint2 w;
    w.x = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
    w.y = __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410);
    return w;
}

// Codes of 8 FP16 values of a group that is not rare, one a byte.
__device__ __forceinline__ uint2 codes8_fast(const QuantOf<__half>::Vec& x, float r) {
    float f[8];
    QuantOf<__half>::unpack(x, f);
    const float2 r2 = make_float2(r, r), zero2 = make_float2(0.f, 0.f);
    const float2 magic2 = make_float2(kRint, kRint), one2 = make_float2(1.f, 1.f);
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = ffma2(ffma2(make_float2(f[2 * i], f[2 * i + 1]), r2, zero2), one2, magic2);
        u[2 * i] = __float_as_uint(t.x);
        u[2 * i + 1] = __float_as_uint(t.y);
    }
    return low_bytes(u);
}

// The code of one value of any group, in the low byte.
template <typename T>
__device__ __forceinline__ uint32_t code1f(float x, const GroupScale& g) {
    const float v = g.s == g.s ? x : 0.f;  // a group that is not finite: codes 0
    if (QuantOf<T>::kF32) {
        const float q0 = __fsub_rn(__fmaf_rn(v, g.r, kRint), kRint);
        const float rest = __fmaf_rn(-q0, g.s, v);
        const float two = 2.f * fabsf(rest);
        const int q = static_cast<int>(q0);
        const bool over = two > g.s || (two == g.s && (q & 1));
        return g.s == g.s ? static_cast<uint32_t>(over ? q + (rest > 0.f ? 1 : -1) : q) : 0u;
    }
    float t = __fmul_rn(v, g.r);
    if (g.rare) t = fmaf(fmaf(-t, g.s, v), g.r, t);
    return g.s == g.s ? __float_as_uint(__fadd_rn(t, kRint)) : 0u;
}
template <typename T>
__device__ __forceinline__ uint32_t code1(T x, const GroupScale& g) {
    return code1f<T>(static_cast<float>(x), g);
}

// Codes of 8 values of any group.
template <typename T>
__device__ __forceinline__ uint2 codes8_rare(const typename QuantOf<T>::Vec& x, const GroupScale& g) {
    float f[8];
    QuantOf<T>::unpack(x, f);
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = code1f<T>(f[i], g);
    return low_bytes(u);
}

// Codes of 8 FP32 values of a finite group: q0 of each, unless a value lies
// within 2^-14 of a border between two codes (in units of s), where q0 may be
// off by one.
__device__ __forceinline__ uint2 codes8_fast(const QuantOf<float>::Vec& x, const GroupScale& g) {
    float f[8];
    QuantOf<float>::unpack(x, f);
    const float2 r2 = make_float2(g.r, g.r), ns2 = make_float2(-g.s, -g.s), one2 = make_float2(1.f, 1.f);
    const float2 magic2 = make_float2(kRint, kRint), nmagic2 = make_float2(-kRint, -kRint);
    uint32_t u[8];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = make_float2(f[2 * i], f[2 * i + 1]);
        const float2 t = ffma2(v, r2, magic2);
        const float2 rest = ffma2(ffma2(t, one2, nmagic2), ns2, v);
        most = fmaxf(most, fmaxf(fabsf(rest.x), fabsf(rest.y)));
        u[2 * i] = __float_as_uint(t.x);
        u[2 * i + 1] = __float_as_uint(t.y);
    }
    if (most >= g.s * (0.5f - 6.10351562e-5f)) return codes8_rare<float>(x, g);
    return low_bytes(u);
}

// Codes of 8 values; `rare`: whether a lane of the warp has a rare group
// (warp-uniform).
template <typename T>
__device__ __forceinline__ uint2 codes8(const typename QuantOf<T>::Vec& x, const GroupScale& g, bool rare) {
    if (rare) return codes8_rare<T>(x, g);
    if constexpr (QuantOf<T>::kF32)
        return codes8_fast(x, g);
    else
        return codes8_fast(x, g.r);
}

// 8 byte codes -> 8 nibbles (the even one in the low half of each byte).
__device__ __forceinline__ uint32_t pack_nibbles(uint2 w) {
    const uint32_t a = w.x & 0x0f0f0f0fu, b = w.y & 0x0f0f0f0fu;
    return __byte_perm(a | (a >> 4), b | (b >> 4), 0x6420);
}

// Signed byte codes as floats, four at a time: the byte, biased to unsigned,
// becomes the low mantissa byte of 2^23 + (q + 128).
__device__ __forceinline__ void bytes_to_f(uint32_t w, float2 (&f)[2]) {
    const uint32_t b = w ^ 0x80808080u;
    const float2 one2 = make_float2(1.f, 1.f), bias2 = make_float2(-8388736.f, -8388736.f);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        f[i] = ffma2(make_float2(__uint_as_float(__byte_perm(b, 0x4b000000u, 0x7440 | (2 * i))),
                                 __uint_as_float(__byte_perm(b, 0x4b000000u, 0x7440 | (2 * i + 1)))),
                     one2, bias2);
}

// Eight nibble codes as floats, in order.
__device__ __forceinline__ void nibbles_to_f(uint32_t w, float2 (&f)[4]) {
    const uint32_t lo = (w & 0x0f0f0f0fu) ^ 0x08080808u, hi = ((w >> 4) & 0x0f0f0f0fu) ^ 0x08080808u;
    const float2 one2 = make_float2(1.f, 1.f), bias2 = make_float2(-8388616.f, -8388616.f);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        f[i] = ffma2(make_float2(__uint_as_float(__byte_perm(lo, 0x4b000000u, 0x7440 | i)),
                                 __uint_as_float(__byte_perm(hi, 0x4b000000u, 0x7440 | i))),
                     one2, bias2);
}

}  // namespace dnb
