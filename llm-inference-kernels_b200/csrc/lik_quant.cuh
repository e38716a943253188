// Row quantization shared by the KV quantizers (quantize.cu) and the rotating
// append (rope.cu): one token row per 8-lane group, codes and scales
// bit-exact with the oracle. Include only in files built with -fmad=false.
#pragma once

#include <cuda_fp16.h>

#include "lik_device.cuh"
#include "lik_internal.h"

namespace lik {

namespace {

constexpr float kAsymScaleFloor = 5.9604644775390625e-8f;  // 2^-24, smallest fp16 subnormal

// Codes are rint(x / s) with x / s the IEEE fp32 quotient (round to
// nearest), as the oracle computes them, without a division in the common
// case. With r = RN(1/s), y = RN(x * r) lies within 2^-22.4 |x / s| of that
// quotient, i.e. within 2.3e-5 for the |x / s| <= 128 these kernels produce;
// so y rounds to the quotient's nearest integer unless it lies within 4e-5 of
// a half-integer, and only those elements (and non-finite ones) take the
// exact division. Rounding adds 1.5 * 2^23 (fp32 addition rounds half to
// even, like rintf): for |v| < 2^22 the sum holds the integer in its low
// mantissa bits, from which the codes are packed without a float-to-int
// conversion.
constexpr float kRoundMagic = 12582912.0f;  // 1.5 * 2^23
constexpr float kNearTie = 0.49996f;        // |y - rint(y)| at or above this: exact division

// bytes 0..3 = low bytes of a, b, c, d
__device__ __forceinline__ uint32_t pack_bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// One 8-lane group per kRowsPerGroup consecutive token rows, 16 channels
// per lane; the rows' loads are issued together.
// MODE kTokI8: int8 codes; kTokI4Sym: packed signed nibbles; kTokI4Asym:
// packed unsigned nibbles with a zero point.
//
// Per element the common path is y = x * RN(1/s) rounded through the magic
// constant; one check per lane sends a lane whose elements include a
// near-tie (or a non-finite value) through the exact division. The symmetric
// formats need no clamp on the common path: |x| <= absmax and s >= absmax /
// qmax rounded to nearest, so |x / s| <= qmax (1 + 2^-24) rounds to at most
// qmax in magnitude.
constexpr int kRowsPerGroup = 2;
constexpr int kLanesPerRow = 8;

// 16 halves of a row held as raw packed pairs (8 registers)
struct Raw16 {
    uint4 a, b;
};
__device__ __forceinline__ Raw16 load_raw16(const __half* src) {
    Raw16 r;
    r.a = *reinterpret_cast<const uint4*>(src);
    r.b = *reinterpret_cast<const uint4*>(src + 8);
    return r;
}
__device__ __forceinline__ __half2 raw_pair(const Raw16& r, int i) {  // elements 2i, 2i+1
    const uint4& u = i < 4 ? r.a : r.b;
    const uint32_t w = (i & 3) == 0 ? u.x : (i & 3) == 1 ? u.y : (i & 3) == 2 ? u.z : u.w;
    return *reinterpret_cast<const __half2*>(&w);
}

// Quantize one token row held by an 8-lane group (16 channels per lane) into
// destination row drow: statistics, scale (and zero), codes, packed stores.
template <int MODE>
__device__ __forceinline__ void quant_row(const Raw16& raw, long long drow, uint8_t* __restrict__ codes,
                                          __half* __restrict__ scale, __half* __restrict__ zero, int l,
                                          unsigned mask) {
    constexpr int NL = kLanesPerRow;
    constexpr int CH = kHeadDim / NL;
    // row statistics on packed fp16 (min / max / |x| are exact in fp16)
    float sc, zf = 0.f, sf;
    if (MODE == kTokI4Asym) {
        __half2 mn2 = raw_pair(raw, 0), mx2 = mn2;
#pragma unroll
        for (int i = 1; i < CH / 2; ++i) {
            mn2 = __hmin2(mn2, raw_pair(raw, i));
            mx2 = __hmax2(mx2, raw_pair(raw, i));
        }
        float mn = fminf(__low2float(mn2), __high2float(mn2));
        float mx = fmaxf(__low2float(mx2), __high2float(mx2));
#pragma unroll
        for (int m = 1; m < NL; m <<= 1) {
            mn = fminf(mn, __shfl_xor_sync(mask, mn, m));
            mx = fmaxf(mx, __shfl_xor_sync(mask, mx, m));
        }
        sc = fmaxf(__fdiv_rn(__fsub_rn(mx, mn), 15.0f), kAsymScaleFloor);
        const __half sh = __float2half_rn(sc);
        const __half zh = __float2half_rn(mn);
        sf = __half2float(sh);
        zf = __half2float(zh);
        if (l == 0) {
            scale[drow] = sh;
            zero[drow] = zh;
        }
    } else {
        constexpr float qmax = (MODE == kTokI8) ? 127.0f : 7.0f;
        __half2 am2 = __habs2(raw_pair(raw, 0));
#pragma unroll
        for (int i = 1; i < CH / 2; ++i) am2 = __hmax2(am2, __habs2(raw_pair(raw, i)));
        float amax = fmaxf(__low2float(am2), __high2float(am2));
#pragma unroll
        for (int m = 1; m < NL; m <<= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, m));
        sc = fmaxf(__fdiv_rn(amax, qmax), 1e-8f);
        sf = sc;
        if (l == 0) scale[drow] = __float2half_rn(sc);
    }
    const float rf = __frcp_rn(sf);
    // common path: tv_i = rint(x_i / s) + 1.5 * 2^23, the code in its low bits
    float xv[CH];
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
        const float2 u = __half22float2(raw_pair(raw, i));
        xv[2 * i] = MODE == kTokI4Asym ? __fsub_rn(u.x, zf) : u.x;
        xv[2 * i + 1] = MODE == kTokI4Asym ? __fsub_rn(u.y, zf) : u.y;
    }
    float tv[CH];
    bool exact = false;  // some element is a near-tie, or not finite
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const float y = __fmul_rn(xv[i], rf);
        float tt = __fadd_rn(y, kRoundMagic);
        exact |= !(fabsf(__fsub_rn(y, __fsub_rn(tt, kRoundMagic))) < kNearTie);
        if (MODE == kTokI4Asym) tt = fminf(fmaxf(tt, kRoundMagic), kRoundMagic + 15.0f);
        tv[i] = tt;
    }
    if (exact) {  // exact quotients for the lane's elements
        constexpr float lo = MODE == kTokI4Asym ? 0.0f : (MODE == kTokI8 ? -127.0f : -7.0f);
        constexpr float hi = MODE == kTokI4Asym ? 15.0f : (MODE == kTokI8 ? 127.0f : 7.0f);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const float qv = fminf(fmaxf(rintf(__fdiv_rn(xv[i], sf)), lo), hi);
            tv[i] = __fadd_rn(qv, kRoundMagic);
        }
    }
    uint32_t c[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) c[i] = static_cast<uint32_t>(__float_as_int(tv[i]));
    if (MODE == kTokI8) {
        reinterpret_cast<uint4*>(codes + drow * kHeadDim)[l] =
            make_uint4(pack_bytes4(c[0], c[1], c[2], c[3]), pack_bytes4(c[4], c[5], c[6], c[7]),
                       pack_bytes4(c[8], c[9], c[10], c[11]), pack_bytes4(c[12], c[13], c[14], c[15]));
    } else {
        uint32_t w0 = 0, w1 = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w0 |= (c[i] & 0xFu) << (4 * i);
            w1 |= (c[8 + i] & 0xFu) << (4 * i);
        }
        reinterpret_cast<uint2*>(codes + drow * (kHeadDim / 2))[l] = make_uint2(w0, w1);
    }
}

}  // namespace

}  // namespace lik
