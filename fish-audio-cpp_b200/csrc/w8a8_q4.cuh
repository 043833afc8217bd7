// What a 4-bit group is, shared by the KV cache and the weights, and the layout of a page of the 4-bit cache.
//
// A group is g consecutive fp16 values x. e is the one of largest magnitude (the positive one where +e and -e are both there),
// s = fp16(e / -8), code = rint(x / s) held to [-8, 7] (half to even; 0 where s is 0), the value it stands for is code * s. The sixteen
// codes are all used, and e itself is held exactly (e / -8 is exact but where it is subnormal). A group that holds an infinity or a NaN
// has the scale NaN and codes 0: it reads as NaN throughout, nothing that is not a number turns into one.
//
// x has 11 significant bits and (k + 1/2) s at most 15, so x / s is either a tie exactly or at least 2^-16 away from one, relatively: any
// quotient that is exact at ties and within 2^-20 elsewhere gives the same codes as 64 bits do.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

namespace w8a8 {
namespace q4 {

// ---- packed arithmetic ----
// Two fp32 numbers in one register pair: the packed arithmetic rounds each as the plain one does.
struct F2 {
    unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 parts(F2 x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x.v));
    return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 operator-(F2 a) { return {a.v ^ 0x8000000080000000ull}; }

// The extremes of a group travel as (max x, max -x): both are maxima that propagate NaN.
__device__ __forceinline__ __half2 extremes(__half a, __half b) {
    const __half2 v = __halves2half2(a, b), n = __hneg2(v);
    return __halves2half2(__hmax_nan(__low2half(v), __high2half(v)), __hmax_nan(__low2half(n), __high2half(n)));
}

struct Scale {
    __half s;      // as stored
    float f, inv;  // s, and 1 / s to within a few ulp; 0 where every code is 0
    __device__ __forceinline__ explicit Scale(__half2 mx) {
        const float hi = __low2float(mx), neg_lo = __high2float(mx);
        s = __float2half_rn((hi >= neg_lo ? hi : -neg_lo) * -0.125f);
        if (!(fmaxf(fabsf(hi), fabsf(neg_lo)) < INFINITY) || isnan(hi) || isnan(neg_lo)) s = __ushort_as_half(0x7fffu);
        f = __half2float(s);
        inv = (f == 0.0f || isnan(f)) ? 0.0f : __frcp_rn(f);
    }
    // One correction by the residual: exact where the quotient is a number of few bits, a tie above all (q * f has 24 bits at most there).
    __device__ __forceinline__ int code(__half x) const {
        if (inv == 0.0f) return 0;
        const float v = __half2float(x), q = v * inv;
        return max(-8, min(7, __float2int_rn(fmaf(fmaf(-q, f, v), inv, q))));
    }
    // Eight codes plus 8 as the nibbles of a word, low first: the same numbers, two at a time. A number below 2^22 that is added to 1.5 2^23 is rounded
    // to a whole one, half to even, in the low bits of the sum.
    __device__ __forceinline__ uint32_t codes_plus_8(const __half2 (&x)[4]) const {
        const F2 i2 = f2(inv, inv), minus_f = f2(-f, -f), magic = f2(12582912.0f, 12582912.0f);
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = __half22float2(x[i]);
            const F2 v = f2(a.x, a.y), q = v * i2;
            const float2 t = parts(fma2(fma2(q, minus_f, v), i2, q) + magic);
            constexpr int kLowest = 0x4b400000 - 8;  // the bits of 1.5 2^23 less 8
            word |= static_cast<uint32_t>(__vimin_s32_relu(__float_as_int(t.x) - kLowest, 15)) << (8 * i);
            word |= static_cast<uint32_t>(__vimin_s32_relu(__float_as_int(t.y) - kLowest, 15)) << (8 * i + 4);
        }
        return inv == 0.0f ? 0x88888888u : word;
    }
};

// ---- a page of the cache: 16 tokens of one (layer, kv head), 128 channels ----
//   [0, 1024)       K codes: token t at 64 t; in it 16 bytes for each quarter j of eight channels of every 32-channel run: the word
//                   16 j + 4 run holds channels 32 run + 8 j + n as nibbles n = 0 .. 7 (low first)
//   [1024, 2048)    V codes: pair of tokens p at 128 p; unit r = 0 .. 7 of 16 bytes; the word 8 half + 4 high of it holds channels
//                   64 high + 16 n + 8 half + r, n = 0 .. 3, of token 2 p as nibbles 0 .. 3 and of token 2 p + 1 as nibbles 4 .. 7
//   [2048, + 32 G)  K scales fp16, G = 128 / group: [pair of tokens][group][token of the pair]
//   [.., + 32 G)    V scales, the same
// Codes are stored plus 8. The orders are those in which a lane's 16-byte read holds what it feeds to the matrix instructions, with no
// exchange between lanes: eight channels of one token for q K^T, four channels by two tokens for P V (the contraction runs over tokens).
constexpr int kTokens = 16, kDim = 128;
constexpr int kVOff = kTokens * kDim / 2, kScaleOff = 2 * kVOff;
__host__ __device__ constexpr int page_bytes(int groups) { return kScaleOff + 4 * kTokens * groups; }
__host__ __device__ __forceinline__ constexpr int scale_off(int groups, int is_v, int token, int group) {
    return kScaleOff + is_v * 2 * kTokens * groups + (((token >> 1) * groups + group) * 2 + (token & 1)) * 2;
}

}  // namespace q4
}  // namespace w8a8
