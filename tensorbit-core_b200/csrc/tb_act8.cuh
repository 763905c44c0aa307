// 8-bit activation checkpoints: the decode used by every kernel that reads one.
// A value is q * 2^(E - 127) with an int8 code q and the exponent byte E of its
// feature and block of TB_ACT8_BLOCK tokens; E = 255 with codes 0 marks a block
// that held a NaN or an infinity and reads back as NaN.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tb_kernels.h"

namespace tb {
namespace act8 {

constexpr int kBlock = TB_ACT8_BLOCK;

// Features at most, in and out: the kernels round their indexes up to tiles of 256 in 32 bits.
constexpr int kMaxFeatures = 0x7FFFFFFF - 255;

// What the kernels need of a tb_act8.
struct View {
    int8_t* codes;
    uint8_t* exps;
    long long ldq, lde;
    long long n;
    int d;
};

// Status of a checkpoint description; fills `v`.
int check(const tb_act8* ck, const char* who, View* v);
// Enqueues the reading back of n > 0 tokens.
int unpack(const View& ck, void* out, int dtype, long long ldo, cudaStream_t st);

// 2^(E - 127) in FP32.  E = 255 gives an infinity, and the zero codes of such a block times it NaN.
__device__ __forceinline__ float scale_f32(uint32_t e) { return __uint_as_float(e << 23); }

// Exponent byte for a block whose largest |x| has the FP32 bits `amax`
// (NaN and infinity order above every finite value): the smallest power of two
// with rint(amax / 2^e) <= 127.  For amax = m 2^k, 1 <= m < 2, that is k - 6
// unless 64 m >= 127.5, which is when the seven top mantissa bits are all ones
// and adding 0x10000 carries into the exponent.
__device__ __forceinline__ uint32_t exponent_of(uint32_t amax) {
    if (amax >= 0x7F800000u) return 255u;
    const int e = static_cast<int>((amax + 0x10000u) >> 23) - 6;
    return static_cast<uint32_t>(e < 1 ? 1 : e);
}
// 2^(127 - E), the factor from values to codes (E of exponent_of, not 255).
__device__ __forceinline__ float inverse_scale(uint32_t e) { return __uint_as_float((254u - e) << 23); }

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
// Two int8 codes in the low bytes of v's halves (the high bytes 0x43) times two
// BF16 scales.  0x4300 | low7 is 128 + low7 and 0x4300 | sign is 128 or 256, so
// their difference is the signed code; both steps are exact.
__device__ __forceinline__ uint32_t decode2(uint32_t v, uint32_t scale2) {
    const uint32_t hi = v & 0xFF7FFF7Fu, lo = v & 0xFF80FF80u;
    const __nv_bfloat162 q = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&hi), *reinterpret_cast<const __nv_bfloat162*>(&lo));
    const __nv_bfloat162 x = __hmul2(q, *reinterpret_cast<const __nv_bfloat162*>(&scale2));
    return *reinterpret_cast<const uint32_t*>(&x);
}

// Eight exponent bytes as four pairs of BF16 scales (255 is an infinity, and 0 times it NaN).
__device__ __forceinline__ void scales8(uint2 e, uint32_t (&s)[4]) {
    s[0] = prmt(e.x, 0, 0x4140u) << 7;
    s[1] = prmt(e.x, 0, 0x4342u) << 7;
    s[2] = prmt(e.y, 0, 0x4140u) << 7;
    s[3] = prmt(e.y, 0, 0x4342u) << 7;
}
// Eight codes times eight scales.
__device__ __forceinline__ uint4 decode8(uint2 w, const uint32_t (&s)[4]) {
    return make_uint4(decode2(prmt(w.x, 0x43434343u, 0x4140u), s[0]), decode2(prmt(w.x, 0x43434343u, 0x4342u), s[1]),
                      decode2(prmt(w.y, 0x43434343u, 0x4140u), s[2]), decode2(prmt(w.y, 0x43434343u, 0x4342u), s[3]));
}

// Element types as IEEE values.
template <int DT>
struct Elem;
template <>
struct Elem<TB_F32> {
    using T = float;
    static __device__ __forceinline__ float load(const void* p, long long i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ T to(float x) { return x; }
};
template <>
struct Elem<TB_F16> {
    using T = __half;
    static __device__ __forceinline__ float load(const void* p, long long i) { return __half2float(static_cast<const __half*>(p)[i]); }
    static __device__ __forceinline__ T to(float x) { return __float2half_rn(x); }
};
template <>
struct Elem<TB_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float load(const void* p, long long i) { return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]); }
    static __device__ __forceinline__ T to(float x) { return __float2bfloat16_rn(x); }
};

}  // namespace act8
}  // namespace tb
