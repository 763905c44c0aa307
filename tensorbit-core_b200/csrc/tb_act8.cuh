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
