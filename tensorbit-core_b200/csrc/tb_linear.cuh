// Tensor-core products of the calibration operators (tb_linear.cu): weight
// gradients, Fisher EMA and Hessian from an 8-bit checkpoint, and the two
// products of a projection with low-rank adapters.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "tb_act8.cuh"

namespace tb {
namespace linear {

// dy as `parts` stacked BF16 matrices [parts * n][ld] that add up to it.
struct Parts {
    const void* base;
    long long ld;
    int parts;
};

int weight_grad(const act8::View& ck, const Parts& dy, int r, const int64_t* samples, int S, void* grads, int g_dtype,
                long long g_stride, cudaStream_t st);
int fisher(const act8::View& ck, const Parts& dy, int r, const int64_t* samples, int S, double alpha, double beta, bool first,
           float* F, cudaStream_t st);
int hessian(const act8::View& ck, float scale, bool accumulate, float* H, cudaStream_t st);

// Two FP32 values as pairs of BF16 parts that add up to them, to 2^-17 of each: hi
// rounded, or cut off where rounding leaves the range; an infinity has no rest.
__device__ __forceinline__ void split_pair(float f0, float f1, uint32_t& hi, uint32_t& lo) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f0, f1);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    float r0 = f0 - __uint_as_float(hi << 16), r1 = f1 - __uint_as_float(hi & 0xFFFF0000u);
    if (fmaxf(fabsf(f0), fabsf(f1)) >= 3.39e38f) {  // (BF16 rounds to an infinity from 3.396e38)
        constexpr uint32_t kInf = 0x7F80u;
        if ((hi & 0x7FFFu) == kInf) hi = (hi & 0xFFFF0000u) | __float_as_uint(f0) >> 16;
        if ((hi >> 16 & 0x7FFFu) == kInf) hi = (hi & 0xFFFFu) | (__float_as_uint(f1) & 0xFFFF0000u);
        r0 = (hi & 0x7FFFu) == kInf ? 0.0f : f0 - __uint_as_float(hi << 16);
        r1 = (hi >> 16 & 0x7FFFu) == kInf ? 0.0f : f1 - __uint_as_float(hi & 0xFFFF0000u);
    }
    const __nv_bfloat162 l = __floats2bfloat162_rn(r0, r1);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

constexpr int kListTokens = 256;              // tokens of one list of adapters
constexpr int kListPitch = kListTokens + 1;   // its count, then its adapters

// out[t][o] = sum_k in[t][k] W(o, k) + sum_j u[t][j] E_a(t)(o, j): forward with W
// row-major [N][K] and E = b, input gradient with W row-major [K][N] and E = a.
struct AdapterProduct {
    long long n;                 // tokens
    int N, K;                    // out and in features of this product
    const __nv_bfloat16* in;
    long long ldin;
    const __nv_bfloat16* w;
    long long ldw;
    __nv_bfloat16* out;
    long long ldout;
    const int32_t* who;          // adapter of each token
    const int32_t* lists;        // [ceil(n / 256)][kListPitch], NULL without adapters
    const float* u;              // [n][rank]
    const __nv_bfloat16* e;      // b (forward: [na * N][lde]) or a (backward: [na * rank][lde])
    long long lde;
    int rank, na;
};
int adapter_forward(const AdapterProduct& p, cudaStream_t st);
int adapter_input_grad(const AdapterProduct& p, cudaStream_t st);

// Error code recorded by these kernels on this device since the previous call
// (0 none, 1 a bounded wait expired, -1 it could not be read); resets it.
int take_error(cudaStream_t st);

}  // namespace linear
}  // namespace tb
