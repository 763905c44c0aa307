// A plain tiled product on the FP32 pipes: C[m][n] = sum_k op.a(m, k) op.b(k, n),
// 64 x 64 outputs per block of 256 threads, 16 k at a time through shared
// memory.  `op` names the operands, the range of k and what becomes of a sum.
#pragma once

#include <cuda_runtime.h>

namespace tb {

template <class Op>
__global__ void __launch_bounds__(256) simple_gemm_kernel(const Op op) {
    __shared__ float As[16][65], Bs[16][65];
    const long long m0 = static_cast<long long>(blockIdx.y) * 64, n0 = static_cast<long long>(blockIdx.x) * 64;
    if (!op.wanted(m0, n0)) return;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (int u = op.first_unit(blockIdx.z); u < op.last_unit(blockIdx.z); ++u) {
        float acc[4][4] = {};
        const long long k1 = op.k_end(u);
        for (long long k0 = op.k_begin(u); k0 < k1; k0 += 16) {
            __syncthreads();
            for (int i = threadIdx.x; i < 16 * 64; i += 256) {
                const int ma = op.kRowA ? i >> 4 : i & 63, ka = op.kRowA ? i & 15 : i >> 6;
                As[ka][ma] = (m0 + ma < op.M && k0 + ka < k1) ? op.a(m0 + ma, k0 + ka) : 0.0f;
                const int nb = op.kRowB ? i & 63 : i >> 4, kb = op.kRowB ? i >> 6 : i & 15;
                Bs[kb][nb] = (n0 + nb < op.N && k0 + kb < k1) ? op.b(k0 + kb, n0 + nb) : 0.0f;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 16; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[k][ty * 4 + i], Bs[k][tx * 4 + j], acc[i][j]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const long long m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
                if (m < op.M && n < op.N) op.store(u, m, n, acc[i][j]);
            }
    }
}

}  // namespace tb
