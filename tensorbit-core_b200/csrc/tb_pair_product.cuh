// One persistent kernel for products of 16-bit operands, instantiated per
// operation.  A pair of CTAs (cta_group::2) owns a 256 x 256 tile of the product:
// each CTA holds its 128 rows of A and 128 of the 256 columns of B of a K slice of
// 64 in shared memory, and its 128 x 256 half of the accumulator in TMEM, which has
// room for two.  Warp 8 loads slices by TMA, warp 9 of the even CTA issues
// tcgen05.mma for both, warps 0-7 take accumulators out of TMEM and hand each
// lane's row of 128 columns to the operation.
//
// The tensor core's additions cut off; an operation says after how many slices
// (kGroup) a sum leaves TMEM and is added in FP32 registers with rounding.
// kParts = 2: operands are pairs hi + lo of FP16 matrices, whose products
// hi hi + hi lo + lo hi keep 22 bits.
//
// An operation OP has kAMn, kBMn (operands whose rows in memory run along M or N;
// otherwise along K), kParts, kF16, kGroup, Params, and the device functions
//   items(P)       units of work, which may depend on counts in device memory
//   work(P, item)  the unit's tile and K range
//   finish(L, w, acc, buf, row, half, lane)
//   error()        where an expired wait is recorded
// `acc` is columns 128 half .. of the tile's row `row` + lane; `buf` is 4 KB of
// shared memory of the warp's own.  Every wait is bounded; on expiry the kernel
// records an error, there and in the word p.failed of its call, and leaves: only
// finished sums reach finish(), and what writes a call's results looks at that word.
#pragma once

#include <algorithm>
#include <mutex>

#include "tb_pair.cuh"
#include "tb_pdl.cuh"

namespace tb {
namespace pair {

struct Work {
    int tm, tn;       // 256 x 256 tile
    int k0, slices;   // K slices of 64
    int which;        // of up to two products in one launch
    int slot;         // share of a unit whose K is shared out, or -1
};

template <class OP>
struct Launch {
    CUtensorMap a[2], b[2][2], o[2][2];  // [part], [product][part]
    typename OP::Params p;
};

template <class OP>
struct ProductCfg {
    static constexpr int kTile = 16384;  // 128 rows (or columns) of a K slice
    static constexpr int kStage = 2 * OP::kParts * kTile;
    static constexpr int kStages = 196608 / kStage;
    static constexpr int kBuf = 8 * kPieceBytes;
    static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStage + kBuf + 1024 + 256;
    static_assert(kSmem <= 232448, "shared memory of a block");
};
// Twelve warps (10 and 11 idle, so that the roles are whole warpgroups) of 168 registers a
// thread, of which the warps with results take 8 x 208 and leave the others 4 x 88.
constexpr int kProductThreads = 384, kProductRegs = 168;
constexpr int kLoadWarp = 8, kIssueWarp = 9;

template <bool F16>
__device__ __forceinline__ void mma_pair16(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}"
        ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u));
}

// Tiles in bands of 8 rows, column by column inside, so that concurrent tiles share operands in L2.
__device__ __forceinline__ void band_tile(int i, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int band = i / (8 * tiles_n), in = i % (8 * tiles_n);
    const int rows = min(8, tiles_m - 8 * band);
    tm = 8 * band + in % rows;
    tn = in / rows;
}
// Share q of `splits` of `all` slices.
__device__ __forceinline__ int share_at(int all, int q, int splits) {
    return static_cast<int>(static_cast<long long>(all) * q / splits);
}

template <class OP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kProductThreads, 1)
product_kernel(const __grid_constant__ Launch<OP> L) {
    using C = ProductCfg<OP>;
    constexpr int kStages = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    // (by offset, so that the compiler still knows it for shared memory)
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* out_buf = smem + kStages * C::kStage;
    uint64_t* ready = reinterpret_cast<uint64_t*>(out_buf + C::kBuf);  // (even CTA) slice loaded by both CTAs
    uint64_t* empty = ready + kStages;                                // slice read by the MMAs
    uint64_t* accfull = empty + kStages;                              // [2] sum finished
    uint64_t* accempty = accfull + 2;                                 // [2] (even CTA) sum taken by both CTAs
    uint64_t* drained = accempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank());

    if (threadIdx.x == kLoadWarp * 32) {
#pragma unroll
        for (int q = 0; q < OP::kParts; ++q) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&L.a[q])) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&L.b[0][q])) : "memory");
        }
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&ready[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&accfull[b]), 1);
            mbar_init(smem_u32(&accempty[b]), 16);
        }
        mbar_init(smem_u32(drained), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    fence_before();
    cluster_sync_all();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();  // nothing above touched memory that an earlier kernel writes
    const int items = OP::items(L.p);
    auto gave_up = [&] {
        abort_pair(abort_flag);
        atomicExch(OP::error(), 1);
        atomicExch(L.p.failed, 1);
    };

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int quad = warp & 3, half = warp >> 2;
        uint8_t* buf = out_buf + warp * kPieceBytes;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(half * 128);
        Ring<2> ac;
        bool ok = true;
        for (int item = blockIdx.x >> 1; item < items && ok; item += gridDim.x >> 1) {
            const Work w = OP::work(L.p, item);
            float acc[128];
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
            for (int left = w.slices; left > 0; left -= OP::kGroup) {
                if (!wait(smem_u32(&accfull[ac.s]), ac.phase, abort_flag)) { ok = false; break; }
                read_accumulator<128>(lane_base + static_cast<uint32_t>(ac.s * 256), smem_u32(&accempty[ac.s]), lane, [&](int c, uint32_t (&x)[16]) {
#pragma unroll
                    for (int i = 0; i < 16; i += 2) add2(acc[c * 16 + i], acc[c * 16 + i + 1], x[i], x[i + 1]);
                });
                ac.next();
            }
            if (ok) OP::finish(L, w, acc, buf, rank * 128 + quad * 32, half, lane);
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if (!ok) gave_up();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == kLoadWarp && lane == 0) {
            Ring<kStages> at;
            const uint32_t ready0 = smem_u32(ready) & kPeerMask, empty0 = smem_u32(empty), stage0 = smem_u32(smem);
            bool ok = true;
            for (int item = blockIdx.x >> 1; item < items && ok; item += gridDim.x >> 1) {
                const Work w = OP::work(L.p, item);
                const int m0 = w.tm * 256 + rank * 128, n0 = w.tn * 256 + rank * 128;
                int k = w.k0 * 64;
#pragma unroll 1
                for (int left = w.slices; left > 0; --left, k += 64, at.next()) {
                    if (!wait(empty0 + 8 * at.s, at.phase ^ 1, abort_flag)) { ok = false; break; }  // (the first round passes at once)
                    const uint32_t bar = ready0 + 8 * at.s;
                    if (rank == 0) mbar_expect_tx(bar, 2 * C::kStage);
#pragma unroll
                    for (int q = 0; q < OP::kParts; ++q) {
                        const uint32_t a = stage0 + at.s * C::kStage + 2 * q * C::kTile, b = a + C::kTile;
                        if constexpr (OP::kAMn) {
                            tma_load_pair(a, &L.a[q], m0, k, bar);
                            tma_load_pair(a + kMnChunk, &L.a[q], m0 + 64, k, bar);
                        } else {
                            tma_load_pair(a, &L.a[q], k, m0, bar);
                        }
                        if constexpr (OP::kBMn) {
                            tma_load_pair(b, &L.b[w.which][q], n0, k, bar);
                            tma_load_pair(b + kMnChunk, &L.b[w.which][q], n0 + 64, k, bar);
                        } else {
                            tma_load_pair(b, &L.b[w.which][q], k, n0, bar);
                        }
                    }
                }
            }
            if (!ok) {
                gave_up();
                // Loads in flight, each stage's last phase waited for within a limit (the odd CTA's count on the
                // even one's barrier).  A stage never used answers at once.
                for (int i = 0; i < kStages && rank == 0; ++i)
                    if (i < at.s || at.phase) wait(smem_u32(&ready[i]), i < at.s ? at.phase : at.phase ^ 1, nullptr);
            }
        }
        if (warp == kIssueWarp && lane == 0 && rank == 0) {
            constexpr uint32_t kFormat = OP::kF16 ? 0u : 1u;
            constexpr uint32_t kIdesc = (1u << 4) | (kFormat << 7) | (kFormat << 10) | (OP::kAMn ? 1u << 15 : 0u) |
                                        (OP::kBMn ? 1u << 16 : 0u) | ((256u >> 3) << 17) | (16u << 24);
            // descriptor steps of one MMA: K-major 32 bytes along a row; MN-major 16 rows
            constexpr uint64_t kStepA = OP::kAMn ? 16 * 128 >> 4 : 2, kStepB = OP::kBMn ? 16 * 128 >> 4 : 2;
            constexpr uint64_t kLo = 2 * C::kTile >> 4;  // from the hi part to the lo part
            Ring<kStages> at;
            Ring<2> ac;
            const uint64_t a_desc = operand_desc(smem_u32(smem), OP::kAMn), b_desc = operand_desc(smem_u32(smem) + C::kTile, OP::kBMn);
            const uint32_t ready0 = smem_u32(ready), empty0 = smem_u32(empty);
            bool ok = true;
            for (int item = blockIdx.x >> 1; item < items && ok; item += gridDim.x >> 1) {
                const Work w = OP::work(L.p, item);
                for (int left = w.slices; left > 0 && ok;) {
                    const uint32_t d = tmem + static_cast<uint32_t>(ac.s * 256);
                    int n = min(left, OP::kGroup);
                    left -= n;
                    if (!wait(smem_u32(&accempty[ac.s]), ac.phase ^ 1, abort_flag)) { ok = false; break; }
                    uint32_t more = 0;
#pragma unroll 1
                    for (; n > 0; --n, at.next()) {
                        const uint64_t a0 = a_desc + at.s * (C::kStage >> 4), b0 = b_desc + at.s * (C::kStage >> 4);
                        if (!wait(ready0 + 8 * at.s, at.phase, abort_flag)) { ok = false; break; }
                        fence_after();
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            const uint64_t a = a0 + kk * kStepA, b = b0 + kk * kStepB;
                            if constexpr (OP::kParts == 2) {  // the small products first
                                mma_pair16<OP::kF16>(d, a + kLo, b, kIdesc, more);
                                mma_pair16<OP::kF16>(d, a, b + kLo, kIdesc, 1);
                                mma_pair16<OP::kF16>(d, a, b, kIdesc, 1);
                            } else {
                                mma_pair16<OP::kF16>(d, a, b, kIdesc, more);
                            }
                            more = 1;
                        }
                        commit_pair(empty0 + 8 * at.s);
                    }
                    if (!ok) break;
                    commit_pair(smem_u32(&accfull[ac.s]));
                    ac.next();
                }
            }
            if (!ok) gave_up();
            if (*abort_flag) drain_pair(smem_u32(drained));
        }
        __syncwarp();
    }
    fence_before();
    cluster_sync_all();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Launches for at most `items` units of work.
template <class OP>
int launch_product(const Launch<OP>& L, long long items, cudaStream_t st) {
    using C = ProductCfg<OP>;
    static std::mutex mu;
    // Per device: the shared-memory limit, and that the launch has the registers that the roles' shares add up to.
    static uint64_t prepared = 0;
    int dev = 0;
    int rc = require_device(&dev);
    if (rc) return rc;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 64 || !(prepared >> dev & 1)) {
            cudaFuncAttributes fa{};
            cudaError_t e = cudaFuncGetAttributes(&fa, product_kernel<OP>);
            if (e == cudaSuccess && fa.numRegs != kProductRegs)
                return fail(TB_ERR_CUDA, "product_kernel has %d registers a thread, not %d", fa.numRegs, kProductRegs);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(product_kernel<OP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::kSmem));
            if (e != cudaSuccess) return cuda_fail(e, "product_kernel setup");
            if (dev < 64) prepared |= 1ull << dev;
        }
    }
    if (items <= 0) return TB_OK;
    const unsigned pairs = static_cast<unsigned>(std::min<long long>(items, kPairs));
    const cudaError_t e = launch_pdl(product_kernel<OP>, dim3(2 * pairs), dim3(kProductThreads), C::kSmem, st, L);
    return e == cudaSuccess ? check_launch("product_kernel") : cuda_fail(e, "product_kernel launch");
}

// An operand of 16-bit values: [rows][cols] in rows of ld, 128-byte swizzle; rows along K
// are boxes of 128 rows (of M or N), rows along M or N boxes of 64 (of K).
inline int operand_map(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld, bool mn) {
    return make_map(map, base, 2, cols, rows, ld, 64, mn ? 64 : 128, true);
}

}  // namespace pair
}  // namespace tb
