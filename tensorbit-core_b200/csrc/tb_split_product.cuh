// A product kernel for matrices whose 256 x 256 tiles would leave SMs idle: a cluster
// of 1 to 8 CTAs owns a 128 x 128 tile and shares its K out.  Each CTA sums its
// slices as the pair kernel does (two accumulators in TMEM, groups added in FP32
// registers); the sums then lie in shared memory, and each CTA adds up its share of
// the rows of all of them, in the cluster's order, through distributed shared memory
// and hands those rows to the operation.  One launch, and no sums in global memory.
// Its tiles need twice the operands of the pair kernel's for each product: with all
// SMs at it, L2 bounds it (k = 1024, 16 slices of two parts: 1.2 us a slice, where
// the tensor core takes 0.42).
//
// Operations as for the pair kernel, with tiles of 128 from
//   split_work(P, tile)
//   fetch_quad(L, row, col)        what four columns need from memory, fetched while their sums arrive
//   finish_quad(L, w, row, col, v, fetched, words)   four columns; `words` go on to, where kMirror,
//   mirror(L, w, words, pitch, row, rows, thread)   the rows' words in shared memory
#pragma once

#include "tb_pair_product.cuh"

namespace tb {
namespace pair {

constexpr int kSplitThreads = 384;  // warps 0-3 sums, 4 loads, 5 MMAs, all of them results
constexpr int kSplitPitch = 132;    // floats of a row of sums: 16-byte accesses without bank conflicts
constexpr int kSplitMost = 8;       // CTAs of a cluster

template <class OP>
struct SplitCfg {
    static constexpr int kTile = 16384;
    static constexpr int kStage = 2 * OP::kParts * kTile;
    static constexpr int kStages = 196608 / kStage;
    static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStage + 1024 + 256;
    static_assert(2 * 128 * kSplitPitch * 4 <= kStages * kStage, "sums lie where the stages were");
};

template <bool F16>
__device__ __forceinline__ void mma_one16(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
        ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u));
}
__device__ __forceinline__ float4 load_cluster4(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile(
        "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\t"
        "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
        : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
        : "r"(addr), "r"(rank)
        : "memory");
    return v;
}
__device__ __forceinline__ int load_cluster_int(uint32_t addr, uint32_t rank) {
    int v;
    asm volatile(
        "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\t"
        "ld.shared::cluster.u32 %0, [a];\n\t}"
        : "=r"(v)
        : "r"(addr), "r"(rank)
        : "memory");
    return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <class OP>
__global__ void __launch_bounds__(kSplitThreads, 1) split_product_kernel(const __grid_constant__ Launch<OP> L, const int ctas) {
    using C = SplitCfg<OP>;
    constexpr int kStages = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* ready = reinterpret_cast<uint64_t*>(smem + kStages * C::kStage);
    uint64_t* empty = ready + kStages;
    uint64_t* accfull = empty + kStages;  // [2]
    uint64_t* accempty = accfull + 2;     // [2]
    uint64_t* drained = accempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank());

    if (threadIdx.x == 4 * 32) {
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
            mbar_init(smem_u32(&accempty[b]), 4);
        }
        mbar_init(smem_u32(drained), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(256));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    Work w = OP::split_work(L.p, static_cast<int>(blockIdx.x) / ctas);
    const int all = w.slices, first = share_at(all, rank, ctas);
    w.k0 = first;
    w.slices = share_at(all, rank + 1, ctas) - first;
    pdl_wait();  // nothing above touched memory that an earlier kernel writes

    auto gave_up = [&] {
        *abort_flag = 1;
        atomicExch(OP::error(), 1);
        atomicExch(L.p.failed, 1);
    };

    float* sums = reinterpret_cast<float*>(smem);
    if (warp < 4) {
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        Ring<2> ac;
        bool ok = true;
        float acc[128];
#pragma unroll
        for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
        for (int left = w.slices; left > 0; left -= OP::kGroup) {
            if (!wait(smem_u32(&accfull[ac.s]), ac.phase, abort_flag)) { ok = false; break; }
            fence_after();
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                uint32_t x[16];
                tmem_ld16(lane_base + static_cast<uint32_t>(ac.s * 128 + 16 * c), x);
                tmem_wait16(x);
#pragma unroll
                for (int i = 0; i < 16; i += 2) add2(acc[c * 16 + i], acc[c * 16 + i + 1], x[i], x[i + 1]);
            }
            fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&accempty[ac.s])) : "memory");
            ac.next();
        }
        // (every MMA of this CTA is done, and so is every load that one of them read)
        if (ok) {
            float* row = sums + (warp * 32 + lane) * kSplitPitch;
#pragma unroll
            for (int i = 0; i < 128; i += 4) *reinterpret_cast<float4*>(row + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
        } else {
            gave_up();
        }
    } else if (warp == 4) {
        if (lane == 0) {
            Ring<kStages> at;
            const uint32_t ready0 = smem_u32(ready), empty0 = smem_u32(empty), stage0 = smem_u32(smem);
            const int m0 = w.tm * 128, n0 = w.tn * 128;
            int k = w.k0 * 64;
            bool ok = true;
#pragma unroll 1
            for (int left = w.slices; left > 0; --left, k += 64, at.next()) {
                if (!wait(empty0 + 8 * at.s, at.phase ^ 1, abort_flag)) { ok = false; break; }  // (the first round passes at once)
                const uint32_t bar = ready0 + 8 * at.s;
                mbar_expect_tx(bar, C::kStage);
#pragma unroll
                for (int q = 0; q < OP::kParts; ++q) {
                    const uint32_t a = stage0 + at.s * C::kStage + 2 * q * C::kTile, b = a + C::kTile;
                    if constexpr (OP::kAMn) {
                        tma_load_2d(a, &L.a[q], m0, k, bar);
                        tma_load_2d(a + kMnChunk, &L.a[q], m0 + 64, k, bar);
                    } else {
                        tma_load_2d(a, &L.a[q], k, m0, bar);
                    }
                    if constexpr (OP::kBMn) {
                        tma_load_2d(b, &L.b[w.which][q], n0, k, bar);
                        tma_load_2d(b + kMnChunk, &L.b[w.which][q], n0 + 64, k, bar);
                    } else {
                        tma_load_2d(b, &L.b[w.which][q], k, n0, bar);
                    }
                }
            }
            if (!ok) {
                gave_up();
                for (int i = 0; i < kStages; ++i)  // loads in flight, within a limit
                    if (i < at.s || at.phase) wait(smem_u32(&ready[i]), i < at.s ? at.phase : at.phase ^ 1, nullptr);
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        if (lane == 0) {
            constexpr uint32_t kFormat = OP::kF16 ? 0u : 1u;
            constexpr uint32_t kIdesc = (1u << 4) | (kFormat << 7) | (kFormat << 10) | (OP::kAMn ? 1u << 15 : 0u) |
                                        (OP::kBMn ? 1u << 16 : 0u) | ((128u >> 3) << 17) | (8u << 24);
            constexpr uint64_t kStepA = OP::kAMn ? 16 * 128 >> 4 : 2, kStepB = OP::kBMn ? 16 * 128 >> 4 : 2;
            constexpr uint64_t kLo = 2 * C::kTile >> 4;
            Ring<kStages> at;
            Ring<2> ac;
            const uint64_t a_desc = operand_desc(smem_u32(smem), OP::kAMn), b_desc = operand_desc(smem_u32(smem) + C::kTile, OP::kBMn);
            const uint32_t ready0 = smem_u32(ready), empty0 = smem_u32(empty);
            bool ok = true;
            for (int left = w.slices; left > 0 && ok;) {
                const uint32_t d = tmem + static_cast<uint32_t>(ac.s * 128);
                int n = min(left, OP::kGroup);
                left -= n;
                if (!wait(smem_u32(&accempty[ac.s]), ac.phase ^ 1, abort_flag)) { ok = false; break; }
                fence_after();
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
                            mma_one16<OP::kF16>(d, a + kLo, b, kIdesc, more);
                            mma_one16<OP::kF16>(d, a, b + kLo, kIdesc, 1);
                            mma_one16<OP::kF16>(d, a, b, kIdesc, 1);
                        } else {
                            mma_one16<OP::kF16>(d, a, b, kIdesc, more);
                        }
                        more = 1;
                    }
                    mma_commit(empty0 + 8 * at.s);
                }
                if (!ok) break;
                mma_commit(smem_u32(&accfull[ac.s]));
                ac.next();
            }
            if (!ok) gave_up();
            if (*abort_flag) drain_one(smem_u32(drained));
        }
        __syncwarp();
    }
    fence_before();
    // this CTA's rows, two at least and an even number
    const int row = 2 * share_at(64, rank, ctas), rows = 2 * share_at(64, rank + 1, ctas) - row;
    if (ctas > 1) {
        cluster_arrive();
        cluster_wait();
    } else {
        __syncthreads();
    }
    uint32_t* words = reinterpret_cast<uint32_t*>(sums + 128 * kSplitPitch);
    // A CTA that gave up has no sums: a lane has another CTA's word, looked at when that CTA's sums are here too.
    int gone = *abort_flag;
    if (lane < ctas && lane != rank) gone = load_cluster_int(smem_u32(const_cast<int*>(abort_flag)), static_cast<uint32_t>(lane));
    {
        constexpr int kBatch = 2;  // quads of a thread whose loads are under way together
        for (int i0 = threadIdx.x; i0 < rows * 32; i0 += kBatch * kSplitThreads) {
            float4 v[kBatch][kSplitMost];
            uint4 ahead[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int i = min(i0 + b * kSplitThreads, rows * 32 - 1);
                float* at = sums + (row + (i >> 5)) * kSplitPitch + 4 * (i & 31);
                ahead[b] = OP::fetch_quad(L, w.tm * 128 + row + (i >> 5), w.tn * 128 + 4 * (i & 31));
                if (ctas == 1) {
                    v[b][0] = *reinterpret_cast<float4*>(at);
                } else {
#pragma unroll
                    for (int q = 0; q < kSplitMost; ++q)
                        if (q < ctas) v[b][q] = load_cluster4(smem_u32(at), static_cast<uint32_t>(q));
                }
            }
            if (__any_sync(~0u, gone)) break;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int i = i0 + b * kSplitThreads;
                if (i >= rows * 32) break;
                float4 x = v[b][0];
#pragma unroll
                for (int q = 1; q < kSplitMost; ++q)
                    if (q < ctas) { x.x += v[b][q].x; x.y += v[b][q].y; x.z += v[b][q].z; x.w += v[b][q].w; }
                const int r = i >> 5, c = 4 * (i & 31);
                uint4 out;
                OP::finish_quad(L, w, w.tm * 128 + row + r, w.tn * 128 + c, x, ahead[b], out);
                if constexpr (OP::kMirror) *reinterpret_cast<uint4*>(words + r * kSplitPitch + c) = out;
            }
        }
    }
    const bool whole = !__any_sync(~0u, gone);
    if (ctas > 1) cluster_arrive();  // (what the others read here has been read once all have arrived)
    if constexpr (OP::kMirror) {
        __syncthreads();
        if (whole) OP::mirror(L, w, words, kSplitPitch, w.tm * 128 + row, rows, static_cast<int>(threadIdx.x));
    }
    if (ctas > 1) cluster_wait();
    __syncthreads();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256));
    }
}

// How many clusters of 1 .. kSplitMost CTAs the device holds at once: SMs belong together in groups
// whose numbers are not all multiples of them (clusters of four: 33, not 37).
struct SplitClusters {
    int most[kSplitMost + 1];
};
template <class OP>
int split_setup(SplitClusters* out) {
    using C = SplitCfg<OP>;
    static std::mutex mu;
    static SplitClusters known[64] = {};
    int dev = 0;
    int rc = require_device(&dev);
    if (rc) return rc;
    std::lock_guard<std::mutex> lk(mu);
    SplitClusters other{};
    SplitClusters& n = dev < 64 ? known[dev] : other;
    if (!n.most[0]) {
        SplitClusters x{};
        cudaError_t e = cudaFuncSetAttribute(split_product_kernel<OP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::kSmem));
        for (int ctas = 1; ctas <= kSplitMost && e == cudaSuccess; ++ctas) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(static_cast<unsigned>(ctas));
            cfg.blockDim = dim3(kSplitThreads);
            cfg.dynamicSmemBytes = C::kSmem;
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = static_cast<unsigned>(ctas);
            at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            e = cudaOccupancyMaxActiveClusters(&x.most[ctas], split_product_kernel<OP>, &cfg);
        }
        if (e != cudaSuccess) return cuda_fail(e, "split_product_kernel setup");
        x.most[0] = 1;
        n = x;
    }
    *out = n;
    return TB_OK;
}

// CTAs of a cluster with which `units` tiles of 128 x 128 of `slices` each are sooner done than `pairs`
// tiles of 256 x 256 by the pair kernel; 0 if with none.  In us (two parts): a slice takes a pair 0.82, and a CTA
// 0.42, or 0.008 for each CTA at work; sums joined, 1.  (k = 1024, both sides measured: Q Q 13 us by clusters of
// two, 22 by pairs; 4096: 300 and 110.)
inline int choose_split(const SplitClusters& clusters, long long units, long long pairs, long long slices) {
    double best = 0.82 * slices * ((pairs + kPairs - 1) / kPairs);
    int ctas = 0;
    for (int c = 1; c <= kSplitMost && c <= slices; ++c) {
        const long long most = clusters.most[c];
        if (most < 1) continue;
        const double cost = (units + most - 1) / most * ((slices + c - 1) / c) * std::max(0.42, 0.008 * std::min(units, most) * c) + (c > 1 ? 1.0 : 0.0);
        if (cost < best) best = cost, ctas = c;
    }
    return ctas;
}

// Launches for `units` tiles of 128 x 128, each by `ctas` CTAs.
template <class OP>
int launch_split(const Launch<OP>& L, long long units, int ctas, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(units * ctas));
    cfg.blockDim = dim3(kSplitThreads);
    cfg.dynamicSmemBytes = SplitCfg<OP>::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(ctas);
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = pdl_allowed(st) ? 1 : 0;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, split_product_kernel<OP>, L, ctas);
    return e == cudaSuccess ? check_launch("split_product_kernel") : cuda_fail(e, "split_product_kernel launch");
}

// By the sooner of the two.
template <class OP>
int launch_either(const Launch<OP>& L, long long units, long long pairs, long long slices, cudaStream_t st) {
    SplitClusters clusters{};
    const int rc = split_setup<OP>(&clusters);
    if (rc) return rc;
    const int ctas = choose_split(clusters, units, pairs, slices);
    return ctas ? launch_split(L, units, ctas, st) : launch_product(L, pairs, st);
}

}  // namespace pair
}  // namespace tb
