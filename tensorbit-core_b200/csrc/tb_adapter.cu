// Low-rank adapters of many requests beside a shared projection: forward and
// backward (contract in include/tb_kernels.h).
#include <algorithm>

#include "tb_act8.cuh"
#include "tb_linear.cuh"
#include "tb_pdl.cuh"
#include "tb_runtime.h"
#include "tb_tcgen05.cuh"

namespace tb {
namespace adapter {
namespace {

using bf16 = __nv_bfloat16;
using act8::View;

struct Args {
    long long n;
    int d, r, rank, na;
    const bf16 *w, *a, *b, *x, *dy;
    long long ldw, lda, ldb, ldx, ldy, lddy, lddx;
    const float* scale;
    const int32_t* who;
    bf16 *y, *dx, *da, *db;
    View x8;
};

__device__ __forceinline__ int adapter_of(const Args& g, long long t) {
    const int a = g.na ? g.who[t] : -1;
    return a >= 0 && a < g.na ? a : -1;
}
// The adapters that occur among 256 tokens, in order of first occurrence: their
// count, then their numbers.
__device__ __forceinline__ void list_adapters(const Args& g, int tile, int* who, int32_t* __restrict__ lists) {
    __shared__ int count[8];
    const int i = threadIdx.x, lane = i & 31, warp = i >> 5;
    const long long t = tile * 256ll + i;
    const int mine = t < g.n ? adapter_of(g, t) : -1;
    who[i] = mine;
    __syncthreads();
    bool first = mine >= 0;
    for (int j = 0; j < i && first; ++j) first = who[j] != mine;
    const unsigned m = __ballot_sync(~0u, first);
    if (lane == 0) count[warp] = __popc(m);
    __syncthreads();
    int at = __popc(m & ((1u << lane) - 1)), total = 0;
    for (int w = 0; w < 8; ++w) {
        if (w < warp) at += count[w];
        total += count[w];
    }
    int32_t* out = lists + static_cast<long long>(tile) * linear::kListPitch;
    if (i == 0) out[0] = total;
    if (first) out[1 + at] = mine;
}

// ---- rank-wide products on mma.sync ------------------------------------------
// m16n8k16 fragments: lane (g, t) = (lane / 4, lane % 4) holds rows g and g + 8
// of A at k = 2t, 2t+1, 2t+8, 2t+9, column g of B at the same k, and rows g and
// g + 8 of D at columns 2t, 2t+1.  Which k, row or column of the problem a slot
// stands for is free as long as both operands agree, so every fragment below is
// filled by whole 8- or 16-byte loads of consecutive values.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first `count` of eight BF16 values, zeros behind them.
__device__ __forceinline__ uint4 first_of(uint4 v, long long count) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 2 * i + 1 < count ? w[i] : 2 * i < count ? w[i] & 0xFFFFu : 0u;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 2 NT bytes, aligned to as many, as words.
__device__ __forceinline__ void load_words(const bf16* p, uint32_t (&w)[1]) { w[0] = __ldg(reinterpret_cast<const uint32_t*>(p)); }
__device__ __forceinline__ void load_words(const bf16* p, uint32_t (&w)[2]) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x; w[1] = v.y;
}
__device__ __forceinline__ void load_words(const bf16* p, uint32_t (&w)[4]) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
}

// Eight values of row t at feature f: BF16 rows, or a checkpoint decoded to BF16 (exact).
struct Rows {
    const bf16* x;   // NULL: the checkpoint
    long long ld;
    View x8;
    int cols;
};
template <bool CODES>
__device__ __forceinline__ uint4 row8(const Rows& s, long long t, int f) {
    uint4 v;
    if constexpr (CODES) {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(s.x8.codes + t * s.x8.ldq + f));
        const uint2 e = __ldg(reinterpret_cast<const uint2*>(s.x8.exps + (t / act8::kBlock) * s.x8.lde + f));
        uint32_t sc[4];
        act8::scales8(e, sc);
        v = act8::decode8(q, sc);
    } else {
        v = __ldg(reinterpret_cast<const uint4*>(s.x + t * s.ld + f));
    }
    return f + 8 <= s.cols ? v : first_of(v, s.cols - f);
}

// The value at `p`'s place in the shared memory of block `rank` of this cluster.
__device__ __forceinline__ float load_peer(const float* p, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
                 : "=f"(v)
                 : "r"(umma::smem_u32(p)), "r"(rank)
                 : "memory");
    return v;
}

// u[t][k] = scale[a] sum_c row_t[c] M_a[k][c] for the tokens with an adapter:
// 16 tokens and RC = 8 NT ranks per block, the features split over its 8 warps
// in groups of 32 and the warps' sums joined in order.  One pass for each
// adapter among the 16 tokens (runs of one request have one; a pass costs what
// the 16 tokens of one adapter do, bound by reading M_a from L2).
// ALONG: M_a = a [rank][lda], features along its rows; else M_a[k][c] = b [c][ldb].
// SPLIT > 1: a cluster of that many blocks shares the features of one tile and
// joins its sums over distributed shared memory, in order.
template <int NT, bool CODES, bool ALONG, int SPLIT>
__device__ __forceinline__ void down_project(const Args& g, const Rows& src, float* __restrict__ u, float (*red)[16][8 * NT],
                                             int* who, int passes, int mine_pass) {
    constexpr int RC = 8 * NT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
    const int share = blockIdx.x % SPLIT;
    const long long t0 = blockIdx.x / SPLIT * 16ll;
    const int rank0 = blockIdx.y * RC;
    if (threadIdx.x < 16) who[threadIdx.x] = t0 + threadIdx.x < g.n ? adapter_of(g, t0 + threadIdx.x) : -1;
    __syncthreads();
    unsigned rem = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) rem |= who[i] >= 0 ? 1u << i : 0u;
    const int groups = (src.cols + 31) / 32;
    for (int pass = 0; rem; ++pass) {
        const int a = who[__ffs(rem) - 1];
        unsigned mine = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) mine |= who[i] == a ? 1u << i : 0u;
        rem &= ~mine;
        if (pass % passes != mine_pass) continue;
        float acc[NT][4] = {};
        const bool r0 = mine >> gq & 1, r1 = mine >> (gq + 8) & 1;
#pragma unroll(NT <= 4 ? 4 : 2)
        for (int kg = share * 8 + warp; kg < groups; kg += 8 * SPLIT) {
            const int f = kg * 32 + 8 * tq;
            const bool in = f < src.cols;
            const uint4 zero = make_uint4(0, 0, 0, 0);
            const uint4 x0 = in && r0 ? row8<CODES>(src, t0 + gq, f) : zero, x1 = in && r1 ? row8<CODES>(src, t0 + gq + 8, f) : zero;
            const uint32_t w0[4] = {x0.x, x0.y, x0.z, x0.w}, w1[4] = {x1.x, x1.y, x1.z, x1.w};
            if constexpr (ALONG) {
                uint4 m[NT];
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const int k = rank0 + gq * NT + i;
                    m[i] = in && k < g.rank ? __ldg(reinterpret_cast<const uint4*>(g.a + (static_cast<long long>(a) * g.rank + k) * g.lda + f)) : zero;
                    if (f + 8 > src.cols) m[i] = first_of(m[i], src.cols - f);
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    mma16816(acc[i], w0[0], w1[0], w0[1], w1[1], m[i].x, m[i].y);
                    mma16816(acc[i], w0[2], w1[2], w0[3], w1[3], m[i].z, m[i].w);
                }
            } else {
                // rows of b at eight consecutive features, NT ranks each
                uint32_t m[8][NT / 2];
                const int k0 = rank0 + gq * NT;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bf16* p = g.b + (static_cast<long long>(a) * g.r + f + j) * g.ldb + k0;
                    const bool have = f + j < src.cols;
                    if (have && k0 + NT <= g.rank) {
                        load_words(p, m[j]);
                    } else {
#pragma unroll
                        for (int i = 0; i < NT / 2; ++i) {  // ranks behind the last are zeros (ldb is even)
                            m[j][i] = have && k0 + 2 * i < g.rank ? __ldg(reinterpret_cast<const uint32_t*>(p) + i) : 0u;
                            if (k0 + 2 * i + 1 >= g.rank) m[j][i] &= 0xFFFFu;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const uint32_t sel = i & 1 ? 0x7632u : 0x5410u;
                    mma16816(acc[i], w0[0], w1[0], w0[1], w1[1], __byte_perm(m[0][i / 2], m[1][i / 2], sel), __byte_perm(m[2][i / 2], m[3][i / 2], sel));
                    mma16816(acc[i], w0[2], w1[2], w0[3], w1[3], __byte_perm(m[4][i / 2], m[5][i / 2], sel), __byte_perm(m[6][i / 2], m[7][i / 2], sel));
                }
            }
        }
        // column 2t + e of fragment i is rank (2t + e) NT + i
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[warp][gq + 8 * (e >> 1)][(2 * tq + (e & 1)) * NT + i] = acc[i][e];
        __syncthreads();
        if constexpr (SPLIT == 1) {
            for (int i = threadIdx.x; i < 16 * RC; i += 256) {
                const int row = i / RC, k = rank0 + i % RC;
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < 8; ++w) sum += red[w][row][i % RC];
                if ((mine >> row & 1) && k < g.rank) u[(t0 + row) * g.rank + k] = g.scale[a] * sum;
            }
            __syncthreads();
        } else {
            for (int i = threadIdx.x; i < 16 * RC; i += 256) {  // each sum has one thread: in place
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < 8; ++w) sum += red[w][i / RC][i % RC];
                red[0][i / RC][i % RC] = sum;
            }
            umma::cluster_sync_all();
            for (int i = share * 256 + threadIdx.x; i < 16 * RC; i += SPLIT * 256) {
                const int row = i / RC, k = rank0 + i % RC;
                float v[SPLIT], sum = 0.0f;
#pragma unroll
                for (int q = 0; q < SPLIT; ++q) v[q] = load_peer(&red[0][row][i % RC], q);
#pragma unroll
                for (int q = 0; q < SPLIT; ++q) sum += v[q];
                if ((mine >> row & 1) && k < g.rank) u[(t0 + row) * g.rank + k] = g.scale[a] * sum;
            }
            umma::cluster_sync_all();  // no block writes its sums again, or leaves, before they have been read
        }
    }
}

// blockIdx.z = passes * q + p.  q = 0: the forward's u (from x) or the backward's
// v (from dy); 1: the backward's u (from the checkpoint).  p: of a tile's
// adapters, every passes-th.
template <int NT, bool BACKWARD, int SPLIT>
__global__ void __cluster_dims__(SPLIT, 1, 1) __launch_bounds__(256) down_kernel(const Args g, const int passes,
                                                                                float* __restrict__ first,
                                                                                float* __restrict__ second,
                                                                                int32_t* __restrict__ lists) {
    __shared__ float red[8][16][8 * NT];
    __shared__ int who[256];
    const int p = blockIdx.z % passes;
    asm volatile("griddepcontrol.launch_dependents;");  // few_tokens_kernel waits before it reads u
    if constexpr (!BACKWARD) {
        down_project<NT, false, true, SPLIT>(g, {g.x, g.ldx, {}, g.d}, first, red, who, passes, p);
    } else {
        if (static_cast<int>(blockIdx.z) < passes) down_project<NT, false, false, SPLIT>(g, {g.dy, g.lddy, {}, g.r}, first, red, who, passes, p);
        else down_project<NT, true, true, SPLIT>(g, {nullptr, 0, g.x8, g.d}, second, red, who, passes, p);
    }
    if (blockIdx.x % (16 * SPLIT) == 0 && blockIdx.y == 0 && blockIdx.z == 0) {
        __syncthreads();
        list_adapters(g, blockIdx.x / (16 * SPLIT), who, lists);
    }
}

// out_a[c][k] = sum over the tokens of adapter a of row_t[c] val_t[k]: 128
// features and RC ranks per block, the tokens of the block's share compacted in
// order and taken 64 at a time, 16 for each pair of warps; val enters as two
// BF16 parts.  The four pairs' sums, and the shares' (grid z), join in order.
// Bound by reading the rows once for each adapter that uses them.
template <int NT, bool CODES>
__global__ void __launch_bounds__(256) outer_kernel(const Args g, const Rows src, const float* __restrict__ val, const int shares,
                                                    const int chunks, float* __restrict__ part, bf16* __restrict__ out) {
    constexpr int RC = 8 * NT, kPitch = RC + 8, kScan = 1024;
    __shared__ union {
        uint32_t vp[2][32][kPitch];  // [part][pair of tokens][rank]
        float sum[128][RC + 1];      // once the tokens are done
    } sm;
    __shared__ int list[kScan + 64];
    __shared__ int warp_count[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
    const int a = blockIdx.y, share = blockIdx.z / chunks, rank0 = (blockIdx.z % chunks) * RC;
    const int f = blockIdx.x * 128 + (warp & 1) * 64 + 8 * gq;
    const long long per = (g.n + shares - 1) / shares, t_end = min(g.n, (share + 1) * per);
    float acc[4][NT][4] = {};
    int have = 0;
    for (long long base = share * per; base < t_end; base += kScan) {
        bool hit[kScan / 256];
#pragma unroll
        for (int i = 0; i < kScan / 256; ++i) {
            const long long t = base + i * 256 + threadIdx.x;
            hit[i] = t < t_end && adapter_of(g, t) == a;
        }
#pragma unroll
        for (int i = 0; i < kScan / 256; ++i) {  // append this adapter's tokens, in order
            const unsigned m = __ballot_sync(~0u, hit[i]);
            if (lane == 0) warp_count[warp] = __popc(m);
            __syncthreads();
            int at = have + __popc(m & ((1u << lane) - 1));
            for (int w = 0; w < 8; ++w) {
                if (w < warp) at += warp_count[w];
                have += warp_count[w];
            }
            if (hit[i]) list[at] = static_cast<int>(base + i * 256 + threadIdx.x);
            __syncthreads();
        }
        const bool flush = base + kScan >= t_end;
        int done = 0;
        for (; have - done >= 64 || (flush && have > done); done += 64) {
            // two tokens' values of a rank as one word, high parts and low parts
            const int pair = threadIdx.x >> 3, i0 = done + 2 * pair;
            const long long ta = i0 < have ? list[i0] : -1, tb = i0 + 1 < have ? list[i0 + 1] : -1;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int k = (threadIdx.x & 7) + 8 * i;
                const bool in = rank0 + k < g.rank;
                const float x = in && ta >= 0 ? val[ta * g.rank + rank0 + k] : 0.0f, y = in && tb >= 0 ? val[tb * g.rank + rank0 + k] : 0.0f;
                const __nv_bfloat162 hi = __floats2bfloat162_rn(x, y);
                const __nv_bfloat162 lo = __floats2bfloat162_rn(x - __low2float(hi), y - __high2float(hi));
                sm.vp[0][pair][k] = *reinterpret_cast<const uint32_t*>(&hi);
                sm.vp[1][pair][k] = *reinterpret_cast<const uint32_t*>(&lo);
            }
            __syncthreads();
            const int slot = done + (warp >> 1) * 16;
            uint32_t w[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // tokens of k slots 2t, 2t+1, 2t+8, 2t+9
                const int i = slot + 2 * tq + (j & 1) + 8 * (j >> 1);
                const uint4 v = i < have && f < src.cols ? row8<CODES>(src, list[i], f) : make_uint4(0, 0, 0, 0);
                w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
            }
            const int p = (warp >> 1) * 8 + tq;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const uint32_t h0 = sm.vp[0][p][8 * i + gq], h1 = sm.vp[0][p + 4][8 * i + gq];
                const uint32_t l0 = sm.vp[1][p][8 * i + gq], l1 = sm.vp[1][p + 4][8 * i + gq];
#pragma unroll
                for (int m = 0; m < 4; ++m) {  // rows g, g+8 of tile m: features 2m, 2m+1 of the lane's eight
                    const uint32_t a0 = __byte_perm(w[0][m], w[1][m], 0x5410), a1 = __byte_perm(w[0][m], w[1][m], 0x7632);
                    const uint32_t a2 = __byte_perm(w[2][m], w[3][m], 0x5410), a3 = __byte_perm(w[2][m], w[3][m], 0x7632);
                    mma16816(acc[m][i], a0, a1, a2, a3, l0, l1);
                    mma16816(acc[m][i], a0, a1, a2, a3, h0, h1);
                }
            }
            __syncthreads();
        }
        // what is left (fewer than 64) moves to the front
        const int left = max(0, have - done);
        const int keep = threadIdx.x < left ? list[done + threadIdx.x] : 0;
        __syncthreads();
        if (threadIdx.x < left) list[threadIdx.x] = keep;
        have = left;
        __syncthreads();
    }
    for (int q = 0; q < 4; ++q) {
        if ((warp >> 1) == q) {
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float& s = sm.sum[(warp & 1) * 64 + 8 * gq + 2 * m + (e >> 1)][8 * i + 2 * tq + (e & 1)];
                        s = q ? s + acc[m][i][e] : acc[m][i][e];
                    }
        }
        __syncthreads();
    }
    // CODES: the gradient of a, [rank][lda]; else of b, [r][ldb]
    const int f0 = blockIdx.x * 128;
    for (int i = threadIdx.x; i < 128 * RC; i += 256) {
        const int c = CODES ? i % 128 : i / RC, k = CODES ? i / 128 : i % RC;
        if (f0 + c >= src.cols || rank0 + k >= g.rank) continue;
        if (part) part[((static_cast<long long>(share) * g.na + a) * src.cols + f0 + c) * g.rank + rank0 + k] = sm.sum[c][k];
        else if (CODES) out[(static_cast<long long>(a) * g.rank + rank0 + k) * g.lda + f0 + c] = __float2bfloat16_rn(sm.sum[c][k]);
        else out[(static_cast<long long>(a) * g.r + f0 + c) * g.ldb + rank0 + k] = __float2bfloat16_rn(sm.sum[c][k]);
    }
}

// Joins the shares of outer_kernel in order.
template <bool CODES>
__global__ void __launch_bounds__(256) join_kernel(const Args g, const int cols, const int shares, const float* __restrict__ part,
                                                   bf16* __restrict__ out) {
    const long long each = static_cast<long long>(g.na) * cols * g.rank;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < each; i += gridDim.x * 256ll) {
        float s = 0.0f;
        for (int q = 0; q < shares; ++q) s += part[q * each + i];
        const int k = static_cast<int>(i % g.rank);
        const long long af = i / g.rank, a = af / cols, c = af % cols;
        out[CODES ? (a * g.rank + k) * g.lda + c : (a * g.r + c) * g.ldb + k] = __float2bfloat16_rn(s);
    }
}

// The forward for few tokens: y = x W^T + u b^T, bound by reading W once.  A
// block has 16 output features (rows of A in m16n8k16) and up to 8 NT tokens;
// its 8 warps take every eighth group of 32 in features, so that the block reads
// 512 consecutive bytes of each row at a time, and join their sums in order.
// Launched while down_kernel still runs: u is not read before the wait.
template <int NT>
__global__ void __launch_bounds__(256) few_tokens_kernel(const Args g, const float* u) {
    __shared__ float red[8][16][8 * NT + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
    const int o0 = blockIdx.x * 16, groups = (g.d + 31) / 32;
    const bf16 *w0 = g.w + (o0 + gq) * g.ldw, *w1 = w0 + 8 * g.ldw;
    const bool r0 = o0 + gq < g.r, r1 = o0 + gq + 8 < g.r;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    float acc[NT][4] = {};
#pragma unroll(NT <= 2 ? 4 : 2)
    for (int kg = warp; kg < groups; kg += 8) {
        const int f = kg * 32 + 8 * tq;
        const bool in = f < g.d;
        uint4 a0 = in && r0 ? __ldcs(reinterpret_cast<const uint4*>(w0 + f)) : zero;
        uint4 a1 = in && r1 ? __ldcs(reinterpret_cast<const uint4*>(w1 + f)) : zero;
        uint4 x[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) x[i] = in && 8 * i + gq < g.n ? __ldg(reinterpret_cast<const uint4*>(g.x + (8 * i + gq) * g.ldx + f)) : zero;
        if (f + 8 > g.d) {
            a0 = first_of(a0, g.d - f);
            a1 = first_of(a1, g.d - f);
#pragma unroll
            for (int i = 0; i < NT; ++i) x[i] = first_of(x[i], g.d - f);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            mma16816(acc[i], a0.x, a1.x, a0.y, a1.y, x[i].x, x[i].y);
            mma16816(acc[i], a0.z, a1.z, a0.w, a1.w, x[i].z, x[i].w);
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[warp][gq + 8 * (e >> 1)][8 * i + 2 * tq + (e & 1)] = acc[i][e];
    __syncthreads();
    pdl_wait();
    for (int i = threadIdx.x; i < 16 * 8 * NT; i += 256) {
        const int row = i & 15, t = i >> 4, o = o0 + row;
        if (t >= g.n || o >= g.r) continue;
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) y += red[w][row][t];
        const int a = adapter_of(g, t);
        if (a >= 0) {
            const bf16* b = g.b + (static_cast<long long>(a) * g.r + o) * g.ldb;
            for (int k = 0; k < g.rank; k += 8) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(b + k));
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k + j < g.rank)
                        y = fmaf(__ldcg(u + t * g.rank + k + j), __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16), y);
            }
        }
        g.y[t * g.ldy + o] = __float2bfloat16_rn(y);
    }
}
constexpr int kFewTokens = 32;

template <int NT>
cudaError_t launch_few(const Args& g, const float* u, cudaStream_t st) {
    return launch_pdl(few_tokens_kernel<NT>, dim3((g.r + 15) / 16), dim3(256), 0, st, g, u);
}

template <int NT, bool BACKWARD>
void launch_down(const Args& g, float* first, float* second, int32_t* lists, cudaStream_t st) {
    const unsigned tiles = static_cast<unsigned>((g.n + 15) / 16), chunks = (g.rank + 8 * NT - 1) / (8 * NT);
    if (g.n <= 1024) {
        // A small batch's tiles do not fill the GPU: a block for each adapter that a tile may hold, and
        // eight for its features.  (One token, 4096 features, rank 16: 9.4 us with one block, 4.7 with eight.)
        const int passes = std::min(16, g.na);
        down_kernel<NT, BACKWARD, 8><<<dim3(8 * tiles, chunks, (second ? 2 : 1) * passes), 256, 0, st>>>(g, passes, first, second, lists);
    } else {
        down_kernel<NT, BACKWARD, 1><<<dim3(tiles, chunks, second ? 2 : 1), 256, 0, st>>>(g, 1, first, second, lists);
    }
}
template <bool BACKWARD>
int down(const Args& g, float* first, float* second, int32_t* lists, cudaStream_t st) {
    if (g.rank <= 16) launch_down<2, BACKWARD>(g, first, second, lists, st);
    else if (g.rank <= 32) launch_down<4, BACKWARD>(g, first, second, lists, st);
    else launch_down<8, BACKWARD>(g, first, second, lists, st);
    return check_launch("down_kernel");
}

// Shares of the tokens for one gradient of `cols` features: enough blocks to
// fill the GPU about four times, but no share below 512 tokens.
int shares_of(const Args& g, int cols) {
    const long long blocks = static_cast<long long>((cols + 127) / 128) * g.na * ((g.rank + 63) / 64);
    return static_cast<int>(std::max(1ll, std::min((600 + blocks - 1) / blocks, g.n / 512)));
}
template <bool CODES>
int launch_outer(const Args& g, const Rows& src, const float* val, float* part, bf16* out, cudaStream_t st) {
    const int shares = shares_of(g, src.cols), chunks = (g.rank + 63) / 64;
    const dim3 grid((src.cols + 127) / 128, g.na, shares * chunks);
    float* p = shares > 1 ? part : nullptr;
    if (g.rank <= 16) outer_kernel<2, CODES><<<grid, 256, 0, st>>>(g, src, val, shares, chunks, p, out);
    else if (g.rank <= 32) outer_kernel<4, CODES><<<grid, 256, 0, st>>>(g, src, val, shares, chunks, p, out);
    else outer_kernel<8, CODES><<<grid, 256, 0, st>>>(g, src, val, shares, chunks, p, out);
    if (shares > 1) {
        const long long each = static_cast<long long>(g.na) * src.cols * g.rank;
        join_kernel<CODES><<<static_cast<unsigned>(std::min((each + 255) / 256, 148ll * 8)), 256, 0, st>>>(g, src.cols, shares, part, out);
    }
    return check_launch("outer_kernel");
}

// One piece of scratch: the lists, u and v, and the shares of a gradient (freed
// through `lists`).  Empty without adapters or tokens.
struct Scratch {
    int32_t* lists;
    float *u, *v, *part;
};
int make_scratch(const Args& g, bool grads, cudaStream_t st, Scratch* s) {
    if (!g.na || !g.n) return TB_OK;
    auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    const size_t list = up((g.n + 255) / 256 * linear::kListPitch * sizeof(int32_t));
    const size_t vals = up(g.n * g.rank * sizeof(float));
    size_t part = 0;
    if (grads)
        for (const int cols : {g.d, g.r}) {
            const int shares = shares_of(g, cols);
            if (shares > 1) part = std::max(part, up(static_cast<size_t>(shares) * g.na * cols * g.rank * sizeof(float)));
        }
    void* p = nullptr;
    const int rc = scratch_alloc(&p, list + (grads ? 2 : 1) * vals + part, st);
    if (rc) return rc;
    char* c = static_cast<char*>(p);
    s->lists = reinterpret_cast<int32_t*>(c);
    s->v = reinterpret_cast<float*>(c + list);
    s->u = grads ? reinterpret_cast<float*>(c + list + vals) : s->v;
    s->part = reinterpret_cast<float*>(c + list + 2 * vals);
    return TB_OK;
}

bool bad_rows(const void* p, int64_t ld, int64_t cols) {
    return !p || reinterpret_cast<uintptr_t>(p) % 16 || ld < cols || ld % 8;
}

// What forward and backward check alike; fills the common part of `g`.
int check_common(const char* who, const tb_adapter_args* p, bool need_w, Args* g) {
    if (!p || p->struct_size != sizeof(tb_adapter_args)) return fail(TB_ERR_ARG, "%s: null args or bad struct_size", who);
    if (p->dtype != TB_BF16) return fail(TB_ERR_UNSUPPORTED, "%s: TB_BF16 only (dtype %d)", who, p->dtype);
    if (p->d <= 0 || p->r <= 0) return fail(TB_ERR_ZERO_SIZE, "%s: empty projection", who);
    if (p->n < 0 || p->n > 0x7FFFFFFFll - 256) return fail(TB_ERR_SHAPE, "%s: %lld tokens", who, static_cast<long long>(p->n));
    if (p->n_adapters < 0 || p->n_adapters > 65535) return fail(TB_ERR_ARG, "%s: %d adapters", who, p->n_adapters);
    if (need_w && bad_rows(p->w, p->ldw, p->d)) return fail(TB_ERR_ARG, "%s: w must be 16-byte aligned, ldw >= d a multiple of 8", who);
    if (p->n_adapters) {
        if (p->rank < 1 || p->rank > 128) return fail(TB_ERR_SHAPE, "%s: rank %d outside 1..128", who, p->rank);
        if (bad_rows(p->a, p->lda, p->d) || bad_rows(p->b, p->ldb, p->rank))
            return fail(TB_ERR_ARG, "%s: a and b must be 16-byte aligned with row strides that are multiples of 8", who);
        if (!p->scale || (p->n > 0 && !p->token_adapter)) return fail(TB_ERR_ARG, "%s: null scale or token_adapter", who);
    }
    g->n = p->n;
    g->d = p->d;
    g->r = p->r;
    g->rank = p->n_adapters ? p->rank : 0;
    g->na = p->n_adapters;
    g->w = static_cast<const bf16*>(p->w);
    g->a = static_cast<const bf16*>(p->a);
    g->b = static_cast<const bf16*>(p->b);
    g->ldw = p->ldw;
    g->lda = p->lda;
    g->ldb = p->ldb;
    g->scale = p->scale;
    g->who = p->token_adapter;
    return TB_OK;
}

}  // namespace
}  // namespace adapter
}  // namespace tb

using namespace tb;
using namespace tb::adapter;

extern "C" int tb_adapter_forward(const tb_adapter_args* p, void* stream) {
    Args g{};
    int rc = check_common("tb_adapter_forward", p, true, &g);
    if (rc) return rc;
    if (g.n == 0) return TB_OK;
    if (bad_rows(p->x, p->ldx, g.d)) return fail(TB_ERR_ARG, "tb_adapter_forward: x must be 16-byte aligned, ldx >= d a multiple of 8");
    if (!p->y || p->ldy < g.r) return fail(TB_ERR_ARG, "tb_adapter_forward: y is null or ldy < r");
    g.x = static_cast<const bf16*>(p->x);
    g.ldx = p->ldx;
    g.y = static_cast<bf16*>(p->y);
    g.ldy = p->ldy;
    if ((rc = require_device(nullptr))) return rc;
    auto st = static_cast<cudaStream_t>(stream);
    Scratch s{};
    if ((rc = make_scratch(g, false, st, &s))) return rc;
    if (g.na) {
        rc = down<false>(g, s.u, nullptr, s.lists, st);
    }
    if (!rc && g.n <= kFewTokens) {
        const cudaError_t e = g.n <= 8 ? launch_few<1>(g, s.u, st) : g.n <= 16 ? launch_few<2>(g, s.u, st) : launch_few<4>(g, s.u, st);
        rc = e == cudaSuccess ? check_launch("few_tokens_kernel") : cuda_fail(e, "few_tokens_kernel launch");
    } else if (!rc) rc = linear::adapter_forward({g.n, g.r, g.d, g.x, g.ldx, g.w, g.ldw, g.y, g.ldy, g.who, s.lists, s.u, g.b, g.ldb, g.rank, g.na}, st);
    scratch_free(s.lists, st);
    return rc;
}

extern "C" int tb_adapter_backward(const tb_adapter_args* p, void* stream) {
    Args g{};
    int rc = check_common("tb_adapter_backward", p, p && p->dx, &g);
    if (rc) return rc;
    if (!p->da != !p->db) return fail(TB_ERR_ARG, "tb_adapter_backward: da and db are given together");
    const bool grads = p->da && g.na;
    if (grads) {
        if ((rc = act8::check(p->x8, "tb_adapter_backward", &g.x8))) return rc;
        if (g.x8.n != g.n || g.x8.d != g.d) return fail(TB_ERR_SHAPE, "tb_adapter_backward: the checkpoint is not of n x d");
    }
    if (g.n > 0 && bad_rows(p->dy, p->lddy, g.r)) return fail(TB_ERR_ARG, "tb_adapter_backward: dy must be 16-byte aligned, lddy >= r a multiple of 8");
    if (p->dx && p->lddx < g.d) return fail(TB_ERR_ARG, "tb_adapter_backward: lddx < d");
    g.dy = static_cast<const bf16*>(p->dy);
    g.lddy = p->lddy;
    g.dx = static_cast<bf16*>(p->dx);
    g.lddx = p->lddx;
    g.da = static_cast<bf16*>(p->da);
    g.db = static_cast<bf16*>(p->db);
    if ((rc = require_device(nullptr))) return rc;
    auto st = static_cast<cudaStream_t>(stream);
    Scratch s{};
    if ((rc = make_scratch(g, grads, st, &s))) return rc;
    if (s.lists) {
        rc = down<true>(g, s.v, grads ? s.u : nullptr, s.lists, st);
    }
    if (!rc && g.dx && g.n)
        rc = linear::adapter_input_grad({g.n, g.d, g.r, g.dy, g.lddy, g.w, g.ldw, g.dx, g.lddx, g.who, s.lists, s.v, g.a, g.lda, g.rank, g.na}, st);
    if (!rc && grads) {
        rc = launch_outer<true>(g, {nullptr, 0, g.x8, g.d}, s.v, s.part, g.da, st);
        if (!rc) rc = launch_outer<false>(g, {g.dy, g.lddy, {}, g.r}, s.u, s.part, g.db, st);
    }
    scratch_free(s.lists, st);
    return rc;
}
