// Low-rank adapters of many requests beside a shared projection: forward and
// backward (contract in include/tb_kernels.h).
#include <algorithm>
#include <atomic>

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
// count, then their numbers.  Called by all threads of a block of 256 or more.
__device__ __forceinline__ void list_adapters(const Args& g, int tile, int* who, int32_t* __restrict__ lists) {
    __shared__ int count[8];
    const int i = threadIdx.x, lane = i & 31, warp = i >> 5;
    const long long t = tile * 256ll + i;
    const int mine = i < 256 && t < g.n ? adapter_of(g, t) : -1;
    if (i < 256) who[i] = mine;
    __syncthreads();
    bool first = mine >= 0;
    for (int j = 0; j < i && first; ++j) first = who[j] != mine;
    const unsigned m = __ballot_sync(~0u, first);
    if (lane == 0 && warp < 8) count[warp] = __popc(m);
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

// NT values of shared memory, aligned to as many.
__device__ __forceinline__ void load_floats(const float* p, float (&v)[2]) {
    const float2 f = *reinterpret_cast<const float2*>(p);
    v[0] = f.x; v[1] = f.y;
}
__device__ __forceinline__ void load_floats(const float* p, float (&v)[4]) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
}
__device__ __forceinline__ void store_words(uint32_t* p, const uint32_t (&w)[2]) { *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]); }
__device__ __forceinline__ void store_words(uint32_t* p, const uint32_t (&w)[4]) { *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]); }

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

// The tokens of each adapter, in order, for batches that are not small (see
// small_batch()): order[start ..] holds them, and every piece of 64 has an entry of
// `tiles` at start / 64 + a + piece (adapters' entries cannot overlap there; an
// entry without a piece has adapter -1).  One block per adapter: it counts the
// tokens of lower adapters, then compacts its own.  Further blocks list the
// adapters of the tiles of 256 tokens.
struct Order {
    int2* span;     // [na] (start, count)
    int2* tiles;    // [n / 64 + na] (adapter, piece)
    int* tokens;    // [n]
};
constexpr int kSmallBatch = 1024;  // tokens at most

__global__ void __launch_bounds__(1024) order_kernel(const Args g, const Order o, int32_t* __restrict__ lists) {
    __shared__ int scan[32], total[2], who[256];
    if (static_cast<int>(blockIdx.x) >= g.na) {  // the blocks behind those of the adapters
        list_adapters(g, blockIdx.x - g.na, who, lists);
        return;
    }
    const int a = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < 2) total[tid] = 0;
    __syncthreads();
    int lower = 0, mine = 0;
    for (long long t = tid; t < g.n; t += 1024) {
        const int w = adapter_of(g, t);
        lower += w >= 0 && w < a;
        mine += w == a;
    }
    lower = __reduce_add_sync(~0u, lower);
    mine = __reduce_add_sync(~0u, mine);
    if (lane == 0) {
        atomicAdd(&total[0], lower);
        atomicAdd(&total[1], mine);
    }
    __syncthreads();
    const int start = total[0], count = total[1];
    if (tid == 0) o.span[a] = make_int2(start, count);
    const int first = start / 64 + a, pieces = (count + 63) / 64, next = (start + count) / 64 + a + 1;
    for (int p = tid; p < next - first; p += 1024) o.tiles[first + p] = make_int2(p < pieces ? a : -1, p);
    if (a == g.na - 1)
        for (long long p = next + tid; p < g.n / 64 + g.na; p += 1024) o.tiles[p] = make_int2(-1, 0);
    int at = start;
    for (long long base = 0; base < g.n; base += 4096) {  // four consecutive tokens a thread
        int t[4], n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long q = base + 4 * tid + i;
            if (q < g.n && adapter_of(g, q) == a) t[n++] = static_cast<int>(q);
        }
        int upto = n;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int v = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += v;
        }
        if (lane == 31) scan[warp] = upto;
        __syncthreads();
        int before = 0, all = 0;
        for (int w = 0; w < 32; ++w) {
            before += w < warp ? scan[w] : 0;
            all += scan[w];
        }
        for (int i = 0; i < n; ++i) o.tokens[at + before + upto - n + i] = t[i];
        at += all;
        __syncthreads();
    }
}

// acc[m][i] += rows of 16 tokens times ranks of adapter a, over every kstep-th
// group of 32 features: lane (g, t) has features 8t..8t+7 of the group, rows
// tok[2m], tok[2m+1] (-1: none) and ranks rank0 + g NT + i.  ALONG: M_a = a
// [rank][lda], features along its rows; else M_a[k][c] = b [c][ldb].
template <int NT, int MT, bool CODES, bool ALONG>
__device__ __forceinline__ void accumulate(const Args& g, const Rows& src, int a, const int (&tok)[2 * MT], int rank0, int kg0,
                                           int kstep, float (&acc)[MT][NT][4]) {
    const int lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
    const int groups = (src.cols + 31) / 32;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    // (Rank 64, 8000 tokens, v and u: 57 us; with two steps of NT = 8 unrolled 63, with three blocks an SM 84, in two chunks of 32 ranks 74.)
#pragma unroll(MT == 1 && NT <= 4 ? 4 : 1)
    for (int kg = kg0; kg < groups; kg += kstep) {
        const int f = kg * 32 + 8 * tq;
        const bool in = f < src.cols;
        uint32_t x[2 * MT][4];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            const uint4 v = in && tok[i] >= 0 ? row8<CODES>(src, tok[i], f) : zero;
            x[i][0] = v.x; x[i][1] = v.y; x[i][2] = v.z; x[i][3] = v.w;
        }
        if constexpr (ALONG) {
            uint4 m[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int k = rank0 + gq * NT + i;
                m[i] = in && k < g.rank ? __ldg(reinterpret_cast<const uint4*>(g.a + (static_cast<long long>(a) * g.rank + k) * g.lda + f)) : zero;
                if (f + 8 > src.cols) m[i] = first_of(m[i], src.cols - f);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int q = 0; q < MT; ++q) {
                    mma16816(acc[q][i], x[2 * q][0], x[2 * q + 1][0], x[2 * q][1], x[2 * q + 1][1], m[i].x, m[i].y);
                    mma16816(acc[q][i], x[2 * q][2], x[2 * q + 1][2], x[2 * q][3], x[2 * q + 1][3], m[i].z, m[i].w);
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
                const uint32_t b0 = __byte_perm(m[0][i / 2], m[1][i / 2], sel), b1 = __byte_perm(m[2][i / 2], m[3][i / 2], sel);
                const uint32_t b2 = __byte_perm(m[4][i / 2], m[5][i / 2], sel), b3 = __byte_perm(m[6][i / 2], m[7][i / 2], sel);
#pragma unroll
                for (int q = 0; q < MT; ++q) {
                    mma16816(acc[q][i], x[2 * q][0], x[2 * q + 1][0], x[2 * q][1], x[2 * q + 1][1], b0, b1);
                    mma16816(acc[q][i], x[2 * q][2], x[2 * q + 1][2], x[2 * q][3], x[2 * q + 1][3], b2, b3);
                }
            }
        }
    }
}
// One warp's 16 x RC sums into its place of `red`: column 2t + e of fragment i is rank (2t + e) NT + i.
template <int NT>
__device__ __forceinline__ void stage_sums(float (*red)[16][8 * NT], const float (&acc)[NT][4]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[warp][gq + 8 * (e >> 1)][(2 * tq + (e & 1)) * NT + i] = acc[i][e];
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

// u[t][k] = scale[a] sum_c row_t[c] M_a[k][c] for the tokens with an adapter.

// Small batches: 16 consecutive tokens per cluster of kSplit blocks, which share
// their features out over 8 kSplit warps and join the sums in order, the blocks'
// over distributed shared memory.  One pass for each adapter among the 16
// tokens; blockIdx.z spreads the passes over blocks (every passes-th).
constexpr int kSplit = 8;
template <int NT, bool CODES, bool ALONG>
__device__ __forceinline__ void down_small(const Args& g, const Rows& src, float* __restrict__ u, float (*red)[16][8 * NT],
                                           int* who, int passes, int mine_pass) {
    constexpr int RC = 8 * NT;
    const int gq = (threadIdx.x & 31) >> 2, share = blockIdx.x % kSplit;
    const int t0 = blockIdx.x / kSplit * 16, rank0 = blockIdx.y * RC;
    if (threadIdx.x < 16) who[threadIdx.x] = t0 + threadIdx.x < g.n ? adapter_of(g, t0 + threadIdx.x) : -1;
    __syncthreads();
    unsigned rem = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) rem |= who[i] >= 0 ? 1u << i : 0u;
    for (int pass = 0; rem; ++pass) {
        const int a = who[__ffs(rem) - 1];
        unsigned mine = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) mine |= who[i] == a ? 1u << i : 0u;
        rem &= ~mine;
        if (pass % passes != mine_pass) continue;
        float acc[1][NT][4] = {};
        const int tok[2] = {mine >> gq & 1 ? t0 + gq : -1, mine >> (gq + 8) & 1 ? t0 + gq + 8 : -1};
        accumulate<NT, 1, CODES, ALONG>(g, src, a, tok, rank0, share * 8 + (threadIdx.x >> 5), 8 * kSplit, acc);
        stage_sums<NT>(red, acc[0]);
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * RC; i += 256) {  // each sum has one thread: in place
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) sum += red[w][i / RC][i % RC];
            red[0][i / RC][i % RC] = sum;
        }
        umma::cluster_sync_all();
        for (int i = share * 256 + threadIdx.x; i < 16 * RC; i += kSplit * 256) {
            const int row = i / RC, k = rank0 + i % RC;
            float v[kSplit], sum = 0.0f;
#pragma unroll
            for (int q = 0; q < kSplit; ++q) v[q] = load_peer(&red[0][row][i % RC], q);
#pragma unroll
            for (int q = 0; q < kSplit; ++q) sum += v[q];
            if ((mine >> row & 1) && k < g.rank) u[(t0 + row) * g.rank + k] = g.scale[a] * sum;
        }
        umma::cluster_sync_all();  // no block writes its sums again, or leaves, before they have been read
    }
}

// blockIdx.z = passes * q + p.  q = 0: the forward's u (from x) or the backward's
// v (from dy); 1: the backward's u (from the checkpoint).
template <int NT, bool BACKWARD>
__global__ void __cluster_dims__(kSplit, 1, 1) __launch_bounds__(256)
down_small_kernel(const Args g, const int passes, const bool few, float* __restrict__ first, float* __restrict__ second,
                  int32_t* __restrict__ lists) {
    __shared__ float red[8][16][8 * NT];
    __shared__ int who[256];
    const int p = blockIdx.z % passes;
    // Only where few_tokens_kernel follows, which waits before it reads u (see launch_pdl's contract).
    if (few) asm volatile("griddepcontrol.launch_dependents;");
    if constexpr (!BACKWARD) {
        down_small<NT, false, true>(g, {g.x, g.ldx, {}, g.d}, first, red, who, passes, p);
    } else {
        if (static_cast<int>(blockIdx.z) < passes) down_small<NT, false, false>(g, {g.dy, g.lddy, {}, g.r}, first, red, who, passes, p);
        else down_small<NT, true, true>(g, {nullptr, 0, g.x8, g.d}, second, red, who, passes, p);
    }
    if (blockIdx.x % (16 * kSplit) == 0 && blockIdx.y == 0 && blockIdx.z == 0) {
        __syncthreads();
        list_adapters(g, blockIdx.x / (16 * kSplit), who, lists);
    }
}

// Larger batches: 64 tokens of one adapter (a piece of Order) per cluster of
// kPieceSplit blocks, 16 for each pair of a block's warps, which share the
// features out over the blocks and the pair; the adapter's factor comes once
// from L2 and four times from L1.  The pair's sums and the blocks' join in
// order, the latter over distributed shared memory.  Bound by the latency of the
// loads.  (8000 tokens, rank 64, v and u: 113 us with the features over all 8
// warps of one block, each with all 64 tokens; 57 us like this.)
constexpr int kPieceSplit = 4;
template <int NT, bool CODES, bool ALONG>
__device__ __forceinline__ void down_piece(const Args& g, const Rows& src, const Order& o, float* __restrict__ u, float (*sums)[8 * NT + 1]) {
    constexpr int RC = 8 * NT;
    const int2 tile = o.tiles[blockIdx.x / kPieceSplit];
    const int a = tile.x, share = blockIdx.x % kPieceSplit;
    if (a < 0) return;
    const int2 span = o.span[a];
    const int* tokens = o.tokens + span.x + 64 * tile.y;
    const int warp = threadIdx.x >> 5, gq = (threadIdx.x & 31) >> 2, tq = threadIdx.x & 3;
    const int count = min(64, span.y - 64 * tile.y), rank0 = blockIdx.y * RC;
    const int row0 = 16 * (warp & 3) + gq, half = warp >> 2;
    const int tok[2] = {row0 < count ? tokens[row0] : -1, row0 + 8 < count ? tokens[row0 + 8] : -1};
    float acc[1][NT][4] = {};
    accumulate<NT, 1, CODES, ALONG>(g, src, a, tok, rank0, share * 2 + half, 2 * kPieceSplit, acc);
    for (int h = 0; h < 2; ++h) {
        if (half == h) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // column 2t + e of fragment i is rank (2t + e) NT + i
                    float& s = sums[row0 + 8 * (e >> 1)][(2 * tq + (e & 1)) * NT + i];
                    s = h ? s + acc[0][i][e] : acc[0][i][e];
                }
        }
        __syncthreads();
    }
    umma::cluster_sync_all();
    for (int i = share * 256 + threadIdx.x; i < 64 * RC; i += kPieceSplit * 256) {
        const int row = i / RC, k = rank0 + i % RC;
        float v[kPieceSplit], sum = 0.0f;
#pragma unroll
        for (int q = 0; q < kPieceSplit; ++q) v[q] = load_peer(&sums[row][i % RC], q);
#pragma unroll
        for (int q = 0; q < kPieceSplit; ++q) sum += v[q];
        if (row < count && k < g.rank) u[static_cast<long long>(tokens[row]) * g.rank + k] = g.scale[a] * sum;
    }
    umma::cluster_sync_all();  // no block leaves before its sums have been read
}
template <int NT, bool BACKWARD>
__global__ void __cluster_dims__(kPieceSplit, 1, 1) __launch_bounds__(256)
down_kernel(const Args g, const Order o, float* __restrict__ first, float* __restrict__ second) {
    __shared__ float sums[64][8 * NT + 1];
    if constexpr (!BACKWARD) {
        down_piece<NT, false, true>(g, {g.x, g.ldx, {}, g.d}, o, first, sums);
    } else {
        if (blockIdx.z == 0) down_piece<NT, false, false>(g, {g.dy, g.lddy, {}, g.r}, o, first, sums);
        else down_piece<NT, true, true>(g, {nullptr, 0, g.x8, g.d}, o, second, sums);
    }
}

// Tokens of each of `shares` shares of `count`: whole pieces of 64.
__device__ __forceinline__ int share_of(int count, int shares) { return ((count + 63) / 64 + shares - 1) / shares * 64; }
// Where element (feature c, rank k) of adapter a's gradient is: of a, [rank][lda], or of b, [r][ldb].
template <bool OF_A>
__device__ __forceinline__ long long grad_at(const Args& g, int a, int c, int k) {
    return OF_A ? (static_cast<long long>(a) * g.rank + k) * g.lda + c : (static_cast<long long>(a) * g.r + c) * g.ldb + k;
}

// Zeros for those of two BF16 values that are not finite.
__device__ __forceinline__ uint32_t finite_of(uint32_t w) {
    if ((w & 0x7F80u) == 0x7F80u) w &= 0xFFFF0000u;
    if ((w & 0x7F800000u) == 0x7F800000u) w &= 0xFFFFu;
    return w;
}

// A copy of BYTES that this thread waits for by itself, or as many zeros.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool have) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(have ? BYTES : 0) : "memory");
}

// The gradients of both factors: out_a[c][k] = sum over adapter a's tokens of
// row_t[c] val_t[k], rows of the checkpoint with v for a, of dy with u for b.
// A block has 128 features and RC ranks of one adapter and a share of its
// tokens, taken 64 at a time, 16 for each pair of warps; val enters as two BF16
// parts.  Bound by the latency of the rows and values: each thread copies what it
// will read itself kAhead steps ahead, through shared memory (8000 tokens, rank
// 64: 104 us one step ahead in registers, 77 so).  The four pairs' sums,
// and the shares', join in a fixed order.
constexpr int kAhead = 2, kRing = kAhead + 1;
template <int NT>
struct OuterSmem {
    uint4 rows[kRing][4][256];        // (codes: 8 bytes of them, 8 of their exponents)
    float vals[kRing][2][256][NT];    // NT ranks of two tokens
    union {
        uint32_t vp[2][32][8 * NT + 8];  // [part][pair of tokens][rank]
        float sum[128][8 * NT + 1];      // once the tokens are done
    };
    int list[kSmallBatch];  // a small batch's tokens of this adapter
    int warp_count[8];
};

template <int NT, bool CODES>
__device__ __forceinline__ void outer_product(const Args& g, const Rows& src, const float* __restrict__ val, const Order& o, int tile,
                                              int share, int shares, int rank0, float* __restrict__ part, bf16* __restrict__ out,
                                              OuterSmem<NT>& sm) {
    constexpr int RC = 8 * NT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3, a = blockIdx.y;
    const int f = tile * 128 + (warp & 1) * 64 + 8 * gq;
    const int* tokens = sm.list;
    int count = 0;
    if (o.tokens) {
        const int2 span = o.span[a];
        tokens = o.tokens + span.x;
        count = span.y;
    } else {
        for (int i = 0; i < kSmallBatch / 256; ++i) {  // compact them here
            const int t = i * 256 + threadIdx.x;
            const bool hit = t < g.n && adapter_of(g, t) == a;
            const unsigned m = __ballot_sync(~0u, hit);
            if (lane == 0) sm.warp_count[warp] = __popc(m);
            __syncthreads();
            int at = count + __popc(m & ((1u << lane) - 1));
            for (int w = 0; w < 8; ++w) {
                if (w < warp) at += sm.warp_count[w];
                count += sm.warp_count[w];
            }
            if (hit) sm.list[at] = t;
            __syncthreads();
        }
    }
    const int per = share_of(count, shares), end = min(count, (share + 1) * per), begin = share * per;
    float acc[4][NT][4] = {};
    const int pair = threadIdx.x >> 3, k8 = threadIdx.x & 7, k0 = rank0 + k8 * NT;
    const bool whole = g.rank % NT == 0;  // copies of NT ranks are aligned
    // Tokens of this thread in the 64 from `from` on, -1 behind the last: four rows, k slots 2t, 2t+1, 2t+8,
    // 2t+9 of the fragments, and two tokens' values.
    int tok[6];
    auto find = [&](int from) {
#pragma unroll
        for (int j = 0; j < 6; ++j) {
            const int i = from + (j < 4 ? (warp >> 1) * 16 + 2 * tq + (j & 1) + 8 * (j >> 1) : 2 * pair + j - 4);
            tok[j] = i < end ? tokens[i] : -1;
        }
    };
    auto fetch = [&](int stage) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool have = tok[j] >= 0 && f < src.cols;
            const long long t = have ? tok[j] : 0;
            const int at = have ? f : 0;
            const uint32_t dst = umma::smem_u32(&sm.rows[stage][j][threadIdx.x]);
            if constexpr (CODES) {
                copy_async<8>(dst, src.x8.codes + t * src.x8.ldq + at, have);
                copy_async<8>(dst + 8, src.x8.exps + t / act8::kBlock * src.x8.lde + at, have);
            } else {
                copy_async<16>(dst, src.x + t * src.ld + at, have);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = tok[4 + i];
            const uint32_t dst = umma::smem_u32(sm.vals[stage][i][threadIdx.x]);
            const float* from = val + static_cast<long long>(max(t, 0)) * g.rank;
            if (whole) {  // (k0 < rank then holds for all NT or none)
                copy_async<4 * NT>(dst, from + (k0 < g.rank ? k0 : 0), t >= 0 && k0 < g.rank);
            } else {
#pragma unroll
                for (int j = 0; j < NT; ++j) copy_async<4>(dst + 4 * j, from + (k0 + j < g.rank ? k0 + j : 0), t >= 0 && k0 + j < g.rank);
            }
        }
    };
    int stage = 0;
    find(begin);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        if (begin + 64 * i < end) fetch(i);
        asm volatile("cp.async.commit_group;" ::: "memory");
        find(begin + 64 * (i + 1));
    }
    for (int from = begin; from < end; from += 64) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        uint32_t w[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint4 v = sm.rows[stage][j][threadIdx.x];
            if constexpr (CODES) {
                uint32_t sc[4];
                act8::scales8(make_uint2(v.z, v.w), sc);
                v = act8::decode8(make_uint2(v.x, v.y), sc);
            }
            if (f + 8 > src.cols) v = first_of(v, src.cols - f);
            w[j][0] = v.x; w[j][1] = v.y; w[j][2] = v.z; w[j][3] = v.w;
        }
        // rows g, g+8 of tile m: features 2m, 2m+1 of the lane's eight
        uint32_t x[4][4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            x[m][0] = __byte_perm(w[0][m], w[1][m], 0x5410);
            x[m][1] = __byte_perm(w[0][m], w[1][m], 0x7632);
            x[m][2] = __byte_perm(w[2][m], w[3][m], 0x5410);
            x[m][3] = __byte_perm(w[2][m], w[3][m], 0x7632);
        }
        __syncthreads();
        uint32_t hi[NT], lo[NT];  // two tokens' values of a rank as one word, high parts and low parts
        float va[NT], vb[NT];
        load_floats(sm.vals[stage][0][threadIdx.x], va);
        load_floats(sm.vals[stage][1][threadIdx.x], vb);
#pragma unroll
        for (int i = 0; i < NT; ++i) linear::split_pair(va[i], vb[i], hi[i], lo[i]);
        store_words(&sm.vp[0][pair][k8 * NT], hi);
        store_words(&sm.vp[1][pair][k8 * NT], lo);
        __syncthreads();
        if (from + 64 * kAhead < end) fetch(stage == 0 ? kRing - 1 : stage - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        find(from + 64 * (kAhead + 1));
        stage = stage == kRing - 1 ? 0 : stage + 1;
        const int p = (warp >> 1) * 8 + tq;
        // Times an infinity of the row a value's low part, which may be zero or of the other sign, would make a
        // NaN of it: such rows have their low products apart, without it.  (An exponent of all ones carries out
        // of the exponent's bits.)
        uint32_t odd = 0;
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) odd |= (x[m][j] & 0x7F807F80u) + 0x00800080u;
        if (__any_sync(~0u, odd & 0x80008000u)) {
#pragma unroll 1
            for (int part = 0; part < 2; ++part) {
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        mma16816(acc[m][i], x[m][0], x[m][1], x[m][2], x[m][3], sm.vp[part][p][8 * i + gq], sm.vp[part][p + 4][8 * i + gq]);
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[m][j] = finite_of(x[m][j]);
            }
            continue;
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint32_t h0 = sm.vp[0][p][8 * i + gq], h1 = sm.vp[0][p + 4][8 * i + gq];
            const uint32_t l0 = sm.vp[1][p][8 * i + gq], l1 = sm.vp[1][p + 4][8 * i + gq];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                mma16816(acc[m][i], x[m][0], x[m][1], x[m][2], x[m][3], l0, l1);
                mma16816(acc[m][i], x[m][0], x[m][1], x[m][2], x[m][3], h0, h1);
            }
        }
    }
    __syncthreads();
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
    if (shares > 1 && begin >= end && share > 0) return;  // nothing of this share: join_kernel does not read it
    const int f0 = tile * 128;
    for (int i = threadIdx.x; i < 128 * RC; i += 256) {
        const int c = CODES ? i % 128 : i / RC, k = CODES ? i / 128 : i % RC;
        if (f0 + c >= src.cols || rank0 + k >= g.rank) continue;
        if (shares > 1) part[((static_cast<long long>(share) * g.na + a) * src.cols + f0 + c) * g.rank + rank0 + k] = sm.sum[c][k];
        else out[grad_at<CODES>(g, a, f0 + c, rank0 + k)] = __float2bfloat16_rn(sm.sum[c][k]);
    }
}

// Blocks (tile of 128 features of a, then of b; adapter; share and rank chunk).
template <int NT>
__global__ void __launch_bounds__(256) outer_kernel(const Args g, const Order o, const float* __restrict__ v, const float* __restrict__ u,
                                                    const int shares, const int chunks, float* __restrict__ part) {
    extern __shared__ uint4 outer_smem[];
    OuterSmem<NT>& sm = *reinterpret_cast<OuterSmem<NT>*>(outer_smem);
    const int tiles_a = (g.d + 127) / 128, share = blockIdx.z / chunks, rank0 = blockIdx.z % chunks * 8 * NT;
    const int tile = blockIdx.x;
    if (tile < tiles_a) outer_product<NT, true>(g, {nullptr, 0, g.x8, g.d}, v, o, tile, share, shares, rank0, part, g.da, sm);
    else outer_product<NT, false>(g, {g.dy, g.lddy, {}, g.r}, u, o, tile - tiles_a, share, shares, rank0,
                                  part + static_cast<long long>(shares) * g.na * g.d * g.rank, g.db, sm);
}

// Joins the shares of outer_kernel in order.
__global__ void __launch_bounds__(256) join_kernel(const Args g, const Order o, const int shares, const float* __restrict__ part) {
    const long long each_a = static_cast<long long>(g.na) * g.d * g.rank, each_b = static_cast<long long>(g.na) * g.r * g.rank;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < each_a + each_b; i += gridDim.x * 256ll) {
        const bool of_a = i < each_a;
        const long long each = of_a ? each_a : each_b, j = of_a ? i : i - each_a;
        const float* p = part + (of_a ? 0 : shares * each_a) + j;
        const int k = static_cast<int>(j % g.rank), cols = of_a ? g.d : g.r;
        const int a = static_cast<int>(j / g.rank / cols), c = static_cast<int>(j / g.rank % cols);
        const int count = o.span[a].y, per = share_of(count, shares);
        float s = p[0];
        for (int q = 1; q < shares && q * per < count; ++q) s += p[q * each];
        if (of_a) g.da[grad_at<true>(g, a, c, k)] = __float2bfloat16_rn(s);
        else g.db[grad_at<false>(g, a, c, k)] = __float2bfloat16_rn(s);
    }
}

// The forward for few tokens: y = x W^T + u b^T, bound by reading W once.  A
// block has 16 output features (rows of A in m16n8k16) and up to 8 NT tokens;
// its 8 warps take every eighth group of 32 in features, so that the block reads
// 512 consecutive bytes of each row at a time, and join their sums in order.
// Launched while down_small_kernel still runs: u is not read before the wait, while
// x and w, which no kernel here writes, are.
constexpr int kMaxRank = 128;
template <int NT>
__global__ void __launch_bounds__(256) few_tokens_kernel(const Args g, const float* u) {
    __shared__ float red[8][16][8 * NT + 1], su[8 * NT * kMaxRank];
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
    pdl_wait();
    // (Read from memory for each output, 19 tokens at rank 128 took 48 us, 10163 features, and 28 so.)
    for (int i = threadIdx.x; i < g.n * g.rank; i += 256) su[i] = __ldcg(u + i);
    __syncthreads();
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
                        y = fmaf(su[t * g.rank + k + j], __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16), y);
            }
        }
        g.y[t * g.ldy + o] = __float2bfloat16_rn(y);
    }
}
// Where it is the sooner: up to 16 tokens, or 32 with at most 2^25 weights or from
// eight adapters on (each in a tile is a slice of its own, about 2.6 us); without
// adapters not where W's rows are longer than 8192.  (us of a call, W from memory,
// tokens of eight adapters of rank 16 mixed, or without adapters; this kernel against
// tiles: 4096 -> 4096, 16 tokens 15.7 and 34.6, without 14.3 and 17.1; 32 tokens 22.6
// and 35.8, without 15.8 and 17.8.  4096 -> 14336, 16 tokens 32.1 and 49.9, without
// 29.8 and 28.8; 24 tokens 47.3 and 50.3, without 42.5 and 29.0.  8192 -> 8192, one
// token 31.4 and 53.0, without 29.6 and 46.9; 24 tokens 59.3 and 58.6, without 55.2
// and 36.2.  14336 -> 4096, one token 44.7 and 47.7, without 43.4 and 36.8; 16 tokens
// 46.1 and 56.7, without 44.4 and 31.7; 32 tokens 59.6 and 57.6, without 48.9 and 32.9.)
bool few_tokens(const Args& g) {
    if (!g.na && g.d > 8192) return false;
    return g.n <= 16 || (g.n <= 32 && (g.na >= 8 || static_cast<long long>(g.r) * g.d <= 1ll << 25));
}

template <int NT>
cudaError_t launch_few(const Args& g, const float* u, cudaStream_t st) {
    // Without adapters the kernel before this one is the caller's, which may still be writing x when it lets go.
    if (!g.na) {
        few_tokens_kernel<NT><<<(g.r + 15) / 16, 256, 0, st>>>(g, u);
        return cudaGetLastError();
    }
    return launch_pdl(few_tokens_kernel<NT>, dim3((g.r + 15) / 16), dim3(256), 0, st, g, u);
}

// One piece of scratch: the lists, u and v, the order of the tokens and the shares
// of the gradients (freed through `lists`).  Empty without adapters or tokens.
struct Scratch {
    int32_t* lists;
    float *u, *v, *part;
    Order order;
    int shares;
};
// Batches whose tokens are taken as they lie, 16 at a time, with a pass for each
// adapter among them, against ordered by adapter first, two launches for one.  The
// passes grow with the tokens and, where those of many adapters are mixed, with the
// adapters; the ordering with the adapters alone.  (Time of whole calls, ordered over
// as they lie, geometric mean of forward and backward, 1024 -> 512 to 4096 -> 14336,
// ranks 8 to 128.  In runs of one adapter each: 4 adapters, 512 tokens 1.10, 768 0.98;
// 16 adapters, 128 tokens 1.06, 256 1.06, 512 0.93, 1024 0.69.  Mixed: 4 adapters, 256
// tokens 0.94, 512 0.75; 16 adapters, 64 tokens 0.87, 128 0.69, 1024 0.22; 64 adapters,
// 64 tokens 0.95, 256 0.74.  An adapter each: 2048 adapters, 130 tokens 0.98,
// 1024 0.82; 8192, forward, 130 tokens 1.47, 1024 1.03.)
bool small_batch(const Args& g) { return g.n <= (g.na > 2048 ? kSmallBatch : g.na < 16 ? 512 : 128); }

int make_scratch(const Args& g, bool grads, cudaStream_t st, Scratch* s) {
    s->shares = 1;
    if (!g.na || !g.n) return TB_OK;
    const bool ordered = !small_batch(g);
    if (grads && ordered) {
        // Enough blocks to fill the GPU about four times, but no share of an even split below 512 tokens.
        const long long blocks = static_cast<long long>((g.d + 127) / 128 + (g.r + 127) / 128) * g.na * ((g.rank + 31) / 32);
        s->shares = static_cast<int>(std::max(1ll, std::min(600 / blocks, g.n / g.na / 512)));
    }
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const size_t lists = take((g.n + 255) / 256 * linear::kListPitch * sizeof(int32_t));
    const size_t v = take(g.n * g.rank * sizeof(float)), u = grads ? take(g.n * g.rank * sizeof(float)) : v;
    const size_t span = take(ordered ? g.na * sizeof(int2) : 0), tiles = take(ordered ? (g.n / 64 + g.na) * sizeof(int2) : 0);
    const size_t tokens = take(ordered ? g.n * sizeof(int) : 0);
    const size_t part = take(s->shares > 1 ? static_cast<size_t>(s->shares) * g.na * (static_cast<size_t>(g.d) + g.r) * g.rank * sizeof(float) : 0);
    void* p = nullptr;
    const int rc = scratch_alloc(&p, at, st);
    if (rc) return rc;
    char* c = static_cast<char*>(p);
    s->lists = reinterpret_cast<int32_t*>(c + lists);
    s->v = reinterpret_cast<float*>(c + v);
    s->u = reinterpret_cast<float*>(c + u);
    if (ordered) s->order = {reinterpret_cast<int2*>(c + span), reinterpret_cast<int2*>(c + tiles), reinterpret_cast<int*>(c + tokens)};
    s->part = reinterpret_cast<float*>(c + part);
    return TB_OK;
}

// u of the forward (into `first`), or v and u of the backward.
template <int NT, bool BACKWARD>
void launch_down(const Args& g, const Scratch& s, bool few, float* first, float* second, cudaStream_t st) {
    const unsigned chunks = (g.rank + 8 * NT - 1) / (8 * NT), two = second ? 2 : 1;
    if (small_batch(g)) {
        // A small batch's tiles do not fill the GPU: a block for each adapter that a tile may hold, and
        // eight for its features.  (One token, 4096 features, rank 16: 9.4 us with one block, 4.7 with eight.)
        const int passes = std::min(16, g.na);
        const unsigned tiles = static_cast<unsigned>((g.n + 15) / 16);
        down_small_kernel<NT, BACKWARD><<<dim3(kSplit * tiles, chunks, two * passes), 256, 0, st>>>(g, passes, few, first, second, s.lists);
    } else {
        order_kernel<<<static_cast<unsigned>(g.na + (g.n + 255) / 256), 1024, 0, st>>>(g, s.order, s.lists);
        down_kernel<NT, BACKWARD><<<dim3(static_cast<unsigned>(kPieceSplit * (g.n / 64 + g.na)), chunks, two), 256, 0, st>>>(g, s.order, first, second);
    }
}
template <bool BACKWARD>
int down(const Args& g, const Scratch& s, bool few, float* first, float* second, cudaStream_t st) {
    if (g.rank <= 16) launch_down<2, BACKWARD>(g, s, few, first, second, st);
    else if (g.rank <= 32) launch_down<4, BACKWARD>(g, s, few, first, second, st);
    else launch_down<8, BACKWARD>(g, s, few, first, second, st);
    return check_launch("down_kernel");
}

template <int NT>
int launch_outer(const Args& g, const Scratch& s, int chunks, cudaStream_t st) {
    constexpr int kBytes = sizeof(OuterSmem<NT>);
    static std::atomic<uint64_t> prepared{0};  // per device: the shared-memory limit
    int dev = 0;
    const int rc = require_device(&dev);
    if (rc) return rc;
    if (dev >= 64 || !(prepared.load() >> dev & 1)) {
        const cudaError_t e = cudaFuncSetAttribute(outer_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        if (e != cudaSuccess) return cuda_fail(e, "outer_kernel setup");
        if (dev < 64) prepared |= 1ull << dev;
    }
    const dim3 grid((g.d + 127) / 128 + (g.r + 127) / 128, g.na, s.shares * chunks);
    outer_kernel<NT><<<grid, 256, kBytes, st>>>(g, s.order, s.v, s.u, s.shares, chunks, s.part);
    return check_launch("outer_kernel");
}
int gradients(const Args& g, const Scratch& s, cudaStream_t st) {
    // 32 ranks a block at most: with 64 (206 registers, one block an SM) rank 64 took 125 + 18 us where this took 102 us
    const int chunks = (g.rank + 31) / 32;
    const int rc = g.rank <= 16 ? launch_outer<2>(g, s, chunks, st) : launch_outer<4>(g, s, chunks, st);
    if (rc) return rc;
    if (s.shares > 1) {
        const long long all = static_cast<long long>(g.na) * (static_cast<long long>(g.d) + g.r) * g.rank;
        join_kernel<<<static_cast<unsigned>(std::min((all + 255) / 256, 148ll * 8)), 256, 0, st>>>(g, s.order, s.shares, s.part);
    }
    return check_launch("join_kernel");
}

bool bad_rows(const void* p, int64_t ld, int64_t cols) {
    return !p || reinterpret_cast<uintptr_t>(p) % 16 || ld < cols || ld % 8;
}

// What forward and backward check alike; fills the common part of `g`.
int check_common(const char* who, const tb_adapter_args* p, bool need_w, Args* g) {
    if (!p || p->struct_size != sizeof(tb_adapter_args)) return fail(TB_ERR_ARG, "%s: null args or bad struct_size", who);
    if (p->dtype != TB_BF16) return fail(TB_ERR_UNSUPPORTED, "%s: TB_BF16 only (dtype %d)", who, p->dtype);
    if (p->d <= 0 || p->r <= 0) return fail(TB_ERR_ZERO_SIZE, "%s: empty projection", who);
    if (p->d > act8::kMaxFeatures || p->r > act8::kMaxFeatures) return fail(TB_ERR_SHAPE, "%s: %d in and %d out features", who, p->d, p->r);
    if (p->n < 0 || p->n > 0x7FFFFFFFll - 65536) return fail(TB_ERR_SHAPE, "%s: %lld tokens", who, static_cast<long long>(p->n));
    if (p->n_adapters < 0 || p->n_adapters > 65535) return fail(TB_ERR_ARG, "%s: %d adapters", who, p->n_adapters);
    if (need_w && bad_rows(p->w, p->ldw, p->d)) return fail(TB_ERR_ARG, "%s: w must be 16-byte aligned, ldw >= d a multiple of 8", who);
    if (p->n_adapters) {
        if (p->rank < 1 || p->rank > kMaxRank) return fail(TB_ERR_SHAPE, "%s: rank %d outside 1..%d", who, p->rank, kMaxRank);
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
    const bool few = few_tokens(g);
    if (g.na) {
        rc = down<false>(g, s, few, s.u, nullptr, st);
    }
    if (!rc && few) {
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
        rc = down<true>(g, s, false, s.v, grads ? s.u : nullptr, st);
    }
    if (!rc && g.dx && g.n)
        rc = linear::adapter_input_grad({g.n, g.d, g.r, g.dy, g.lddy, g.w, g.ldw, g.dx, g.lddx, g.who, s.lists, s.v, g.a, g.lda, g.rank, g.na}, st);
    if (!rc && grads) rc = gradients(g, s, st);
    scratch_free(s.lists, st);
    return rc;
}
