// Softmax cross entropy at the LM head and its gradients, without the logits in
// memory.
//
//   z_tv = cap(h_t . w_v), cap(x) = x or c tanh(x / c)
//   lse_t = log sum_v exp z_tv,  loss_t = lse_t - z_t,target
//   g_tv = cap'(h_t . w_v) ((dloss_t + dlse_t) exp(z_tv - lse_t) - dloss_t [v = target])
//   dh = G W,  dW = G^T h
//
// Tokens that are left out are sorted out first: the others' rows are copied
// together (their number stays on the device), so that they cost nothing and
// whatever they hold reaches nothing.  The forward is one product whose epilogue
// keeps, for each token and 128 entries of the vocabulary, the largest logit and
// the sum of exponentials below it, and joins those.  The backward goes through the
// vocabulary in pieces: the logits of a piece again, turned into G in BF16 as they
// leave the tensor core, then G W added to dh in FP32 and G^T h, which is whole.
#include <algorithm>

#include "tb_lm_loss.cuh"
#include "tb_pair_product.cuh"

#ifndef TBG
#define TBG 16
#endif
namespace tb {
namespace loss {
namespace {

using namespace tb::pair;
using bf16 = __nv_bfloat16;

__device__ int g_loss_error;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
    long long n;
    int d, vocab;
    const bf16* h;
    long long ldh;
    const bf16* w;
    long long ldw;
    const int64_t* target;
    float cap;
    float* loss;
    float* lse;
    const float* dloss;
    const float* dlse;
    bf16* dh;
    long long lddh;
    bf16* dw;
    long long lddw;
};

// What is known of a kept token.  The backward's factors are relative to a unit that
// all tokens share, the largest |dloss|, which dh and dW are multiplied by in FP32:
// where all tokens count the same, the target's -1 is then exact in BF16.  (Tokens of
// 1/1536 each: 2-norm of dW's error 2.6e-3 without a unit, UNIT_ERR with it, 1.7e-3 of
// that the rounding of dW itself.)
struct __align__(16) Row {
    float lse2;   // lse in powers of two
    float both;   // dloss + dlse
    float dloss;
    int target;   // -1 behind the last token
};

// Of a number of tokens: how many are kept, their largest finite |dloss| and |dlse|.
struct Tally {
    int kept;
    float dloss, dlse;
};

struct Scratch {
    long long rows;   // n in whole tiles
    long long ld;     // of h's copy
    int* count;       // kept tokens
    float* unit;
    Tally* tallies;   // [ceil(n / kScan)], or NULL
    long long* token; // [rows] the kept tokens, in order
    Row* row;         // [rows]
    bf16* h;          // [rows][ld]; zeros from the last token to the end of its tile
    float* top;       // [rows] the target's logit
    float2* stats;    // [2 tiles of the vocabulary][rows]
    bf16* g;          // [rows][piece]
    float* part;      // [splits][rows][ldp] dh in FP32
    long long ldp;
};

constexpr int kScan = 4096;    // targets that are counted ahead in one piece
constexpr int kGather = 8;     // tokens of a gathering block, one a warp

__device__ __forceinline__ bool kept(const Args& a, long long t) {
    const int64_t y = __ldg(a.target + t);
    return y >= 0 && y < a.vocab;
}
__device__ __forceinline__ float finite_size(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.0f; }
template <bool BACKWARD>
__device__ __forceinline__ void add_token(const Args& a, long long t, Tally& v) {
    if (!kept(a, t)) return;
    ++v.kept;
    if (BACKWARD) {
        v.dloss = fmaxf(v.dloss, finite_size(__ldg(a.dloss + t)));
        if (a.dlse) v.dlse = fmaxf(v.dlse, finite_size(__ldg(a.dlse + t)));
    }
}
__device__ __forceinline__ void add_tally(Tally& v, const Tally& x) {
    v.kept += x.kept;
    v.dloss = fmaxf(v.dloss, x.dloss);
    v.dlse = fmaxf(v.dlse, x.dlse);
}
// Of 256 threads, for all of them.
__device__ __forceinline__ Tally block_tally(Tally v, Tally* shared) {
    v.kept = __reduce_add_sync(~0u, v.kept);  // (magnitudes compare as integers)
    v.dloss = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(v.dloss)));
    v.dlse = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(v.dlse)));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    Tally s{0, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; ++i) add_tally(s, shared[i]);
    return s;
}
template <bool BACKWARD>
__global__ void __launch_bounds__(256) tally_kernel(const Args a, Tally* tallies) {
    __shared__ Tally shared[8];
    const long long t0 = static_cast<long long>(blockIdx.x) * kScan;
    Tally v{0, 0.0f, 0.0f};
    for (int i = threadIdx.x; i < kScan; i += 256)
        if (t0 + i < a.n) add_token<BACKWARD>(a, t0 + i, v);
    v = block_tally(v, shared);
    if (threadIdx.x == 0) tallies[blockIdx.x] = v;
}
// Copies the kept tokens' rows together and zeros behind them up to the end of a tile;
// results of tokens left out are zeros.
template <bool BACKWARD>
__global__ void __launch_bounds__(256) gather_kernel(const Args a, const Scratch s) {
    __shared__ Tally shared[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long t0 = static_cast<long long>(blockIdx.x) * kGather;
    Tally before{0, 0.0f, 0.0f}, all{0, 0.0f, 0.0f};
    if (s.tallies) {
        const int blocks = static_cast<int>((a.n + kScan - 1) / kScan), own = static_cast<int>(t0 / kScan);
        for (int i = threadIdx.x; i < blocks; i += 256) {
            const Tally x = s.tallies[i];
            add_tally(all, x);
            if (i < own) add_tally(before, x);
        }
        for (long long t = static_cast<long long>(own) * kScan + threadIdx.x; t < t0; t += 256) add_token<false>(a, t, before);
    } else {
        for (long long t = threadIdx.x; t < a.n; t += 256) {
            add_token<BACKWARD>(a, t, all);
            if (t < t0) add_token<false>(a, t, before);
        }
    }
    before = block_tally(before, shared);
    all = block_tally(all, shared);
    const float unit = all.dloss > 0.0f ? all.dloss : all.dlse;
    const bool usual = unit > 1e-30f && unit < 1e30f;  // (whose reciprocal exists)
    const float inverse = usual ? 1.0f / unit : 1.0f;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *s.count = all.kept;
        *s.unit = usual ? unit : 1.0f;
    }
    const long long t = t0 + warp;
    const bool mine = t < a.n && kept(a, t);
    if (t < a.n) {
        const int units = (a.d + 7) / 8;
        if (mine) {
            long long to = before.kept;
            for (int i = 0; i < warp; ++i) to += kept(a, t0 + i);
            const uint4* from = reinterpret_cast<const uint4*>(a.h + t * a.ldh);
            uint4* dst = reinterpret_cast<uint4*>(s.h + to * s.ld);
#pragma unroll 8
            for (int i = lane; i < units; i += 32) dst[i] = __ldg(from + i);
            if (lane == 0) {
                s.token[to] = t;
                Row r{0.0f, 0.0f, 0.0f, static_cast<int>(a.target[t])};
                if (BACKWARD) {
                    r.lse2 = a.lse[t] * kLog2e;
                    const float dl = a.dloss[t];
                    r.dloss = dl == unit ? 1.0f : dl * inverse;
                    r.both = a.dlse ? fmaf(a.dlse[t], inverse, r.dloss) : r.dloss;
                }
                s.row[to] = r;
            }
        } else if (BACKWARD) {
            if (a.dh)
                for (int i = lane; i < a.d; i += 32) a.dh[t * a.lddh + i] = __float2bfloat16_rn(0.0f);
        } else if (lane == 0) {
            a.loss[t] = 0.0f;
            a.lse[t] = 0.0f;
        }
    }
    // rows behind the last token, each warp's share
    const long long end = (all.kept + 255) / 256 * 256;
    for (long long r = all.kept + t0 + warp; r < end; r += static_cast<long long>(gridDim.x) * kGather) {
        uint4* dst = reinterpret_cast<uint4*>(s.h + r * s.ld);
        for (int i = lane; i < s.ld / 8; i += 32) dst[i] = make_uint4(0, 0, 0, 0);
        if (lane == 0) s.row[r] = Row{0.0f, 0.0f, 0.0f, -1};
    }
}

struct Params {
    const int* count;
    const float* unit;
    int tiles_n;
    int cols;          // columns of the product that exist
    int k;             // K of the product (dW: counted on the device)
    int col0;          // first entry of the vocabulary of this piece
    int splits;        // dh
    int first;         // dh: the piece is the first
    float cap;
    long long rows;
    const Row* row;
    float* top;
    float2* stats;
    void* out;
    long long ldo;
    int out_rows;      // dW: rows that exist
    int out_tma;
};
__device__ __forceinline__ int kept_tiles(const Params& p) { return (*p.count + 255) / 256; }

// Sums of 512 terms in the tensor core: a logit is off by 2.6e-7 of its terms' magnitude at most.
struct Logits {
    static constexpr bool kAMn = false, kBMn = false, kF16 = false;
    static constexpr int kParts = 1, kGroup = TBG;
    using Params = loss::Params;
    static __device__ __forceinline__ int* error() { return &g_loss_error; }
    static __device__ __forceinline__ int items(const Params& p) { return kept_tiles(p) * p.tiles_n; }
    static __device__ __forceinline__ Work work(const Params& p, int item) {
        Work w{0, 0, 0, (p.k + 63) / 64, 0, -1};
        band_tile(item, kept_tiles(p), p.tiles_n, w.tm, w.tn);
        return w;
    }
    static __device__ __forceinline__ void finish(const Launch<Logits>& L, const Work& w, float (&acc)[128], uint8_t*, int row_in, int half, int lane) {
        const Params& p = L.p;
        const long long row = w.tm * 256ll + row_in + lane;
        const int col = w.tn * 256 + half * 128, cols = p.cols - col;
        if (p.cap > 0.0f) {
            const float inverse = 1.0f / p.cap;
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = p.cap * tanhf(acc[i] * inverse);
        }
        if (cols < 128) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
                if (i >= cols) acc[i] = -INFINITY;
        }
        float m = acc[0];
#pragma unroll
        for (int i = 1; i < 128; ++i) m = fmaxf(m, acc[i]);
        const float base = m == -INFINITY ? 0.0f : m * kLog2e;
        float s[4] = {};
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i & 3] += exp2f(fmaf(acc[i], kLog2e, -base));
        p.stats[(2 * w.tn + half) * p.rows + row] = make_float2(m, (s[0] + s[1]) + (s[2] + s[3]));
        const int at = p.row[row].target - col;
        if (at >= 0 && at < 128) {
            float z = 0.0f;
#pragma unroll
            for (int i = 0; i < 128; ++i) z = i == at ? acc[i] : z;
            p.top[row] = z;
        }
    }
};

// The same product, turned into G.  G enters its products as BF16, as every operand does: an error of
// 2^-8 of each of its values at most, which are summed with signs that do not depend on the errors'.
struct Gradient {
    static constexpr bool kAMn = false, kBMn = false, kF16 = false;
    static constexpr int kParts = 1, kGroup = 1 << 30;
    using Params = loss::Params;
    static __device__ __forceinline__ int* error() { return &g_loss_error; }
    static __device__ __forceinline__ int items(const Params& p) { return kept_tiles(p) * p.tiles_n; }
    static __device__ __forceinline__ Work work(const Params& p, int item) { return Logits::work(p, item); }
    static __device__ __forceinline__ void finish(const Launch<Gradient>& L, const Work& w, float (&acc)[128], uint8_t* buf, int row_in, int half, int lane) {
        const Params& p = L.p;
        const int row0 = w.tm * 256 + row_in, col = w.tn * 256 + half * 128;
        const Row r = p.row[row0 + lane];
        const int at = r.target - p.col0 - col;
        const bool hit = at >= 0 && at < 128;
        const float inverse = 1.0f / p.cap;
#pragma unroll
        for (int i = 0; i < 128; ++i) {
            float z = acc[i], slope = 1.0f;
            if (p.cap > 0.0f) {
                const float t = tanhf(z * inverse);
                z = p.cap * t;
                slope = fmaf(-t, t, 1.0f);
            }
            float g = r.both * exp2f(fmaf(z, kLog2e, -r.lse2));
            if (hit && i == at) g -= r.dloss;
            acc[i] = p.cap > 0.0f ? g * slope : g;
        }
        store_tma<true, 1>(&L.o[0][0], buf, acc, col, row0, 0, static_cast<int>(p.ldo), false, lane);
    }
};

// A piece's part of dh, added in FP32.
struct InputGrad {
    static constexpr bool kAMn = false, kBMn = true, kF16 = false;
    static constexpr int kParts = 1, kGroup = 1 << 30;
    using Params = loss::Params;
    static __device__ __forceinline__ int* error() { return &g_loss_error; }
    static __device__ __forceinline__ int items(const Params& p) { return kept_tiles(p) * p.tiles_n * p.splits; }
    static __device__ __forceinline__ Work work(const Params& p, int item) {
        const int all = (p.k + 63) / 64, q = item % p.splits;
        Work w{0, 0, share_at(all, q, p.splits), 0, 0, q};
        w.slices = share_at(all, q + 1, p.splits) - w.k0;
        band_tile(item / p.splits, kept_tiles(p), p.tiles_n, w.tm, w.tn);
        return w;
    }
    static __device__ __forceinline__ void finish(const Launch<InputGrad>& L, const Work& w, float (&acc)[128], uint8_t* buf, int row_in, int half, int lane) {
        const int row0 = w.tm * 256 + row_in, col = w.tn * 256 + half * 128;
        store_tma<false, 1>(&L.o[0][0], buf, acc, col, row0, w.slot, L.p.cols, !L.p.first, lane);
    }
};

// A piece's rows of dW, over all kept tokens.
struct WeightGrad {
    static constexpr bool kAMn = true, kBMn = true, kF16 = false;
    static constexpr int kParts = 1, kGroup = 1 << 30;
    using Params = loss::Params;
    static __device__ __forceinline__ int* error() { return &g_loss_error; }
    static __device__ __forceinline__ int items(const Params& p) { return (p.out_rows + 255) / 256 * p.tiles_n; }
    static __device__ __forceinline__ Work work(const Params& p, int item) {
        Work w{0, 0, 0, (*p.count + 63) / 64, 0, -1};
        band_tile(item, (p.out_rows + 255) / 256, p.tiles_n, w.tm, w.tn);
        return w;
    }
    static __device__ __forceinline__ void finish(const Launch<WeightGrad>& L, const Work& w, float (&acc)[128], uint8_t* buf, int row_in, int half, int lane) {
        const Params& p = L.p;
        const int row0 = w.tm * 256 + row_in, col = w.tn * 256 + half * 128;
        const int rows = min(32, p.out_rows - row0), cols = p.cols - col;
        if (rows <= 0 || cols <= 0) return;
        const float unit = *p.unit;
#pragma unroll
        for (int i = 0; i < 128; ++i) acc[i] *= unit;
        if (p.out_tma) store_tma<true, 1>(&L.o[0][0], buf, acc, col, row0, 0, p.cols, false, lane);
        else store_rows<true>(buf, acc, static_cast<bf16*>(p.out) + row0 * p.ldo + col, p.ldo, rows, cols, lane);
    }
};

// Joins a token's pieces of the vocabulary: eight tokens a block, 32 threads each.
__global__ void __launch_bounds__(256) join_loss_kernel(const Args a, const Scratch s, const int pieces) {
    __shared__ float2 shared[32][9];
    pdl_wait();
    const int count = *s.count, tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
    const long long r = static_cast<long long>(blockIdx.x) * 8 + tx;
    if (blockIdx.x * 8ll >= count) return;
    float m = -INFINITY, sum = 0.0f;
    auto add = [&](float2 x) {
        const float top = fmaxf(m, x.x), base = top == -INFINITY ? 0.0f : top;
        sum = sum * exp2f((m - base) * kLog2e) + x.y * exp2f((x.x - base) * kLog2e);
        m = top;
    };
    if (r < count) {
#pragma unroll 4
        for (int i = ty; i < pieces; i += 32) add(s.stats[i * s.rows + r]);
    }
    shared[ty][tx] = make_float2(m, sum);
    __syncthreads();
    if (ty == 0 && r < count) {
        m = -INFINITY;
        sum = 0.0f;
#pragma unroll 4
        for (int i = 0; i < 32; ++i) add(shared[i][tx]);
        const float rest = logf(sum);
        const long long t = s.token[r];
        a.lse[t] = m + rest;
        a.loss[t] = (m - s.top[r]) + rest;  // (the difference of like logits first: it is exact)
    }
}
// dh from its shares, in order: a row a warp.
__global__ void __launch_bounds__(256) join_dh_kernel(const Args a, const Scratch s, const int splits) {
    pdl_wait();
    const long long r = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (r >= *s.count) return;
    const int lane = threadIdx.x & 31;
    const float unit = *s.unit;
    const float* part = s.part + r * s.ldp;
    bf16* out = a.dh + s.token[r] * a.lddh;
    const bool wide = (reinterpret_cast<uintptr_t>(out) & 7) == 0;
    for (int i = 4 * lane; i < a.d; i += 128) {
        float4 v = *reinterpret_cast<const float4*>(part + i);
        for (int q = 1; q < splits; ++q) {
            const float4 x = *reinterpret_cast<const float4*>(part + q * s.rows * s.ldp + i);
            v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        v.x *= unit; v.y *= unit; v.z *= unit; v.w *= unit;
        if (wide && i + 4 <= a.d) {
            *reinterpret_cast<uint2*>(out + i) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
        } else {
            const float x[4] = {v.x, v.y, v.z, v.w};
            for (int e = 0; e < 4 && i + e < a.d; ++e) out[i + e] = __float2bfloat16_rn(x[e]);
        }
    }
}

long long up(long long v, long long m) { return (v + m - 1) / m * m; }

// The scratch that both directions need, `more` bytes behind it.
int make_scratch(const Args& a, size_t more, Scratch* s, void** base, char** rest, cudaStream_t st) {
    s->rows = up(a.n, 256);
    s->ld = up(a.d, 8);
    const long long blocks = (a.n + kScan - 1) / kScan;
    const size_t sizes[5] = {256, a.n > 2 * kScan ? sizeof(Tally) * static_cast<size_t>(blocks) : 0, sizeof(long long) * s->rows, sizeof(Row) * s->rows,
                             sizeof(bf16) * s->rows * s->ld};
    size_t all = more;
    for (size_t b : sizes) all += up(b, 256);
    const int rc = scratch_alloc(base, all, st);
    if (rc) return rc;
    char* p = static_cast<char*>(*base);
    auto take = [&](size_t b) { char* q = p; p += up(b, 256); return q; };
    s->count = reinterpret_cast<int*>(take(sizes[0]));
    s->unit = reinterpret_cast<float*>(s->count + 1);
    s->tallies = sizes[1] ? reinterpret_cast<Tally*>(take(sizes[1])) : nullptr;
    s->token = reinterpret_cast<long long*>(take(sizes[2]));
    s->row = reinterpret_cast<Row*>(take(sizes[3]));
    s->h = reinterpret_cast<bf16*>(take(sizes[4]));
    *rest = p;
    return TB_OK;
}
template <bool BACKWARD>
int gather(const Args& a, const Scratch& s, cudaStream_t st) {
    if (s.tallies) tally_kernel<BACKWARD><<<static_cast<unsigned>((a.n + kScan - 1) / kScan), 256, 0, st>>>(a, s.tallies);
    gather_kernel<BACKWARD><<<static_cast<unsigned>((a.n + kGather - 1) / kGather), 256, 0, st>>>(a, s);
    return check_launch("gather_kernel");
}
template <typename... P, typename... A>
int launch_small(const char* what, void (*kernel)(P...), long long blocks, cudaStream_t st, A&&... args) {
    const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, args...);
    return e == cudaSuccess ? check_launch(what) : cuda_fail(e, what);
}

int forward(const Args& a, cudaStream_t st) {
    const int tiles_m = tiles(a.n, 256), tiles_n = tiles(a.vocab, 256);
    if (static_cast<long long>(tiles_m) * tiles_n > 0x3FFFFFFFll) return fail(TB_ERR_CAPACITY, "tb_lm_loss: %lld tiles", static_cast<long long>(tiles_m) * tiles_n);
    Scratch s{};
    void* base = nullptr;
    char* rest = nullptr;
    const long long rows = up(a.n, 256);
    int rc = make_scratch(a, sizeof(float) * rows + sizeof(float2) * rows * 2 * tiles_n, &s, &base, &rest, st);
    if (rc) return rc;
    s.top = reinterpret_cast<float*>(rest);
    s.stats = reinterpret_cast<float2*>(s.top + rows);
    rc = gather<false>(a, s, st);
    pair::Launch<Logits> L{};
    L.p.count = s.count;
    L.p.tiles_n = tiles_n;
    L.p.cols = a.vocab;
    L.p.k = a.d;
    L.p.cap = a.cap;
    L.p.rows = rows;
    L.p.row = s.row;
    L.p.top = s.top;
    L.p.stats = s.stats;
    if (!rc) rc = operand_map(&L.a[0], s.h, rows, a.d, s.ld, false);
    if (!rc) rc = operand_map(&L.b[0][0], a.w, a.vocab, a.d, a.ldw, false);
    if (!rc) rc = launch_product(L, static_cast<long long>(tiles_m) * tiles_n, st);
    if (!rc) rc = launch_small("join_loss_kernel", join_loss_kernel, (a.n + 7) / 8, st, a, s, 2 * tiles_n);
    scratch_free(base, st);
    return rc;
}

constexpr long long kPieceG = 128ll << 20;  // bytes of G in one piece of the vocabulary

int backward(const Args& a, cudaStream_t st) {
    const int tiles_m = tiles(a.n, 256), tiles_d = tiles(a.d, 256);
    const long long rows = up(a.n, 256);
    const long long piece = std::min(up(a.vocab, 256), std::max(256ll, kPieceG / (2 * rows) / 256 * 256));
    if (tiles_m * (piece / 256) > 0x3FFFFFFFll || tiles_m * static_cast<long long>(tiles_d) * kPairs > 0x3FFFFFFFll || piece / 256 * tiles_d > 0x3FFFFFFFll)
        return fail(TB_ERR_CAPACITY, "tb_lm_loss_backward: %lld tokens of %d", a.n, a.d);
    // dh's tiles share out their K where they do not fill the GPU
    int splits = 1;
    while (2ll * splits * tiles_m * tiles_d <= kPairs && piece / 64 / (2 * splits) >= 4) splits *= 2;
    Scratch s{};
    void* base = nullptr;
    char* rest = nullptr;
    const long long ldp = up(a.d, 4);
    const size_t g_bytes = sizeof(bf16) * rows * piece, part_bytes = a.dh ? sizeof(float) * splits * rows * ldp : 0;
    int rc = make_scratch(a, g_bytes + part_bytes, &s, &base, &rest, st);
    if (rc) return rc;
    s.g = reinterpret_cast<bf16*>(rest);
    s.part = reinterpret_cast<float*>(rest + g_bytes);
    s.ldp = ldp;
    rc = gather<true>(a, s, st);
    for (long long v0 = 0; v0 < a.vocab && !rc; v0 += piece) {
        const int cols = static_cast<int>(std::min<long long>(piece, a.vocab - v0));
        const bf16* w = a.w + v0 * a.ldw;
        Params p{};
        p.count = s.count;
        p.unit = s.unit;
        p.cap = a.cap;
        p.rows = rows;
        p.row = s.row;
        {
            pair::Launch<Gradient> L{};
            L.p = p;
            L.p.tiles_n = tiles(cols, 256);
            L.p.cols = cols;
            L.p.k = a.d;
            L.p.col0 = static_cast<int>(v0);
            L.p.ldo = piece;
            rc = operand_map(&L.a[0], s.h, rows, a.d, s.ld, false);
            if (!rc) rc = operand_map(&L.b[0][0], w, cols, a.d, a.ldw, false);
            if (!rc) rc = make_out_map(&L.o[0][0], s.g, true, piece, rows, 1, piece, rows * piece);
            if (!rc) rc = launch_product(L, static_cast<long long>(tiles_m) * L.p.tiles_n, st);
        }
        if (!rc && a.dh) {
            pair::Launch<InputGrad> L{};
            L.p = p;
            L.p.tiles_n = tiles_d;
            L.p.cols = a.d;
            L.p.k = cols;
            L.p.splits = splits;
            L.p.first = v0 == 0;
            rc = operand_map(&L.a[0], s.g, rows, cols, piece, false);
            if (!rc) rc = operand_map(&L.b[0][0], w, cols, a.d, a.ldw, true);
            if (!rc) rc = make_out_map(&L.o[0][0], s.part, false, a.d, rows, splits, ldp, rows * ldp);
            if (!rc) rc = launch_product(L, static_cast<long long>(tiles_m) * tiles_d * splits, st);
        }
        if (!rc && a.dw) {
            pair::Launch<WeightGrad> L{};
            L.p = p;
            L.p.tiles_n = tiles_d;
            L.p.cols = a.d;
            L.p.out_rows = cols;
            L.p.out = a.dw + v0 * a.lddw;
            L.p.ldo = a.lddw;
            // (a TMA store writes whole 16 bytes of a row, whatever the row's length)
            L.p.out_tma = reinterpret_cast<uintptr_t>(a.dw) % 16 == 0 && a.lddw % 8 == 0 && a.d % 8 == 0;
            rc = operand_map(&L.a[0], s.g, rows, cols, piece, true);
            if (!rc) rc = operand_map(&L.b[0][0], s.h, rows, a.d, s.ld, true);
            if (!rc && L.p.out_tma) rc = make_out_map(&L.o[0][0], L.p.out, true, a.d, cols, 1, a.lddw, a.lddw * cols);
            if (!rc) rc = launch_product(L, static_cast<long long>(tiles(cols, 256)) * tiles_d, st);
        }
    }
    if (!rc && a.dh) rc = launch_small("join_dh_kernel", join_dh_kernel, (a.n + 7) / 8, st, a, s, splits);
    scratch_free(base, st);
    return rc;
}

bool bad_rows(const void* p, int64_t ld, int64_t cols) {
    return !p || reinterpret_cast<uintptr_t>(p) % 16 || ld < cols || ld % 8;
}
int check_args(const char* who, const tb_lm_loss_args* p, Args* a) {
    if (!p || p->struct_size != sizeof(tb_lm_loss_args)) return fail(TB_ERR_ARG, "%s: null args or bad struct_size", who);
    if (p->dtype != TB_BF16) return fail(TB_ERR_UNSUPPORTED, "%s: TB_BF16 only (dtype %d)", who, p->dtype);
    if (p->d <= 0 || p->vocab <= 0) return fail(TB_ERR_ZERO_SIZE, "%s: empty head", who);
    if (p->d > 0x7FFFFFFF - 256 || p->vocab > 0x7FFFFFFF - 256) return fail(TB_ERR_SHAPE, "%s: %d features, %d entries", who, p->d, p->vocab);
    if (p->n < 0 || p->n > 0x7FFFFFFFll - 65536) return fail(TB_ERR_SHAPE, "%s: %lld tokens", who, static_cast<long long>(p->n));
    if (!(p->softcap >= 0.0f && p->softcap < INFINITY)) return fail(TB_ERR_CONFIG, "%s: softcap %g", who, p->softcap);
    if (bad_rows(p->w, p->ldw, p->d)) return fail(TB_ERR_ARG, "%s: w must be 16-byte aligned, ldw >= d a multiple of 8", who);
    if (p->n > 0) {
        if (bad_rows(p->h, p->ldh, p->d)) return fail(TB_ERR_ARG, "%s: h must be 16-byte aligned, ldh >= d a multiple of 8", who);
        if (!p->target || !p->lse) return fail(TB_ERR_ARG, "%s: null target or lse", who);
    }
    a->n = p->n;
    a->d = p->d;
    a->vocab = p->vocab;
    a->h = static_cast<const bf16*>(p->h);
    a->ldh = p->ldh;
    a->w = static_cast<const bf16*>(p->w);
    a->ldw = p->ldw;
    a->target = p->target;
    a->cap = p->softcap;
    a->loss = p->loss;
    a->lse = p->lse;
    a->dloss = p->dloss;
    a->dlse = p->dlse;
    a->dh = static_cast<bf16*>(p->dh);
    a->lddh = p->lddh;
    a->dw = static_cast<bf16*>(p->dw);
    a->lddw = p->lddw;
    return TB_OK;
}

}  // namespace

int take_error(cudaStream_t st) {
    int h = 0, zero = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&h, g_loss_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_loss_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    return e == cudaSuccess ? h : -1;
}

}  // namespace loss
}  // namespace tb

using namespace tb;

extern "C" int tb_lm_loss(const tb_lm_loss_args* p, void* stream) {
    loss::Args a{};
    int rc = loss::check_args("tb_lm_loss", p, &a);
    if (rc) return rc;
    if (a.n == 0) return TB_OK;
    if (!a.loss) return fail(TB_ERR_ARG, "tb_lm_loss: null loss");
    if ((rc = require_device(nullptr))) return rc;
    return loss::forward(a, static_cast<cudaStream_t>(stream));
}

extern "C" int tb_lm_loss_backward(const tb_lm_loss_args* p, void* stream) {
    loss::Args a{};
    int rc = loss::check_args("tb_lm_loss_backward", p, &a);
    if (rc) return rc;
    if (a.n > 0 && !a.dloss) return fail(TB_ERR_ARG, "tb_lm_loss_backward: null dloss");
    if (a.dh && a.lddh < a.d) return fail(TB_ERR_ARG, "tb_lm_loss_backward: lddh < d");
    if (a.dw && a.lddw < a.d) return fail(TB_ERR_ARG, "tb_lm_loss_backward: lddw < d");
    if ((!a.dh || a.n == 0) && !a.dw) return TB_OK;
    if ((rc = require_device(nullptr))) return rc;
    auto st = static_cast<cudaStream_t>(stream);
    if (a.n == 0) {
        const cudaError_t e = cudaMemset2DAsync(a.dw, sizeof(loss::bf16) * a.lddw, 0, sizeof(loss::bf16) * a.d, a.vocab, st);
        return e == cudaSuccess ? TB_OK : cuda_fail(e, "tb_lm_loss_backward: zeros");
    }
    return loss::backward(a, st);
}
