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
#include "tb_split_product.cuh"

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
// 1/1536 each: 2-norm of dW's error 2.6e-3 without a unit, 1.9e-3 with it, 1.7e-3 of
// that the rounding of dW itself.)
struct __align__(16) Row {
    float lse;
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
    int* failed;      // 1 once a wait has expired in one of the call's products
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

constexpr int kScan = 1024;    // targets that are counted ahead in one piece, from two such pieces on (8000 tokens of 100 features: every block counting all 27 us, so 14)
constexpr int kFewGather = 512; // up to so many tokens, a gathering block has one, of which each warp copies a part; else eight, one a warp

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
template <bool BACKWARD, bool ONE>
__global__ void __launch_bounds__(256) gather_kernel(const Args a, const Scratch s) {
    __shared__ Tally shared[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long t0 = static_cast<long long>(blockIdx.x) * (ONE ? 1 : 8);
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
    const float most = all.dloss > 1e-15f * all.dlse ? all.dloss : all.dlse;  // (with dlse far above dloss, that)
    const float unit = most > 1e-30f && most < 1e30f ? most : 1.0f, inverse = 1.0f / unit;  // (a reciprocal that exists)
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        *s.count = all.kept;
        *s.unit = unit;
        *s.failed = 0;
    }
    const long long t = t0 + (ONE ? 0 : warp);
    const int part = ONE ? threadIdx.x : lane;  // of a row's units
    constexpr int kParts = ONE ? 256 : 32;
    const bool mine = t < a.n && kept(a, t);
    if (t < a.n) {
        const int units = (a.d + 7) / 8;
        if (mine) {
            long long to = before.kept;
            for (int i = 0; !ONE && i < warp; ++i) to += kept(a, t0 + i);
            const uint4* from = reinterpret_cast<const uint4*>(a.h + t * a.ldh);
            uint4* dst = reinterpret_cast<uint4*>(s.h + to * s.ld);
#pragma unroll 8
            for (int i = part; i < units; i += kParts) dst[i] = __ldg(from + i);
            if (part == 0) {
                s.token[to] = t;
                Row r{0.0f, 0.0f, 0.0f, static_cast<int>(a.target[t])};
                if (BACKWARD) {
                    r.lse = a.lse[t];
                    const float dl = a.dloss[t];
                    auto scaled = [&](float x) { return x == unit ? 1.0f : x * inverse; };
                    r.dloss = scaled(dl);
                    r.both = a.dlse ? scaled(dl + a.dlse[t]) : r.dloss;  // (the sum first: it is exact where the two nearly cancel)
                }
                s.row[to] = r;
            }
        } else if (BACKWARD) {
            if (a.dh)
                for (int i = part; i < a.d; i += kParts) a.dh[t * a.lddh + i] = __float2bfloat16_rn(0.0f);
        } else if (part == 0) {
            a.loss[t] = 0.0f;
            a.lse[t] = 0.0f;
        }
    }
    // rows behind the last token, each warp's share
    const long long end = (all.kept + 255) / 256 * 256;
    for (long long r = all.kept + blockIdx.x * 8ll + warp; r < end; r += gridDim.x * 8ll) {
        uint4* dst = reinterpret_cast<uint4*>(s.h + r * s.ld);
        for (int i = lane; i < s.ld / 8; i += 32) dst[i] = make_uint4(0, 0, 0, 0);
        if (lane == 0) s.row[r] = Row{0.0f, 0.0f, 0.0f, -1};
    }
}

// tanh of each of v / c, in place: an odd polynomial of degree 9 up to 1/2 (2.6e-8 of the value, 8.4e-8 as FP32 evaluates it;
// fitted at Chebyshev points in 64 bits) where all of the warp's values lie there, which takes a quarter of tanhf's time.  Where
// some do not, looking costs its share.  (Loss of 8000 tokens, 512 features, 32000 entries: small logits 273 us, 373 by tanhf
// alone; logits of the cap's order 449 and 390.  2048 tokens, 4096 features, behind whose products most of it hides: 363 and 385; 487 and 493.)
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
// 1 / c within FP32: a logit of zero stays zero under the smallest cap too.
__device__ __forceinline__ float inverse_cap(float cap) { return fminf(1.0f / cap, 3.4028235e38f); }
template <int N>
__device__ __forceinline__ void tanh_of(float* v, float inverse) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] *= inverse;
        most = fmaxf(most, fabsf(v[i]));
        if (!(v[i] == v[i])) most = INFINITY;
    }
    if (__any_sync(~0u, most > 0.5f)) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = tanhf(v[i]);
        return;
    }
    const uint64_t c1 = pack2(-0.3333307206630707f, -0.3333307206630707f), c2 = pack2(0.13324828445911407f, 0.13324828445911407f);
    const uint64_t c3 = pack2(-0.05298924073576927f, -0.05298924073576927f), c4 = pack2(0.017141319811344147f, 0.017141319811344147f), zero = pack2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const uint64_t x = pack2(v[i], v[i + 1]), y = fma2(x, x, zero);
        const uint64_t t = fma2(fma2(fma2(fma2(fma2(c4, y, c3), y, c2), y, c1), y, zero), x, x);  // x + x (c1 y + ...)
        asm("mov.b64 {%0, %1}, %2;" : "=f"(v[i]), "=f"(v[i + 1]) : "l"(t));
    }
}

// exp(v - from) for `v` in place.  The difference first: it is exact where the two are alike, so that a maximum's exponential
// is 1, where the difference of rounded products with log2(e) is off by up to |from| 2^-24.
template <int N>
__device__ __forceinline__ void exp_below(float (&v)[N], float from) {
    const uint64_t one = pack2(1.0f, 1.0f), minus = pack2(-from, -from), log2e = pack2(kLog2e, kLog2e), zero = pack2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const uint64_t x = fma2(fma2(pack2(v[i], v[i + 1]), one, minus), log2e, zero);
        asm("mov.b64 {%0, %1}, %2;" : "=f"(v[i]), "=f"(v[i + 1]) : "l"(x));
        v[i] = exp2f(v[i]);
        v[i + 1] = exp2f(v[i + 1]);
    }
}

struct Params {
    const int* count;
    const float* unit;
    int* failed;
    int tiles_n;
    int cols;          // columns of the product that exist
    int k;             // K of the product (dW: counted on the device)
    int col0;          // first entry of the vocabulary of this piece
    int splits;        // shares of K of dh's tiles, and of dW's
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

// Sums of 1024 terms in the tensor core.  (2048 tokens, 4096 features, 2-norm of the loss's error: 1.6e-7 with
// sums of 256, 3.1e-7 of 512, 6.5e-7 of 1024, which is what FP32 products have too, 3.1e-6 with one of all; tiles
// of 35200 cycles with 1024, 34200 with one, of which the products need 32768.)
struct Logits {
    static constexpr bool kAMn = false, kBMn = false, kF16 = false;
    static constexpr int kParts = 1, kGroup = 16;
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
            const float inverse = inverse_cap(p.cap);
#pragma unroll
            for (int c = 0; c < 128; c += 32) tanh_of<32>(acc + c, inverse);
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] *= p.cap;
        }
        if (cols < 128) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
                if (i >= cols) acc[i] = -INFINITY;
        }
        float m = acc[0];
#pragma unroll
        for (int i = 1; i < 128; ++i) m = fmaxf(m, acc[i]);
        const int at = p.row[row].target - col;
        if (at >= 0 && at < 128) {
            float z = 0.0f;
#pragma unroll
            for (int i = 0; i < 128; ++i) z = i == at ? acc[i] : z;
            p.top[row] = z;
        }
        exp_below(acc, m == -INFINITY ? 0.0f : m);
        float s[4] = {};
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i & 3] += acc[i];
        p.stats[(2 * w.tn + half) * p.rows + row] = make_float2(m, (s[0] + s[1]) + (s[2] + s[3]));
    }
};

// The same product in the same sums, so that its logits are the forward's to the last bit, turned into G.  What the tensor
// core cuts off has one sign where the terms have: logits that are low beside lse make every p low, and p - 1 of a
// token that is nearly certain a multiple of what it is.  (8192 terms of one sign in one sum, a logit of 60: p low by 6e-4,
// where p - 1 may be 1e-4.)  G enters its products as BF16, as every operand does: an error of
// 2^-8 of each of its values at most, which are summed with signs that do not depend on the errors'.
struct Gradient {
    static constexpr bool kAMn = false, kBMn = false, kF16 = false;
    static constexpr int kParts = 1, kGroup = Logits::kGroup;
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
        if (p.cap > 0.0f) {
            const float inverse = inverse_cap(p.cap);
#pragma unroll
            for (int c = 0; c < 128; c += 32) {
                tanh_of<32>(acc + c, inverse);
                float e[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) e[i] = p.cap * acc[c + i];
                exp_below(e, r.lse);
#pragma unroll
                for (int i = c; i < c + 32; ++i) {
                    const float t = acc[i];
                    float g = r.both * e[i - c];
                    if (hit && i == at) g -= r.dloss;
                    acc[i] = g * fmaf(-t, t, 1.0f);
                }
            }
        } else {
            exp_below(acc, r.lse);
#pragma unroll
            for (int i = 0; i < 128; ++i) {
                const float g = r.both * acc[i];
                acc[i] = hit && i == at ? g - r.dloss : g;
            }
        }
        store_tma<true, 1>(&L.o[0][0], buf, acc, col, row0, 0, static_cast<int>(p.ldo), false, lane);
    }
};

// A piece's part of dh, in sums of 4096 entries, added in FP32.
struct InputGrad {
    static constexpr bool kAMn = false, kBMn = true, kF16 = false;
    static constexpr int kParts = 1, kGroup = 64;
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
        if (row0 >= *L.p.count) return;
        store_tma<false, 1>(&L.o[0][0], buf, acc, col, row0, w.slot, L.p.cols, !L.p.first, lane);
    }
};

// A piece's rows of dW, over all kept tokens, in sums of 4096 of them (each of whose 256 steps cuts off up to 2^-23).
struct WeightGrad {
    static constexpr bool kAMn = true, kBMn = true, kF16 = false;
    static constexpr int kParts = 1, kGroup = 64;
    using Params = loss::Params;
    static __device__ __forceinline__ int* error() { return &g_loss_error; }
    static __device__ __forceinline__ int items(const Params& p) { return (p.out_rows + 255) / 256 * p.tiles_n * p.splits; }
    static __device__ __forceinline__ Work work(const Params& p, int item) {
        const int all = (*p.count + 63) / 64, q = item % p.splits;
        Work w{0, 0, share_at(all, q, p.splits), 0, 0, q};
        w.slices = share_at(all, q + 1, p.splits) - w.k0;
        band_tile(item / p.splits, (p.out_rows + 255) / 256, p.tiles_n, w.tm, w.tn);
        return w;
    }
    static __device__ __forceinline__ void finish(const Launch<WeightGrad>& L, const Work& w, float (&acc)[128], uint8_t* buf, int row_in, int half, int lane) {
        const Params& p = L.p;
        const int row0 = w.tm * 256 + row_in, col = w.tn * 256 + half * 128;
        const int rows = min(32, p.out_rows - row0), cols = p.cols - col;
        if (rows <= 0 || cols <= 0) return;
        if (p.splits > 1) {
            store_tma<false, 1>(&L.o[0][0], buf, acc, col, row0, w.slot, p.cols, false, lane);
            return;
        }
        const float unit = *p.unit;
        if (*p.failed) return;
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
    const int count = *s.count, failed = *s.failed, tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
    const long long r = static_cast<long long>(blockIdx.x) * 8 + tx;
    if (blockIdx.x * 8ll >= count || failed) return;
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
        a.loss[t] = (m - s.top[r]) + rest;  // (the difference of like logits first: it is exact; neither is below zero, as the maximum's exponential is 1)
    }
}
// dh from its shares, in order: 1024 columns of a row a block.
__global__ void __launch_bounds__(256) join_dh_kernel(const Args a, const Scratch s, const int splits) {
    pdl_wait();
    const int chunks = (a.d + 1023) / 1024;
    const long long r = blockIdx.x / chunks;
    const int i = static_cast<int>(blockIdx.x % chunks) * 1024 + 4 * threadIdx.x;
    if (r >= *s.count || i >= a.d || *s.failed) return;
    const float unit = *s.unit;
    const float* part = s.part + r * s.ldp + i;
    float4 v = *reinterpret_cast<const float4*>(part);
#pragma unroll 4
    for (int q = 1; q < splits; ++q) {
        const float4 x = *reinterpret_cast<const float4*>(part + q * s.rows * s.ldp);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    }
    v.x *= unit; v.y *= unit; v.z *= unit; v.w *= unit;
    bf16* out = a.dh + s.token[r] * a.lddh + i;
    if ((reinterpret_cast<uintptr_t>(out) & 7) == 0 && i + 4 <= a.d) {
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    } else {
        const float x[4] = {v.x, v.y, v.z, v.w};
        for (int e = 0; e < 4 && i + e < a.d; ++e) out[e] = __float2bfloat16_rn(x[e]);
    }
}

// A piece's dW from its shares, in order: 1024 columns of a row a block.
__global__ void __launch_bounds__(256) join_dw_kernel(const float* part, const long long ldp, const int rows, const int d, const int splits, const Scratch s, bf16* out,
                                                      const long long ldo) {
    pdl_wait();
    const int chunks = (d + 1023) / 1024, r = blockIdx.x / chunks, i = static_cast<int>(blockIdx.x % chunks) * 1024 + 4 * threadIdx.x;
    if (i >= d || *s.failed) return;
    const float unit = *s.unit;
    float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int q = 0; q < splits; ++q) {
        const float4 x = *reinterpret_cast<const float4*>(part + (static_cast<long long>(q) * rows + r) * ldp + i);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    }
    const float f[4] = {v.x * unit, v.y * unit, v.z * unit, v.w * unit};
    for (int e = 0; e < 4 && i + e < d; ++e) out[r * ldo + i + e] = __float2bfloat16_rn(f[e]);
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
    s->failed = s->count + 2;
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
    if (a.n <= kFewGather) gather_kernel<BACKWARD, true><<<static_cast<unsigned>(a.n), 256, 0, st>>>(a, s);
    else gather_kernel<BACKWARD, false><<<static_cast<unsigned>((a.n + 7) / 8), 256, 0, st>>>(a, s);
    return check_launch("gather_kernel");
}
template <typename... P, typename... A>
int launch_small(const char* what, void (*kernel)(P...), long long blocks, cudaStream_t st, A&&... args) {
    const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, args...);
    return e == cudaSuccess ? check_launch(what) : cuda_fail(e, what);
}

// ---- few tokens: one pass over w --------------------------------------------------------
// Up to 128 tokens leave the logits bound by the reading of w.  Tokens are the N of the
// product here and the vocabulary is M: a CTA takes `tile` rows of w (up to 256, two MMAs of 128), a
// share that is even over all SMs, and streams them past the tokens' slices; a thread has one entry of the
// vocabulary and all tokens.  Sums of 64 terms in the tensor core, which costs nothing here, added in one order in both
// directions: p is of the difference of the backward's logits and the forward's lse.  (The backward from the last features on, which
// L2 still has, is 3 % sooner for 37 tokens, 4096 x 32000, with gradients, but adds in another order: 3e-5 of a logit of 60.)
// (32000 x 4096, whole calls: 53 us for 1 token, 54 for 37, 64 for 128, by tiles of 256 tokens 70; w at the measured
// copy rate 41.  128000 x 4096, 8 tokens: 167, at that rate 162.)
constexpr int kFewMost = 128;
constexpr int kFewThreads = 320;  // warps 0-7 results, 8 loads, 9 MMAs
constexpr int kFewCtas = 148;     // at most
constexpr int kFewGroup = 1;
template <int NT>
struct FewCfg {
    static constexpr int kStage = 32768 + NT * 128;
    static constexpr int kStages = NT <= 32 ? 6 : NT <= 64 ? 5 : 4;
    static constexpr int kExtra = 8 * NT * 8 + NT * 16;  // the warps' maxima and sums; the tokens' rows
    static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStage + kExtra + 1024 + 256;
    static_assert(kSmem <= 232448, "shared memory of a block");
};
struct FewParams {
    int tile, tiles, vocab, d;
    int col0;          // first entry of the vocabulary; `vocab` counts from it
    int n;             // forward: tokens as they are
    const int* count;  // backward: those kept
    const int64_t* target;
    const Row* row;
    float cap;
    float* top;        // [NT]
    float2* stats;     // [tiles][NT]
    bf16* g;           // [NT][ldg]
    long long ldg;
    int* failed;       // forward: a word a CTA; backward: the call's
};
struct FewMaps {
    CUtensorMap w, h;
};
// N columns (16 or 32) over a warp's 32 rows: column `lane` % N of this lane in the end.  Each step halves
// the columns that a lane has (37 tokens' forward, 64 columns: 64 us with five exchanges a column, 55 so).
template <int N, class F>
__device__ __forceinline__ float reduce_columns(float (&v)[N], int lane, F&& f) {
    if constexpr (N == 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = f(v[i], __shfl_xor_sync(~0u, v[i], 16));
    }
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const float keep = upper ? v[i + o] : v[i], send = upper ? v[i] : v[i + o];
            v[i] = f(keep, __shfl_xor_sync(~0u, send, o));
        }
    }
    return v[0];
}

template <int NT, bool GRAD>
__global__ void __launch_bounds__(kFewThreads, 1) few_logits_kernel(const __grid_constant__ FewMaps maps, const __grid_constant__ FewParams p) {
    using C = FewCfg<NT>;
    constexpr int kStages = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    float2* joined = reinterpret_cast<float2*>(smem + kStages * C::kStage);  // [8][NT]
    Row* rows = reinterpret_cast<Row*>(joined + 8 * NT);
    uint64_t* ready = reinterpret_cast<uint64_t*>(rows + NT);
    uint64_t* empty = ready + kStages;
    uint64_t* accfull = empty + kStages;  // [2]
    uint64_t* accempty = accfull + 2;     // [2]
    uint64_t* drained = accempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr uint32_t kColumns = NT <= 16 ? 64 : NT <= 32 ? 128 : NT <= 64 ? 256 : 512;  // two sums of two halves

    if (threadIdx.x == 8 * 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.w)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.h)) : "memory");
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&ready[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&accfull[b]), 1);
            mbar_init(smem_u32(&accempty[b]), 8);
        }
        mbar_init(smem_u32(drained), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kColumns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    pdl_wait();  // nothing above touched memory that an earlier kernel writes
    if (threadIdx.x < NT) {
        const int t = threadIdx.x;
        Row r{0.0f, 0.0f, 0.0f, -1};
        if (GRAD) {
            if (t < *p.count) r = p.row[t];
        } else if (t < p.n) {
            const int64_t y = p.target[t];
            if (y >= 0 && y < p.vocab) r.target = static_cast<int>(y);  // (all of the vocabulary, from 0)
        }
        rows[t] = r;
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    const int slices = (p.d + 63) / 64, kept = GRAD ? *p.count : 0;

    if (warp < 8) {
        const int quad = warp & 3, half = warp >> 2;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(half * NT);
        Ring<2> ac;
        bool ok = true;
        for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
            float z[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) z[i] = 0.0f;
            for (int left = slices; left > 0; left -= kFewGroup) {
                if (!wait(smem_u32(&accfull[ac.s]), ac.phase, abort_flag)) { ok = false; break; }
                fence_after();
#pragma unroll
                for (int c = 0; c < NT / 16; ++c) {
                    uint32_t x[16];
                    tmem_ld16(lane_base + static_cast<uint32_t>(ac.s * 2 * NT + 16 * c), x);
                    tmem_wait16(x);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) add2(z[16 * c + i], z[16 * c + i + 1], x[i], x[i + 1]);
                }
                fence_before();
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&accempty[ac.s])) : "memory");
                ac.next();
            }
            if (!ok) break;
            const int in = half * 128 + quad * 32 + lane;
            const long long entry = static_cast<long long>(tile) * p.tile + in;
            const bool inside = in < p.tile && entry < p.vocab;
            if (p.cap > 0.0f) {
                const float inverse = inverse_cap(p.cap);
#pragma unroll
                for (int i = 0; i < NT; ++i) z[i] = tanhf(z[i] * inverse);  // (not as what other tokens hold decides: some may be left out)
            }
            if constexpr (GRAD) {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const Row r = rows[i];
                    float x = z[i], slope = 1.0f;
                    if (p.cap > 0.0f) {
                        slope = fmaf(-x, x, 1.0f);
                        x *= p.cap;
                    }
                    float g = r.both * exp2f((x - r.lse) * kLog2e);
                    if (r.target - p.col0 == entry) g -= r.dloss;
                    // (a token behind the last kept one, of which z is what w times zeros gives, counts as zero)
                    if (inside) p.g[i * p.ldg + entry] = __float2bfloat16_rn(i < kept ? g * slope : 0.0f);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    if (p.cap > 0.0f) z[i] *= p.cap;
                    if (inside && rows[i].target == entry) p.top[i] = z[i];
                    if (!inside) z[i] = -INFINITY;
                }
                constexpr int N = NT % 32 ? 16 : 32;
                float2* mine = joined + warp * NT;
#pragma unroll
                for (int c = 0; c < NT; c += N) {
                    float v[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] = z[c + i];
                    const float most = reduce_columns(v, lane, [](float x, float y) { return fmaxf(x, y); });
                    if (lane < N) mine[c + lane].x = most;
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float m = mine[c + i].x;
                        v[i] = exp2f((z[c + i] - (m == -INFINITY ? 0.0f : m)) * kLog2e);
                    }
                    const float sum = reduce_columns(v, lane, [](float x, float y) { return x + y; });
                    if (lane < N) mine[c + lane].y = sum;
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x < NT) {
                    float m = -INFINITY, sum = 0.0f;
#pragma unroll
                    for (int q = 0; q < 8; ++q) m = fmaxf(m, joined[q * NT + threadIdx.x].x);
                    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const float2 x = joined[q * NT + threadIdx.x];
                        sum += x.y * exp2f((x.x - base) * kLog2e);
                    }
                    p.stats[static_cast<long long>(tile) * NT + threadIdx.x] = make_float2(m, sum);
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
        }
        if (!ok) {
            *abort_flag = 1;
            atomicExch(&g_loss_error, 1);
        }
    } else if (warp == 8) {
        if (lane == 0) {
            Ring<kStages> at;
            bool ok = true;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
#pragma unroll 1
                for (int i = 0; i < slices; ++i, at.next()) {
                    if (!wait(smem_u32(&empty[at.s]), at.phase ^ 1, abort_flag)) { ok = false; break; }  // (the first round passes at once)
                    const uint32_t stage = smem_u32(smem + at.s * C::kStage), bar = smem_u32(&ready[at.s]);
                    mbar_expect_tx(bar, static_cast<uint32_t>(p.tile) * 128 + NT * 128);
                    tma_load_2d(stage, &maps.w, 64 * i, tile * p.tile, bar);
                    tma_load_2d(stage + 32768, &maps.h, 64 * i, 0, bar);
                }
            }
            if (!ok) {
                *abort_flag = 1;
                atomicExch(&g_loss_error, 1);
                for (int i = 0; i < kStages; ++i)  // loads in flight, within a limit
                    if (i < at.s || at.phase) wait(smem_u32(&ready[i]), i < at.s ? at.phase : at.phase ^ 1, nullptr);
            }
        }
        __syncwarp();
    } else {
        if (lane == 0) {
            constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(NT >> 3) << 17) | (8u << 24);
            Ring<kStages> at;
            Ring<2> ac;
            bool ok = true;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
                for (int left = slices; left > 0 && ok;) {
                    int n = min(left, kFewGroup);
                    left -= n;
                    if (!wait(smem_u32(&accempty[ac.s]), ac.phase ^ 1, abort_flag)) { ok = false; break; }
                    fence_after();
                    uint32_t more = 0;
#pragma unroll 1
                    for (; n > 0; --n, at.next()) {
                        if (!wait(smem_u32(&ready[at.s]), at.phase, abort_flag)) { ok = false; break; }
                        fence_after();
                        const uint64_t a = operand_desc(smem_u32(smem + at.s * C::kStage), false), b = a + (32768 >> 4);
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            mma_one16<false>(tmem + ac.s * 2 * NT, a + 2 * kk, b + 2 * kk, kIdesc, more);
                            if (p.tile > 128) mma_one16<false>(tmem + ac.s * 2 * NT + NT, a + (16384 >> 4) + 2 * kk, b + 2 * kk, kIdesc, more);
                            more = 1;
                        }
                        mma_commit(smem_u32(&empty[at.s]));
                    }
                    if (!ok) break;
                    mma_commit(smem_u32(&accfull[ac.s]));
                    ac.next();
                }
            }
            if (!ok) {
                *abort_flag = 1;
                atomicExch(&g_loss_error, 1);
            }
            if (*abort_flag) drain_one(smem_u32(drained));
        }
        __syncwarp();
    }
    fence_before();
    __syncthreads();
    if (threadIdx.x == 0) {
        if (!GRAD) p.failed[blockIdx.x] = *abort_flag;
        else if (*abort_flag) atomicExch(p.failed, 1);
    }
    __syncwarp();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns));
    }
}
// A token a block: its tiles' maxima and sums.
__global__ void __launch_bounds__(256) join_few_kernel(const Args a, const float* top, const float2* stats, const int tiles, const int pitch, const int* failed) {
    __shared__ float2 shared[8];
    pdl_wait();
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (!kept(a, t)) {
        if (threadIdx.x == 0) a.loss[t] = a.lse[t] = 0.0f;
        return;
    }
    const int gone = threadIdx.x < min(tiles, kFewCtas) ? failed[threadIdx.x] : 0;
    float m = -INFINITY, sum = 0.0f;
    auto add = [&](float2 x) {
        const float most = fmaxf(m, x.x), base = most == -INFINITY ? 0.0f : most;
        sum = sum * exp2f((m - base) * kLog2e) + x.y * exp2f((x.x - base) * kLog2e);
        m = most;
    };
#pragma unroll 4
    for (int i = threadIdx.x; i < tiles; i += 256) add(stats[static_cast<long long>(i) * pitch + t]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float x = __shfl_xor_sync(~0u, m, o), y = __shfl_xor_sync(~0u, sum, o);
        // (the same result in both lanes: the lower one's first)
        const float m0 = lane & o ? x : m, s0 = lane & o ? y : sum, m1 = lane & o ? m : x, s1 = lane & o ? sum : y;
        m = m0;
        sum = s0;
        add(make_float2(m1, s1));
    }
    if (lane == 0) shared[warp] = make_float2(m, sum);
    if (__syncthreads_or(gone) || threadIdx.x) return;
    m = shared[0].x;
    sum = shared[0].y;
    for (int q = 1; q < 8; ++q) add(shared[q]);
    const float rest = logf(sum);
    a.lse[t] = m + rest;
    a.loss[t] = (m - top[t]) + rest;  // (the difference of like logits first: it is exact)
}

int few_tokens(long long n) { return n <= 16 ? 16 : n <= 32 ? 32 : n <= 48 ? 48 : n <= 64 ? 64 : n <= 96 ? 96 : 128; }
template <int NT, bool GRAD>
int launch_few(const FewMaps& maps, const FewParams& p, cudaStream_t st) {
    static std::mutex mu;
    static uint64_t prepared = 0;  // per device: the shared-memory limit
    int dev = 0;
    const int rc = require_device(&dev);
    if (rc) return rc;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 64 || !(prepared >> dev & 1)) {
            const cudaError_t e = cudaFuncSetAttribute(few_logits_kernel<NT, GRAD>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(FewCfg<NT>::kSmem));
            if (e != cudaSuccess) return cuda_fail(e, "few_logits_kernel setup");
            if (dev < 64) prepared |= 1ull << dev;
        }
    }
    const cudaError_t e = launch_pdl(few_logits_kernel<NT, GRAD>, dim3(std::min(p.tiles, kFewCtas)), dim3(kFewThreads), FewCfg<NT>::kSmem, st, maps, p);
    return e == cudaSuccess ? check_launch("few_logits_kernel") : cuda_fail(e, "few_logits_kernel launch");
}
// The shares of the vocabulary: as few passes of up to 256 entries as 148 CTAs need, each as even as eights allow.
template <bool GRAD>
int few_logits(const Args& a, const bf16* h, long long ldh, const bf16* w, FewParams& p, cudaStream_t st) {
    const int nt = few_tokens(a.n);
    FewMaps maps{};
    int rc = make_map(&maps.w, w, 2, a.d, p.vocab, a.ldw, 64, p.tile, true);
    if (!rc) rc = make_map(&maps.h, h, 2, a.d, a.n, ldh, 64, nt, true);
    if (rc) return rc;
    switch (nt) {
        case 16: return launch_few<16, GRAD>(maps, p, st);
        case 32: return launch_few<32, GRAD>(maps, p, st);
        case 48: return launch_few<48, GRAD>(maps, p, st);
        case 64: return launch_few<64, GRAD>(maps, p, st);
        case 96: return launch_few<96, GRAD>(maps, p, st);
        default: return launch_few<128, GRAD>(maps, p, st);
    }
}
FewParams few_params(const Args& a, int col0, int cols) {
    FewParams p{};
    const long long passes = (cols + kFewCtas * 256ll - 1) / (kFewCtas * 256ll), share = (cols + kFewCtas * passes - 1) / (kFewCtas * passes);
    p.tile = static_cast<int>((share + 7) / 8 * 8);
    p.tiles = static_cast<int>((cols + static_cast<long long>(p.tile) - 1) / p.tile);
    p.vocab = cols;
    p.col0 = col0;
    p.d = a.d;
    p.n = static_cast<int>(a.n);
    p.target = a.target;
    p.cap = a.cap;
    return p;
}
int forward_few(const Args& a, cudaStream_t st) {
    FewParams p = few_params(a, 0, a.vocab);
    const int nt = few_tokens(a.n);
    void* base = nullptr;
    constexpr size_t kTop = sizeof(float) * kFewMost, kFailed = sizeof(int) * 160;
    static_assert(kFailed >= sizeof(int) * kFewCtas && (kTop + kFailed) % 16 == 0, "a word for each CTA");
    int rc = scratch_alloc(&base, kTop + kFailed + sizeof(float2) * nt * static_cast<size_t>(p.tiles), st);
    if (rc) return rc;
    p.top = static_cast<float*>(base);
    p.failed = reinterpret_cast<int*>(static_cast<char*>(base) + kTop);
    p.stats = reinterpret_cast<float2*>(static_cast<char*>(base) + kTop + kFailed);
    pdl_fence(st);  // the caller may have queued a cross-stream wait
    rc = few_logits<false>(a, a.h, a.ldh, a.w, p, st);
    if (!rc) {
        const cudaError_t e = launch_pdl(join_few_kernel, dim3(static_cast<unsigned>(a.n)), dim3(256), 0, st, a, p.top, p.stats, p.tiles, nt, p.failed);
        rc = e == cudaSuccess ? check_launch("join_few_kernel") : cuda_fail(e, "join_few_kernel launch");
    }
    scratch_free(base, st);
    return rc;
}

int forward(const Args& a, cudaStream_t st) {
    if (a.n <= kFewMost) return forward_few(a, st);
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
    L.p.failed = s.failed;
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

// Shares of K for each of dh's tiles: those whose last wave wastes least, a share's FP32 sums
// (a tile written and read again) counted as the time of 8 slices.
int dh_splits(long long tiles, long long slices) {
    double best = 0;
    int splits = 1;
    for (int s = 1; s <= 32 && s <= slices; ++s) {
        const double cost = static_cast<double>((tiles * s + kPairs - 1) / kPairs) * ((slices + s - 1) / s + 8);
        if (s == 1 || cost < 0.97 * best) best = cost, splits = s;
    }
    return splits;
}
constexpr long long kPieceG = 128ll << 20;  // bytes of G in one piece of the vocabulary

int backward(const Args& a, cudaStream_t st) {
    const int tiles_m = tiles(a.n, 256), tiles_d = tiles(a.d, 256);
    const long long rows = up(a.n, 256);
    const bool few = a.n <= kFewMost;
    const long long g_rows = few ? few_tokens(a.n) : rows;
    const long long piece = std::min(up(a.vocab, few ? 8 : 256), std::max(256ll, kPieceG / (2 * g_rows) / 256 * 256));
    if (tiles_m * (piece / 256) > 0x3FFFFFFFll || tiles_m * static_cast<long long>(tiles_d) * kPairs > 0x3FFFFFFFll || piece / 256 * tiles_d > 0x3FFFFFFFll)
        return fail(TB_ERR_CAPACITY, "tb_lm_loss_backward: %lld tokens of %d", a.n, a.d);
    // dh's tiles share out their K where they do not fill the GPU
    const int splits = dh_splits(static_cast<long long>(tiles_m) * tiles_d, (piece + 63) / 64);
    Scratch s{};
    void* base = nullptr;
    char* rest = nullptr;
    const long long ldp = up(a.d, 4);
    // dW's tiles share out theirs, the tokens, where there are many and the tiles leave most SMs idle (small heads):
    // sixteen slices each, as the kernel that joins them takes the time of thirty.  (With gradients, 8000 tokens, 130 x 100: 122 us
    // without shares, 89 with; 1000 tokens, 1000 x 200: 63 and 80.)
    const long long dw_tiles = piece >= a.vocab ? tiles(a.vocab, 256) * static_cast<long long>(tiles_d) : kPairs, dw_slices = (a.n + 63) / 64;
    const int dw_splits = dw_slices < 64 ? 1 : static_cast<int>(std::max(1ll, std::min(kPairs / dw_tiles, dw_slices / 16)));
    const size_t g_bytes = up(sizeof(bf16) * g_rows * piece, 256), part_bytes = a.dh ? up(sizeof(float) * splits * rows * ldp, 256) : 0;
    const size_t dw_bytes = a.dw && dw_splits > 1 ? sizeof(float) * dw_splits * a.vocab * ldp : 0;
    int rc = make_scratch(a, g_bytes + part_bytes + dw_bytes, &s, &base, &rest, st);
    if (rc) return rc;
    float* dw_part = reinterpret_cast<float*>(rest + g_bytes + part_bytes);
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
        p.failed = s.failed;
        p.cap = a.cap;
        p.rows = rows;
        p.row = s.row;
        if (few) {
            FewParams q = few_params(a, static_cast<int>(v0), cols);
            q.count = s.count;
            q.failed = s.failed;
            q.row = s.row;
            q.g = s.g;
            q.ldg = piece;
            rc = few_logits<true>(a, s.h, s.ld, w, q, st);
        } else {
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
            rc = operand_map(&L.a[0], s.g, g_rows, cols, piece, false);
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
            rc = operand_map(&L.a[0], s.g, g_rows, cols, piece, true);
            if (!rc) rc = operand_map(&L.b[0][0], s.h, rows, a.d, s.ld, true);
            L.p.splits = dw_splits;
            if (!rc && dw_splits > 1) rc = make_out_map(&L.o[0][0], dw_part, false, a.d, cols, dw_splits, ldp, ldp * cols);
            else if (!rc && L.p.out_tma) rc = make_out_map(&L.o[0][0], L.p.out, true, a.d, cols, 1, a.lddw, a.lddw * cols);
            if (!rc) rc = launch_product(L, static_cast<long long>(tiles(cols, 256)) * tiles_d * dw_splits, st);
            if (!rc && dw_splits > 1)
                rc = launch_small("join_dw_kernel", join_dw_kernel, static_cast<long long>(cols) * ((a.d + 1023) / 1024), st, dw_part, ldp, cols, a.d, dw_splits, s, a.dw, a.lddw);
        }
    }
    if (!rc && a.dh) rc = launch_small("join_dh_kernel", join_dh_kernel, a.n * ((a.d + 1023) / 1024), st, a, s, splits);
    scratch_free(base, st);
    return rc;
}

bool bad_rows(const void* p, int64_t ld, int64_t cols) {
    return !p || reinterpret_cast<uintptr_t>(p) % 16 || ld < cols || ld % 8;
}
bool misaligned(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }
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
        if (!p->target || !p->lse || misaligned(p->target, 8) || misaligned(p->lse, 4)) return fail(TB_ERR_ARG, "%s: null or misaligned target or lse", who);
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
    if (!a.loss || loss::misaligned(a.loss, 4)) return fail(TB_ERR_ARG, "tb_lm_loss: null or misaligned loss");
    if ((rc = require_device(nullptr))) return rc;
    return loss::forward(a, static_cast<cudaStream_t>(stream));
}

extern "C" int tb_lm_loss_backward(const tb_lm_loss_args* p, void* stream) {
    loss::Args a{};
    int rc = loss::check_args("tb_lm_loss_backward", p, &a);
    if (rc) return rc;
    if (a.n > 0 && (!a.dloss || loss::misaligned(a.dloss, 4) || loss::misaligned(a.dlse, 4))) return fail(TB_ERR_ARG, "tb_lm_loss_backward: null or misaligned dloss or dlse");
    if (a.dh && (a.lddh < a.d || loss::misaligned(a.dh, 2))) return fail(TB_ERR_ARG, "tb_lm_loss_backward: dh is misaligned or lddh < d");
    if (a.dw && (a.lddw < a.d || loss::misaligned(a.dw, 2))) return fail(TB_ERR_ARG, "tb_lm_loss_backward: dw is misaligned or lddw < d");
    if ((!a.dh || a.n == 0) && !a.dw) return TB_OK;
    if ((rc = require_device(nullptr))) return rc;
    auto st = static_cast<cudaStream_t>(stream);
    if (a.n == 0) {
        const cudaError_t e = cudaMemset2DAsync(a.dw, sizeof(loss::bf16) * a.lddw, 0, sizeof(loss::bf16) * a.d, a.vocab, st);
        return e == cudaSuccess ? TB_OK : cuda_fail(e, "tb_lm_loss_backward: zeros");
    }
    return loss::backward(a, st);
}
