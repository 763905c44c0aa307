// Orthogonalised updates by Newton-Schulz products, and the masked step of a pruned
// weight that uses them.
//
//   X = U / (|U| + eps);  `steps` times X <- (a I + b A + c A^2) X,  A = X X^T
//
// on the shorter side of U (X^T X and X (...) where U is tall).  The polynomials
// P(A) commute with A, so that several steps need X once:
//
//   P = a I + b A + c A^2,  Q <- P Q,  A <- P A P,  ...,  X <- Q X
//
// which takes symmetric products of the short side only, half of whose tiles are
// computed.  What rounding adds to A grows by up to a^2 = 11.9 with each step that A is
// carried through, in the directions whose singular values are far below the norm:
// X is formed anew after at most three steps, and A from it.  (Five steps in one
// go, with FP32's roundings: up to 6e-3 of the result for spectra that fall off; as three and
// two 2e-4; BF16 results are off by 1.7e-3 in any case.  For k x d, products counted
// by their tiles: 6 k^2 d + 14 k^3 so, 15 k^2 d + 5 k^3 with X formed in each step.)
//
// Operands are pairs of FP16 parts, hi + lo, of the values times a power of two that
// each matrix has for good: 22 bits, as FP32 has 24, at the tensor core's FP16 rate; a
// single FP16 (BF16) part would put 2e-3 (2e-2) of A's error into the directions
// above.  Entries: |X|, |A|, |P A| <= 1.5, |P| <= 3.5, |Q| <= 3.5^3, which FP16's 65504 bounds.
// Where |U| is far below eps, so is |X| below 1, and FP16 ends at 2^-24: X then has another power of two 2^s beside its
// own, which brings |X| to one, less 2^6 with each forming of X anew, in which three steps make it 3.5^3 times larger at most.
#include <algorithm>
#include <cuda_fp16.h>

#include "tb_muon.cuh"
#include "tb_pair_product.cuh"
#include "tb_split_product.cuh"

namespace tb {
namespace muon {
namespace {

using namespace tb::pair;
using bf16 = __nv_bfloat16;

__device__ int g_muon_error;

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr int kExpX = 14, kExpK = 13, kExpQ = 10;  // the powers of two of X; of A, P and P A; of Q
constexpr int kSegment = 3;                        // steps between two formings of X
constexpr int kGrowth = 6;                         // 2^6 > 3.5^kSegment
constexpr int kMostShift = 60;                     // of s: its factors stay in FP32's range
constexpr int kMostSegments = (32 + kSegment - 1) / kSegment;
// What a segment's sums are multiplied by on account of s: those of X X^T, those of the next X, those of the result.
struct Factors {
    float gram, next, result;
};

// The FP16 parts hi + lo of two FP32 values: hi parts in one word, lo parts in another.
__device__ __forceinline__ void split16x2(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// ---- U, and X from it ---------------------------------------------------------------
// The .tb mask: a byte for each `group` weights, in the order of rows, bit k for the k-th; NULL keeps all.
struct Mask {
    const uint8_t* bytes;
    int group, shift;  // shift: the group's logarithm, or -1
};
// Bits 0..3: whether weights i .. i + 3 are kept (of those that exist).
__device__ __forceinline__ uint32_t kept4(const Mask& m, long long i, int exist) {
    if (!m.bytes) return 15u;
    if (m.shift == 2 && i % 4 == 0) return __ldg(m.bytes + (i >> 2));
    if (m.shift == 3 && i % 4 == 0) return __ldg(m.bytes + (i >> 3)) >> (i & 4);
    uint32_t bits = 0;
    long long at = m.shift >= 0 ? i >> m.shift : static_cast<long long>(static_cast<unsigned long long>(i) / static_cast<unsigned>(m.group));
    int in = static_cast<int>(i - at * m.group);
    for (int e = 0; e < 4 && e < exist; ++e) {
        bits |= (__ldg(m.bytes + at) >> in & 1u) << e;
        if (++in == m.group) in = 0, ++at;
    }
    return bits;
}

struct Source {
    int r, d;
    const void* g;
    int g_bf16;
    long long ldg;
    float* m;         // momentum, or NULL
    long long ldm;
    float beta;
    int nesterov;
    Mask mask;
};
// Four columns from `col`, zeros behind the row's end and for pruned weights.
template <typename T>
__device__ __forceinline__ void load4(const T* row, int col, int d, bool wide, float (&v)[4]) {
    if (wide && col + 4 <= d) {
        if constexpr (sizeof(T) == 4) {
            const float4 f = *reinterpret_cast<const float4*>(row + col);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
            const uint2 f = *reinterpret_cast<const uint2*>(row + col);
            v[0] = __uint_as_float(f.x << 16); v[1] = __uint_as_float(f.x & 0xFFFF0000u);
            v[2] = __uint_as_float(f.y << 16); v[3] = __uint_as_float(f.y & 0xFFFF0000u);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = col + e < d ? static_cast<float>(row[col + e]) : 0.0f;
}
__device__ __forceinline__ bool wide_rows(const void* p, long long ld, int size) {
    return ((reinterpret_cast<uintptr_t>(p) | static_cast<unsigned long long>(ld) * size) & (4 * size - 1)) == 0;
}
// Four columns of g and m as they are, and of U.  Loads apart from what follows them, so that
// several are under way in a thread.
struct Four {
    float g[4], m[4];
    uint32_t keep;
};
__device__ __forceinline__ void load_four(const Source& s, bool g_wide, bool m_wide, long long row, int col, Four& x) {
    if (s.g_bf16) load4(static_cast<const bf16*>(s.g) + row * s.ldg, col, s.d, g_wide, x.g);
    else load4(static_cast<const float*>(s.g) + row * s.ldg, col, s.d, g_wide, x.g);
    x.keep = kept4(s.mask, row * s.d + col, s.d - col);
    if (s.m) load4(s.m + row * s.ldm, col, s.d, m_wide, x.m);
}
// The momentum's new value (written if UPDATE), and U.
template <bool UPDATE>
__device__ __forceinline__ void update_four(const Source& s, bool m_wide, long long row, int col, Four& x, float (&u)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = x.keep >> e & 1 ? x.g[e] : 0.0f;
    if (!s.m) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (UPDATE) x.m[e] = x.keep >> e & 1 ? fmaf(s.beta, x.m[e], u[e]) : 0.0f;
        u[e] = s.nesterov ? fmaf(s.beta, x.m[e], u[e]) : x.m[e];
    }
    if constexpr (UPDATE) {
        float* at = s.m + row * s.ldm + col;
        if (m_wide && col + 4 <= s.d) *reinterpret_cast<float4*>(at) = make_float4(x.m[0], x.m[1], x.m[2], x.m[3]);
        else
            for (int e = 0; e < 4 && col + e < s.d; ++e) at[e] = x.m[e];
    }
}
// f(row, col, u) for all of U, by the threads of the grid: kBatch fours a thread at a time.  (The 4096 x 4096 step's first pass:
// 55 us one at a time, 44 so, 65 with four in 76 registers; 27 at the measured copy rate.)
template <bool UPDATE, class F>
__device__ __forceinline__ void for_update(const Source& s, F&& f) {
    constexpr int kBatch = 2;
    const bool g_wide = wide_rows(s.g, s.ldg, s.g_bf16 ? 2 : 4), m_wide = wide_rows(s.m, s.ldm, 4);
    const unsigned units = (s.d + 3) / 4;
    const long long all = static_cast<long long>(s.r) * units, step = gridDim.x * 256ll;
    for (long long i0 = blockIdx.x * 256ll + threadIdx.x; i0 < all; i0 += kBatch * step) {
        Four x[kBatch];
        long long row[kBatch];
        int col[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const long long i = min(i0 + b * step, all - 1);  // (behind the last one: that one again, not used)
            row[b] = all < 0xFFFFFFFFll ? static_cast<unsigned>(i) / units : static_cast<long long>(static_cast<unsigned long long>(i) / units);
            col[b] = 4 * static_cast<int>(i - row[b] * units);
            load_four(s, g_wide, m_wide, row[b], col[b], x[b]);
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (i0 + b * step >= all) break;
            float u[4];
            update_four<UPDATE>(s, m_wide, row[b], col[b], x[b], u);
            f(row[b], col[b], u);
        }
    }
}
constexpr int kNormBlocks = 592;
// Of 256 threads, in a fixed order; for all of them.
__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += shared[i];
    return s;
}
// The momentum's step, and each block's part of |U|^2.  (In 64 bits, as the squares of small and
// large gradients leave FP32's range.)
__global__ void __launch_bounds__(256, 4) norm_kernel(const Source s, double* partial) {
    __shared__ double shared[8];
    double sum = 0.0;
    for_update<true>(s, [&](long long, int, const float (&u)[4]) {
        const float most = fmaxf(fmaxf(fabsf(u[0]), fabsf(u[1])), fmaxf(fabsf(u[2]), fabsf(u[3])));
        if (most > 1e-15f && most < 1e15f) {  // four squares that FP32 holds
            sum += static_cast<double>(fmaf(u[0], u[0], u[1] * u[1]) + fmaf(u[2], u[2], u[3] * u[3]));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = fma(static_cast<double>(u[e]), static_cast<double>(u[e]), sum);
        }
    });
    sum = block_sum(sum, shared);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}
// X's parts, in rows of ld, and the segments' factors; `failed` is reset.
__global__ void __launch_bounds__(256, 4) scale_kernel(const Source s, const double* partial, const int parts, const float eps, uint16_t* hi, uint16_t* lo,
                                                    const long long ld, Factors* factors, int* failed, const int segments) {
    __shared__ double shared[8];
    pdl_wait();
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) sum += partial[i];
    sum = block_sum(sum, shared);
    const double size = sqrt(sum), below = size + static_cast<double>(eps);
    const bool some = size > 0.0 && size < INFINITY;
    const int shift = some ? min(max(-ilogb(size / below) - 1, 0), kMostShift) : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *failed = 0;
    if (blockIdx.x == 0 && threadIdx.x < segments) {
        const int now = max(shift - kGrowth * static_cast<int>(threadIdx.x), 0), then = max(now - kGrowth, 0);
        factors[threadIdx.x] = Factors{ldexpf(1.0f, -2 * now), ldexpf(1.0f, then - now), ldexpf(1.0f, -now)};
    }
    const double scale = ldexp(1.0, kExpX + shift) / below;
    const bool usual = scale > 1e-30 && scale < 1e30;
    const float factor = static_cast<float>(scale);
    for_update<false>(s, [&](long long row, int col, float (&u)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = usual ? u[e] * factor : sum == 0.0 ? 0.0f : static_cast<float>(u[e] * scale);
        uint2 h, l;
        split16x2(u[0], u[1], h.x, l.x);
        split16x2(u[2], u[3], h.y, l.y);
        const long long at = row * ld + col;
        *reinterpret_cast<uint2*>(hi + at) = h;
        *reinterpret_cast<uint2*>(lo + at) = l;
    });
}

// ---- products -----------------------------------------------------------------------
struct Params {
    int m, n, k;          // of the product
    int tiles_m, tiles_n;
    int products;
    float alpha[2];       // powers of two (times c): of what the sums are multiplied by
    const float* factor;  // one more factor of them, in device memory, or NULL
    float beta, diagonal; // P: of A and I
    const uint16_t* c[2]; // P: A's parts
    uint16_t* out[2][2];  // [product][part]
    long long ld;         // of c and out
    int* failed;          // 1 once a wait has expired in one of the call's kernels: no results then
    // results
    void* result;
    long long ldr;
    Mask mask;
    int w_bf16;
    float decay, step;    // W <- mask (decay W - step O)
};
// Four weights' step; `exist` of them are the row's.
__device__ __forceinline__ void update_weights(const Mask& mask, long long flat, bool w_bf16, void* row, int col, int exist, float decay, const float (&change)[4]) {
    const uint32_t keep = kept4(mask, flat, exist);
    if (w_bf16) {
        bf16* w = static_cast<bf16*>(row) + col;
        if (exist >= 4 && reinterpret_cast<uintptr_t>(w) % 8 == 0) {
            const uint2 x = *reinterpret_cast<const uint2*>(w);
            const float f[4] = {__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xFFFF0000u), __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xFFFF0000u)};
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = keep >> e & 1 ? fmaf(decay, f[e], -change[e]) : 0.0f;
            *reinterpret_cast<uint2*>(w) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
        } else {
            for (int e = 0; e < 4 && e < exist; ++e) w[e] = __float2bfloat16_rn(keep >> e & 1 ? fmaf(decay, __bfloat162float(w[e]), -change[e]) : 0.0f);
        }
    } else {
        float* w = static_cast<float*>(row) + col;
        if (exist >= 4 && reinterpret_cast<uintptr_t>(w) % 16 == 0) {
            const float4 x = *reinterpret_cast<const float4*>(w);
            const float f[4] = {x.x, x.y, x.z, x.w};
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = keep >> e & 1 ? fmaf(decay, f[e], -change[e]) : 0.0f;
            *reinterpret_cast<float4*>(w) = make_float4(y[0], y[1], y[2], y[3]);
        } else {
            for (int e = 0; e < 4 && e < exist; ++e) w[e] = keep >> e & 1 ? fmaf(decay, w[e], -change[e]) : 0.0f;
        }
    }
}
// Where rows of weights are whole sixteen (BF16: eight) bytes, `rows` of 32 columns from a piece of O: four columns
// of every fourth row a lane, all loads before the first store.  (A column a lane, its parameters read again for each
// weight, made the 4096 x 4096 step's last product 600 us; so 309, and 282 where it is not a step.)
template <bool BF16>
__device__ __forceinline__ void update_piece(const uint8_t* buf, const Mask& mask, char* w, long long pitch, long long flat, int n, int rows, float decay, float step, int lane) {
    const int sub = lane >> 3, unit = lane & 7;
    uint4 x[8];
    uint32_t keep[8];
    constexpr int kUnit = BF16 ? 8 : 16;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = min(4 * i + sub, rows - 1);
        if constexpr (BF16) {
            const uint2 v = *reinterpret_cast<const uint2*>(w + r * pitch + unit * kUnit);
            x[i].x = v.x;
            x[i].y = v.y;
        } else {
            x[i] = *reinterpret_cast<const uint4*>(w + r * pitch + unit * kUnit);
        }
        keep[i] = kept4(mask, flat + static_cast<long long>(r) * n + 4 * unit, 4);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + sub;
        const float4 o = *reinterpret_cast<const float4*>(buf + piece_at(r, 16 * unit));
        const float change[4] = {step * o.x, step * o.y, step * o.z, step * o.w};
        float f[4], y[4];
        if constexpr (BF16) {
            f[0] = __uint_as_float(x[i].x << 16); f[1] = __uint_as_float(x[i].x & 0xFFFF0000u);
            f[2] = __uint_as_float(x[i].y << 16); f[3] = __uint_as_float(x[i].y & 0xFFFF0000u);
        } else {
            f[0] = __uint_as_float(x[i].x); f[1] = __uint_as_float(x[i].y); f[2] = __uint_as_float(x[i].z); f[3] = __uint_as_float(x[i].w);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = keep[i] >> e & 1 ? fmaf(decay, f[e], -change[e]) : 0.0f;
        if (r >= rows) continue;
        if constexpr (BF16) *reinterpret_cast<uint2*>(w + r * pitch + unit * kUnit) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
        else *reinterpret_cast<float4*>(w + r * pitch + unit * kUnit) = make_float4(y[0], y[1], y[2], y[3]);
    }
}

// Fills a piece of 64 columns x 32 rows with the lane's row of one part.
__device__ __forceinline__ void fill_part(uint8_t* buf, const uint32_t (&v)[32], int lane) {
    uint8_t* row = buf + lane * 128;
#pragma unroll
    for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(row + ((j ^ (lane & 7)) << 4)) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}
__device__ __forceinline__ void store_part(const CUtensorMap* map, uint8_t* buf, int col, int row, int lane) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
        asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(col),
                     "r"(row), "r"(0), "r"(smem_u32(buf))
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}
// The lane's row of 64 columns as rows of both parts.
__device__ __forceinline__ void store_split(const CUtensorMap (&maps)[2], uint8_t* buf, const uint32_t (&hi)[32], const uint32_t (&lo)[32], int col, int row0, int lane) {
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
    fill_part(buf, hi, lane);
    store_part(&maps[0], buf, col, row0, lane);
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
    fill_part(buf, lo, lane);
    store_part(&maps[1], buf, col, row0, lane);
}

// Tile `unit` of those on and below the diagonal, row by row.
__device__ __forceinline__ void lower_tile(int unit, int& tm, int& tn) {
    tm = static_cast<int>((sqrtf(8.0f * static_cast<float>(unit) + 1.0f) - 1.0f) * 0.5f);
    while (tm * (tm + 1) / 2 > unit) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= unit) ++tm;
    tn = unit - tm * (tm + 1) / 2;
}

// A symmetric matrix: its tiles on and below the diagonal, each written where it is
// and mirrored.  MN: operands in memory along M and N (X^T X).  Sums of 256 terms in the
// tensor core.
template <bool MN>
struct Symmetric {
    static constexpr bool kAMn = MN, kBMn = MN, kF16 = true;
    static constexpr int kParts = 2, kGroup = 4;
    using Params = muon::Params;
    static __device__ __forceinline__ int* error() { return &g_muon_error; }
    static __device__ __forceinline__ int items(const Params& p) { return p.tiles_m * (p.tiles_m + 1) / 2 * p.products; }
    static __device__ __forceinline__ Work work(const Params& p, int item) {
        Work w{0, 0, 0, (p.k + 63) / 64, p.products > 1 ? item & 1 : 0, -1};
        lower_tile(p.products > 1 ? item >> 1 : item, w.tm, w.tn);
        return w;
    }
    static __device__ __forceinline__ Work split_work(const Params& p, int item) { return work(p, item); }
    static constexpr bool kMirror = true;
    // C's parts; without C, the factor
    static __device__ __forceinline__ uint4 fetch_quad(const Launch<Symmetric>& L, int row, int col) {
        const Params& p = L.p;
        if (p.factor) return make_uint4(__float_as_uint(*p.factor), 0, 0, 0);
        if (!p.c[0] || row >= p.m || col >= p.n) return make_uint4(0, 0, 0, 0);
        const long long at = row * p.ld + col;  // (rows of ld, a multiple of 8)
        const uint2 h = *reinterpret_cast<const uint2*>(p.c[0] + at), l = *reinterpret_cast<const uint2*>(p.c[1] + at);
        return make_uint4(h.x, h.y, l.x, l.y);
    }
    static __device__ __forceinline__ void finish_quad(const Launch<Symmetric>& L, const Work& w, int row, int col, const float4& v, const uint4& c, uint4& words) {
        const Params& p = L.p;
        const float alpha = p.alpha[w.which] * (p.factor ? __uint_as_float(c.x) : 1.0f);
        const bool inside = row < p.m && col < p.n;
        const long long at = row * p.ld + col;  // (rows of ld, a multiple of 8)
        float x[4] = {v.x * alpha, v.y * alpha, v.z * alpha, v.w * alpha};
        if (p.c[0] && inside) {
            const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&c.x)), h1 = __half22float2(*reinterpret_cast<const __half2*>(&c.y));
            const float2 l0 = __half22float2(*reinterpret_cast<const __half2*>(&c.z)), l1 = __half22float2(*reinterpret_cast<const __half2*>(&c.w));
            const float hs[4] = {h0.x, h0.y, h1.x, h1.y}, ls[4] = {l0.x, l0.y, l1.x, l1.y};
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaf(p.beta, hs[e], fmaf(p.beta, ls[e], x[e])) + (row == col + e ? p.diagonal : 0.0f);
        }
        uint2 hi, lo;
        split16x2(x[0], x[1], hi.x, lo.x);
        split16x2(x[2], x[3], hi.y, lo.y);
        words = make_uint4(hi.x, hi.y, lo.x, lo.y);
        if (inside) {
            *reinterpret_cast<uint2*>(p.out[w.which][0] + at) = hi;
            *reinterpret_cast<uint2*>(p.out[w.which][1] + at) = lo;
        }
    }
    // Two rows of a column at a time (columns left of the diagonal's tile all exist).
    static __device__ __forceinline__ void mirror(const Launch<Symmetric>& L, const Work& w, const uint32_t* words, int pitch, int row0, int rows, int thread) {
        if (w.tm == w.tn) return;
        const Params& p = L.p;
        uint16_t* hi = p.out[w.which][0];
        uint16_t* lo = p.out[w.which][1];
        const int pairs = min(rows, p.m - row0 + 1) / 2;
        for (int c = 4 * (thread >> 5); c < 128; c += kSplitThreads / 8)
            for (int r = 2 * (thread & 31); r < 2 * pairs; r += 64) {  // (a warp writes consecutive rows of four columns)
                const uint4 a = *reinterpret_cast<const uint4*>(words + r * pitch + c), b = *reinterpret_cast<const uint4*>(words + (r + 1) * pitch + c);
                const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
                long long at = (w.tn * 128 + c) * p.ld + row0 + r;
#pragma unroll
                for (int e = 0; e < 2; ++e, at += 2 * p.ld) {
                    *reinterpret_cast<uint32_t*>(hi + at) = low_halves(x[e], y[e]);
                    *reinterpret_cast<uint32_t*>(hi + at + p.ld) = high_halves(x[e], y[e]);
                    *reinterpret_cast<uint32_t*>(lo + at) = low_halves(x[2 + e], y[2 + e]);
                    *reinterpret_cast<uint32_t*>(lo + at + p.ld) = high_halves(x[2 + e], y[2 + e]);
                }
            }
    }
    static __device__ __forceinline__ void finish(const Launch<Symmetric>& L, const Work& w, float (&acc)[128], uint8_t* buf, int row_in, int half, int lane) {
        const Params& p = L.p;
        const int row0 = w.tm * 256 + row_in, row = row0 + lane, col = w.tn * 256 + half * 128;
        if (col / 128 > row0 / 128 || row0 >= p.m || col >= p.n) return;
        const float alpha = p.alpha[w.which] * (p.factor ? *p.factor : 1.0f);
        const bool mirrored = col / 128 != row0 / 128, odd = lane & 1;
        // selectors of the halves that a lane sends to its neighbour, and of what it makes of those that it gets
        const uint32_t send = odd ? 0x5410u : 0x7632u, take_hi = odd ? 0x3254u : 0x5410u, take_lo = odd ? 0x3276u : 0x7610u;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int col0 = col + 64 * c;
            if (col0 >= p.n) break;
            float* x = acc + 64 * c;
#pragma unroll
            for (int i = 0; i < 64; ++i) x[i] *= alpha;
            if (p.c[0]) {  // (rows of ld, a multiple of 8)
                const long long at = min(row, p.m - 1) * p.ld + col0;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    uint4 h[4], l[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool inside = col0 + 32 * q + 8 * j < p.n;
                        h[j] = l[j] = make_uint4(0, 0, 0, 0);
                        if (inside) h[j] = *reinterpret_cast<const uint4*>(p.c[0] + at + 32 * q + 8 * j);
                        if (inside) l[j] = *reinterpret_cast<const uint4*>(p.c[1] + at + 32 * q + 8 * j);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t hw[4] = {h[j].x, h[j].y, h[j].z, h[j].w}, lw[4] = {l[j].x, l[j].y, l[j].z, l[j].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&hw[e])), lf = __half22float2(*reinterpret_cast<const __half2*>(&lw[e]));
                            float* to = x + 32 * q + 8 * j + 2 * e;
                            to[0] = fmaf(p.beta, hf.x, fmaf(p.beta, lf.x, to[0]));
                            to[1] = fmaf(p.beta, hf.y, fmaf(p.beta, lf.y, to[1]));
                        }
                    }
                }
                if (!mirrored) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) x[i] += col0 + i == row ? p.diagonal : 0.0f;
                }
            }
            uint32_t hi[32], lo[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) split16x2(x[2 * i], x[2 * i + 1], hi[i], lo[i]);
            store_split(L.o[w.which], buf, hi, lo, col0, row0, lane);
            if (!mirrored) continue;
            // two lanes exchange, so that each has two rows of one column
            const long long at = (col0 + odd) * p.ld + (row & ~1);
            uint16_t* out_hi = p.out[w.which][0] + at;
            uint16_t* out_lo = p.out[w.which][1] + at;
            const bool both = (row | 1) < p.m, one = (row & ~1) < p.m;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t other = __shfl_xor_sync(~0u, __byte_perm(hi[i], lo[i], send), 1);
                const uint32_t h = __byte_perm(hi[i], other, take_hi), l = __byte_perm(lo[i], other, take_lo);
                if (both) {
                    *reinterpret_cast<uint32_t*>(out_hi) = h;
                    *reinterpret_cast<uint32_t*>(out_lo) = l;
                } else if (one) {
                    *out_hi = static_cast<uint16_t>(h);
                    *out_lo = static_cast<uint16_t>(l);
                }
                out_hi += 2 * p.ld;
                out_lo += 2 * p.ld;
            }
        }
    }
};

// X's product with Q: X's parts again, BF16 results, or the weights' step.  BMN: Q X, else X Q.
enum Out { kSplit = 0, kBf16 = 1, kWeights = 2 };
template <bool BMN, int OUT>
struct Apply {
    static constexpr bool kAMn = false, kBMn = BMN, kF16 = true;
    static constexpr int kParts = 2, kGroup = 4;
    using Params = muon::Params;
    static __device__ __forceinline__ int* error() { return &g_muon_error; }
    static __device__ __forceinline__ int items(const Params& p) { return p.tiles_m * p.tiles_n; }
    static __device__ __forceinline__ Work work(const Params& p, int item) {
        Work w{0, 0, 0, (p.k + 63) / 64, 0, -1};
        band_tile(item, p.tiles_m, p.tiles_n, w.tm, w.tn);
        return w;
    }
    static __device__ __forceinline__ void finish(const Launch<Apply>& L, const Work& w, float (&acc)[128], uint8_t* buf, int row_in, int half, int lane) {
        const Params& p = L.p;
        const int row0 = w.tm * 256 + row_in, col = w.tn * 256 + half * 128;
        const int rows = min(32, p.m - row0), cols = p.n - col;
        if (rows <= 0 || cols <= 0) return;
        const float alpha = p.alpha[0] * *p.factor;
        if (OUT != kSplit && *p.failed) return;
        if constexpr (OUT == kSplit) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (64 * c >= cols) break;
                uint32_t hi[32], lo[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) split16x2(acc[64 * c + 2 * i] * alpha, acc[64 * c + 2 * i + 1] * alpha, hi[i], lo[i]);
                store_split(L.o[0], buf, hi, lo, col + 64 * c, row0, lane);
            }
        } else if constexpr (OUT == kBf16) {
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] *= alpha;
            store_rows<true>(buf, acc, static_cast<bf16*>(p.result) + row0 * p.ldr + col, p.ldr, rows, cols, lane);
        } else {
            const Mask mask = p.mask;
            const float step = p.step * alpha, decay = p.decay;
            const bool w_bf16 = p.w_bf16;
            const int n = p.n, size = w_bf16 ? 2 : 4;
            const long long pitch = p.ldr * size;
            char* w0 = static_cast<char*>(p.result) + row0 * pitch;
            const bool whole = (reinterpret_cast<uintptr_t>(p.result) | pitch) % (4 * size) == 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int col0 = col + 32 * c, left = cols - 32 * c;
                if (left <= 0) break;
                __syncwarp();
                fill_piece<false>(buf, acc, c, lane);
                __syncwarp();
                const long long flat = static_cast<long long>(row0) * n + col0;
                if (whole && left >= 32) {
                    if (w_bf16) update_piece<true>(buf, mask, w0 + col0 * 2, pitch, flat, n, rows, decay, step, lane);
                    else update_piece<false>(buf, mask, w0 + col0 * 4, pitch, flat, n, rows, decay, step, lane);
                } else {
                    const int unit = 4 * (lane & 7);
#pragma unroll 1
                    for (int r = lane >> 3; r < rows && unit < left; r += 4) {
                        const float4 o = *reinterpret_cast<const float4*>(buf + piece_at(r, 4 * unit));
                        const float change[4] = {step * o.x, step * o.y, step * o.z, step * o.w};
                        update_weights(mask, flat + static_cast<long long>(r) * n + unit, w_bf16, w0 + r * pitch, col0 + unit, left - unit, decay, change);
                    }
                }
            }
        }
    }
    static __device__ __forceinline__ Work split_work(const Params& p, int tile) {
        const int tiles = (p.n + 127) / 128;
        return Work{tile / tiles, tile % tiles, 0, (p.k + 63) / 64, 0, -1};
    }
    static constexpr bool kMirror = false;
    static __device__ __forceinline__ uint4 fetch_quad(const Launch<Apply>& L, int, int) {
        return make_uint4(__float_as_uint(*L.p.factor), OUT != kSplit ? static_cast<uint32_t>(*L.p.failed) : 0u, 0, 0);
    }
    static __device__ __forceinline__ void finish_quad(const Launch<Apply>& L, const Work&, int row, int col, const float4& v, const uint4& c, uint4&) {
        const Params& p = L.p;
        if (row >= p.m || col >= p.n || c.y) return;
        const float alpha = p.alpha[0] * __uint_as_float(c.x), factor = OUT == kWeights ? alpha * p.step : alpha;
        const float x[4] = {v.x * factor, v.y * factor, v.z * factor, v.w * factor};
        if constexpr (OUT == kSplit) {
            uint2 hi, lo;
            split16x2(x[0], x[1], hi.x, lo.x);
            split16x2(x[2], x[3], hi.y, lo.y);
            const long long at = row * p.ld + col;
            *reinterpret_cast<uint2*>(p.out[0][0] + at) = hi;
            *reinterpret_cast<uint2*>(p.out[0][1] + at) = lo;
        } else if constexpr (OUT == kBf16) {
            bf16* out = static_cast<bf16*>(p.result) + row * p.ldr + col;
            if (col + 4 <= p.n && reinterpret_cast<uintptr_t>(out) % 8 == 0) {
                *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < p.n) out[e] = __float2bfloat16_rn(x[e]);
            }
        } else {
            char* w = static_cast<char*>(p.result) + row * p.ldr * (p.w_bf16 ? 2 : 4);
            update_weights(p.mask, static_cast<long long>(row) * p.n + col, p.w_bf16, w, col, p.n - col, p.decay, x);
        }
    }
};

// ---- short sides up to 128 -----------------------------------------------------------------
// All of the iteration in one launch, by a cluster of up to 4 CTAs that share the long side out, up to two chunks of 128 each.
// Each sums its part of A; the cluster's CTAs add up a share of A's rows each, through distributed shared memory,
// and copy the others'; then each forms Q by itself, and its own part of Q X.
//
// A (then P A), P and Q lie in shared memory as operands, 64 KB each, every product of them one 128 x 128
// tile; a thread turns 32 columns of a row of the accumulator into the next operand's parts.  A chunk of X, 128 of its long side, is
// four tiles of 64 columns x 128 rows (hi, hi, lo, lo) in the places of P and Q, which are not needed then.  The same
// tile in memory is an operand along its rows and one along its columns.
// (128 x 128, whole call: 56 us, of which a product of the chain takes 1.65; as eight launches 79.  16 x 512: 61 and 66; 128 x 1024: 80
// and 81; 128 x 2048: 89 and 83.)  With `core` the kernel forms Q from A alone: of longer sides
// A comes from clusters of 8, and Q X is shared out over all SMs.
constexpr int kShortThreads = 512, kShortMatrix = 65536, kShortTile = 16384;  // thread 0 also loads and issues MMAs
constexpr int kShortChunks = 8, kShortCtas = 4;  // the most that the whole iteration is done here with, two chunks a CTA
constexpr size_t kShortSmem = 3 * kShortMatrix + 1024 + 128;
struct ShortMaps {
    CUtensorMap x[2];  // X's parts, or A's
};
struct ShortParams {
    int k, r, d, tall, chunks;
    int steps, segments;
    int core;
    const Factors* factors;  // each segment's
    int* failed;
    uint16_t* x[2];    // X's parts, written anew between segments; or Q's
    long long ld;
    void* result;
    long long ldr;
    Mask mask;
    int w_bf16;
    float decay, step;
};
__device__ __forceinline__ uint4 load_cluster_u4(uint32_t addr, uint32_t rank) {
    uint4 v;
    asm volatile(
        "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\t"
        "ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [a];\n\t}"
        : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
        : "r"(addr), "r"(rank)
        : "memory");
    return v;
}
// Place of 8 columns from `col` of row r in a matrix's operand: slices of 64 columns, each a tile of hi and one of lo parts.
__device__ __forceinline__ int operand_at(int r, int col, int part) {
    return (2 * (col >> 6) + part) * kShortTile + r * 128 + ((((col & 63) >> 3) ^ (r & 7)) << 4);
}
template <int OUT>
__global__ void __launch_bounds__(kShortThreads, 1) short_kernel(const __grid_constant__ ShortMaps maps, const __grid_constant__ ShortParams p, const int ctas) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t* loaded = reinterpret_cast<uint64_t*>(smem + 3 * kShortMatrix);  // [2] a chunk's buffer filled
    uint64_t* used = loaded + 2;                                            // [2] and read
    uint64_t* done = used + 2;                                              // [2] an accumulator finished
    uint64_t* taken = done + 2;                                             // [2] and read (products with X)
    uint64_t* drained = taken + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank());
    if (threadIdx.x == 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.x[0])) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.x[1])) : "memory");
    }
    if (threadIdx.x == 0) {
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&loaded[b]), 1);
            mbar_init(smem_u32(&used[b]), 1);
            mbar_init(smem_u32(&done[b]), 1);
            mbar_init(smem_u32(&taken[b]), 16);
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
    pdl_wait();

    const bool issuer = threadIdx.x == 0;
    const int row = (warp & 3) * 32 + lane, part4 = warp >> 2;  // a thread has columns 32 part4 .. of `row`
    const int first = share_at(p.chunks, rank, ctas), own = share_at(p.chunks, rank + 1, ctas) - first;
    constexpr uint32_t kIdesc = (1u << 4) | (8u << 24);  // FP16 operands, FP32 sums, M = 128
    constexpr uint32_t kN128 = (128u >> 3) << 17, kAlongM = 1u << 15, kAlongN = 1u << 16;
    constexpr uint64_t kLoMatrix = kShortTile >> 4, kLoChunk = 2 * kShortTile >> 4;  // from hi to lo: of a matrix's slice, of a chunk's tile
    auto buffer = [&](int b) { return smem_u32(smem + b * kShortMatrix); };
    // columns along memory's rows: K steps of 32 bytes; rows along K: steps of 16 rows, chunks of M or N a tile apart
    auto tile_desc = [&](uint32_t at, bool mn) {
        return static_cast<uint64_t>((at >> 4) & 0x3FFFu) | (static_cast<uint64_t>(mn ? kShortTile >> 4 : 1) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
    };
    auto gave_up = [&] {  // (what follows goes on, but no result is written)
        *abort_flag = 1;
        atomicExch(&g_muon_error, 1);
        atomicExch(p.failed, 1);
    };
    // the issuer's counts: loads into each buffer, products with X into each accumulator
    int loads[2] = {0, 0}, products[2] = {0, 0};
    auto load_chunk = [&](int i, int b) {  // X's chunk `first` + i into buffer 1 + b
        if (*abort_flag) return;
        if (loads[b] && !wait(smem_u32(&used[b]), (loads[b] - 1) & 1, abort_flag)) return gave_up();
        mbar_expect_tx(smem_u32(&loaded[b]), kShortMatrix);
        const int at = 128 * (first + i);
        for (int q = 0; q < 4; ++q)
            tma_load_2d(buffer(1 + b) + q * kShortTile, &maps.x[q >> 1], (p.tall ? 0 : at) + 64 * (q & 1), p.tall ? at : 0, smem_u32(&loaded[b]));
        ++loads[b];
    };
    auto chunk_ready = [&](int b) {
        if (*abort_flag) return false;
        if (!wait(smem_u32(&loaded[b]), (loads[b] - 1) & 1, abort_flag)) {
            gave_up();
            return false;
        }
        fence_after();
        return true;
    };
    uint32_t phase[2] = {0, 0};  // of `done`
    auto finished = [&](int d) {
        if (!wait(smem_u32(&done[d]), phase[d], abort_flag) && !*abort_flag) gave_up();
        phase[d] ^= 1;
        __syncwarp();
        fence_after();
    };
    float f[32];
    auto read_sums = [&](int d) { tmem_ld32(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + static_cast<uint32_t>(128 * d + 32 * part4), f); };
    uint32_t hi[16], lo[16];
    auto split_sums = [&] {
#pragma unroll
        for (int i = 0; i < 16; ++i) split16x2(f[2 * i], f[2 * i + 1], hi[i], lo[i]);
    };
    auto put = [&](int to) {  // as an operand
        uint8_t* at = smem + to * kShortMatrix;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            *reinterpret_cast<uint4*>(at + operand_at(row, 32 * part4 + 8 * j, 0)) = make_uint4(hi[4 * j], hi[4 * j + 1], hi[4 * j + 2], hi[4 * j + 3]);
            *reinterpret_cast<uint4*>(at + operand_at(row, 32 * part4 + 8 * j, 1)) = make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]);
        }
    };
    auto meet = [&](bool x_too) {  // what was written here (and to X) may be read by MMAs (and TMA), and the accumulators be written
        if (x_too) asm volatile("fence.proxy.async;" ::: "memory");
        else asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        fence_before();
        __syncthreads();
        fence_after();
    };
    // accumulator d = the product of the matrices in buffers x and y
    auto product = [&](int d, int x, int y) {
        if (!issuer || *abort_flag) return;
        const uint64_t xd = tile_desc(buffer(x), false), yd = tile_desc(buffer(y), false);
        for (int s = 0; s < (p.k > 64 ? 2 : 1); ++s)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                const uint64_t a = xd + s * 2 * kLoMatrix + 2 * kk, b = yd + s * 2 * kLoMatrix + 2 * kk;
                mma_one16<true>(tmem + 128 * d, a + kLoMatrix, b, kIdesc | kN128, s | kk);
                mma_one16<true>(tmem + 128 * d, a, b + kLoMatrix, kIdesc | kN128, 1);
                mma_one16<true>(tmem + 128 * d, a, b, kIdesc | kN128, 1);
            }
        mma_commit(smem_u32(&done[d]));
    };
    // the accumulator's values times alpha (plus beta C + diagonal I), split
    auto take = [&](int d, float alpha, int c, float beta, float diagonal) {
        finished(d);
        read_sums(d);
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] *= alpha;
        if (c >= 0) {
            const uint8_t* at = smem + c * kShortMatrix;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4 h = *reinterpret_cast<const uint4*>(at + operand_at(row, 32 * part4 + 8 * j, 0)), l = *reinterpret_cast<const uint4*>(at + operand_at(row, 32 * part4 + 8 * j, 1));
                const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 hf = __half22float2(*reinterpret_cast<const __half2*>(&hw[e])), lf = __half22float2(*reinterpret_cast<const __half2*>(&lw[e]));
                    f[8 * j + 2 * e] = fmaf(beta, hf.x, fmaf(beta, lf.x, f[8 * j + 2 * e]));
                    f[8 * j + 2 * e + 1] = fmaf(beta, hf.y, fmaf(beta, lf.y, f[8 * j + 2 * e + 1]));
                }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] += 32 * part4 + i == row && row < p.k ? diagonal : 0.0f;
        }
        split_sums();
    };

    constexpr float kDown = 1.0f / (1 << kExpK);  // A, P and P A all have this power of two
    constexpr float kGram = 1.0f / (1 << (2 * kExpX - kExpK));
    for (int seg = 0; seg < p.segments; ++seg) {
        const Factors factors = p.core ? Factors{1.0f, 1.0f, 1.0f} : p.factors[seg];
        const float gram = kGram * factors.gram;
        // ---- A into buffer 0 ----
        if (p.core) {
            if (issuer) {
                mbar_expect_tx(smem_u32(&loaded[0]), kShortMatrix);
                for (int q = 0; q < 4; ++q) tma_load_2d(buffer(0) + q * kShortTile, &maps.x[q & 1], 64 * (q >> 1), 0, smem_u32(&loaded[0]));
                ++loads[0];
                chunk_ready(0);
            }
            meet(false);
        } else {
            if (issuer) {
                load_chunk(0, 0);
                for (int i = 0; i < own; ++i) {
                    const int b = i & 1;
                    if (i + 1 < own) load_chunk(i + 1, b ^ 1);
                    if (!chunk_ready(b)) break;
                    // (an accumulator for each chunk)
                    for (int s = 0; s < (p.tall || 64 < p.d - 128 * (first + i) ? 2 : 1); ++s)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            const uint64_t x = p.tall ? tile_desc(buffer(1 + b), true) + (4 * s + kk) * 128 : tile_desc(buffer(1 + b) + s * kShortTile, false) + 2 * kk;
                            const uint32_t idesc = kIdesc | kN128 | (p.tall ? kAlongM | kAlongN : 0u);
                            mma_one16<true>(tmem + 128 * b, x + kLoChunk, x, idesc, s || kk);
                            mma_one16<true>(tmem + 128 * b, x, x + kLoChunk, idesc, 1);
                            mma_one16<true>(tmem + 128 * b, x, x, idesc, 1);
                        }
                    mma_commit(smem_u32(&used[b]));
                }
                mma_commit(smem_u32(&done[0]));
                if (own > 1) mma_commit(smem_u32(&done[1]));
            }
            __syncwarp();
            finished(0);
            read_sums(0);
            if (own > 1) {
                finished(1);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t x[16];
                    tmem_ld16(tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + static_cast<uint32_t>(128 + 32 * part4 + 16 * c), x);
                    tmem_wait16(x);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) add2(f[16 * c + i], f[16 * c + i + 1], x[i], x[i + 1]);
                }
            }
            if (ctas == 1) {
#pragma unroll
                for (int i = 0; i < 32; ++i) f[i] *= gram;
                split_sums();
                put(0);
            }
            if (ctas > 1) {
                float* sums = reinterpret_cast<float*>(smem + kShortMatrix);  // rows of kSplitPitch, where the chunks were
#pragma unroll
                for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(sums + row * kSplitPitch + 32 * part4 + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
                __syncwarp();
                cluster_arrive();
                cluster_wait();
                // (a CTA that gave up has no sums)
                if (lane < ctas && lane != rank && load_cluster_int(smem_u32(const_cast<int*>(abort_flag)), static_cast<uint32_t>(lane))) *abort_flag = 1;
                const int row0 = 2 * share_at(64, rank, ctas), rows = 2 * share_at(64, rank + 1, ctas) - row0;
                for (int i = threadIdx.x; i < rows * 32; i += kShortThreads) {
                    const int r = row0 + (i >> 5), c = 4 * (i & 31);
                    float4 v[kShortCtas];
#pragma unroll
                    for (int q = 0; q < kShortCtas; ++q)
                        if (q < ctas) v[q] = load_cluster4(smem_u32(sums + r * kSplitPitch + c), static_cast<uint32_t>(q));
#pragma unroll
                    for (int q = 1; q < kShortCtas; ++q)
                        if (q < ctas) { v[0].x += v[q].x; v[0].y += v[q].y; v[0].z += v[q].z; v[0].w += v[q].w; }
                    uint2 h, l;
                    split16x2(v[0].x * gram, v[0].y * gram, h.x, l.x);
                    split16x2(v[0].z * gram, v[0].w * gram, h.y, l.y);
                    *reinterpret_cast<uint2*>(smem + operand_at(r, c, 0) + (c & 4) * 2) = h;
                    *reinterpret_cast<uint2*>(smem + operand_at(r, c, 1) + (c & 4) * 2) = l;
                }
                __syncwarp();
                cluster_arrive();
                cluster_wait();
                for (int i = threadIdx.x; i < 128 * 32; i += kShortThreads) {
                    const int r = i >> 5, unit = i & 31;
                    if (r >= row0 && r < row0 + rows) continue;
                    int owner = 0;
                    while (2 * share_at(64, owner + 1, ctas) <= r) ++owner;
                    const int at = operand_at(r, 8 * (unit & 15), unit >> 4);
                    *reinterpret_cast<uint4*>(smem + at) = load_cluster_u4(smem_u32(smem + at), static_cast<uint32_t>(owner));
                }
                __syncwarp();
                cluster_arrive();  // (nobody's A, nor sums, change before all have read them)
                cluster_wait();
            }
            meet(false);
        }
        // ---- Q of this segment's steps into buffer 0 ----
        const int steps = p.steps * (seg + 1) / p.segments - p.steps * seg / p.segments;
        int P = 1, Q = 1;
        for (int i = 0; i < steps; ++i) {
            const bool last = i == steps - 1;
            if (i) P = 3 - Q;
            product(0, 0, 0);
            take(0, kC * kDown, 0, kB, kA * (1 << kExpK));
            put(last && i == 0 ? 0 : P);  // (buffer 0: what a thread writes there it alone has read)
            meet(false);
            if (last && i == 0) break;
            const float down_q = i == 1 ? 1.0f / (1 << (2 * kExpK - kExpQ)) : kDown;
            if (last) {
                product(0, P, Q);
                take(0, down_q, -1, 0, 0);
                put(0);
                meet(false);
                break;
            }
            product(0, P, 0);
            if (i) product(1, P, Q);
            take(0, kDown, -1, 0, 0);
            put(0);  // (the products that read A, and Q, ...
            if (i) {
                take(1, down_q, -1, 0, 0);
                put(Q);  // ... are done)
            }
            meet(false);
            product(0, P, 0);
            take(0, kDown, -1, 0, 0);
            put(0);
            meet(false);
        }
        if (p.core) {
            if (row < p.k && !*abort_flag) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int col = 32 * part4 + 8 * j;
                    if (col >= p.ld) break;
                    *reinterpret_cast<uint4*>(p.x[0] + row * p.ld + col) = make_uint4(hi[4 * j], hi[4 * j + 1], hi[4 * j + 2], hi[4 * j + 3]);
                    *reinterpret_cast<uint4*>(p.x[1] + row * p.ld + col) = make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]);
                }
            }
            continue;
        }
        // ---- this CTA's part of Q X (tall: X Q) ----
        const int exp_q = steps > 1 ? kExpQ : kExpK;
        const bool end = seg == p.segments - 1;
        const float alpha = 1.0f / static_cast<float>(1 << (end ? exp_q + kExpX - 13 : exp_q)) * (end ? factors.result / 8192 : factors.next);
        auto multiply = [&](int i) {
            const int b = i & 1;
            if (!chunk_ready(b)) return;
            if (products[b] && !wait(smem_u32(&taken[b]), (products[b] - 1) & 1, abort_flag)) return gave_up();
            ++products[b];
            fence_after();
            const uint64_t qd = tile_desc(buffer(0), false);
            const uint64_t x = tile_desc(buffer(1 + b), !p.tall);
            const uint32_t idesc = kIdesc | kN128 | (p.tall ? 0u : kAlongN);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
                if (kk == 4 && p.k <= 64) break;
                const uint64_t q = qd + (kk >> 2) * 2 * kLoMatrix + 2 * (kk & 3);
                const uint64_t at = x + (p.tall ? (kk >> 2) * (kShortTile >> 4) + 2 * (kk & 3) : kk * 128);
                if (p.tall) {
                    mma_one16<true>(tmem + 128 * b, at + kLoChunk, q, idesc, kk);
                    mma_one16<true>(tmem + 128 * b, at, q + kLoMatrix, idesc, 1);
                    mma_one16<true>(tmem + 128 * b, at, q, idesc, 1);
                } else {
                    mma_one16<true>(tmem + 128 * b, q + kLoMatrix, at, idesc, kk);
                    mma_one16<true>(tmem + 128 * b, q, at + kLoChunk, idesc, 1);
                    mma_one16<true>(tmem + 128 * b, q, at, idesc, 1);
                }
            }
            mma_commit(smem_u32(&used[b]));
            mma_commit(smem_u32(&done[b]));
        };
        if (issuer) {
            load_chunk(0, 0);
            if (own > 1) load_chunk(1, 1);
            multiply(0);
        }
        for (int i = 0; i < own; ++i) {
            const int b = i & 1, at = 128 * (first + i);
            if (issuer && i + 1 < own) {
                multiply(i + 1);
            }
            __syncwarp();
            finished(b);
            if (*abort_flag) break;
            read_sums(b);
            fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&taken[b])) : "memory");
            const int r = p.tall ? at + row : row, col = (p.tall ? 0 : at) + 32 * part4;
            if (r >= p.r || col >= p.d) continue;
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] *= alpha;
            if (!end) {  // (rows of ld, a multiple of 8)
                split_sums();
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (col + 8 * j >= p.d) break;
                    *reinterpret_cast<uint4*>(p.x[0] + r * p.ld + col + 8 * j) = make_uint4(hi[4 * j], hi[4 * j + 1], hi[4 * j + 2], hi[4 * j + 3]);
                    *reinterpret_cast<uint4*>(p.x[1] + r * p.ld + col + 8 * j) = make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]);
                }
            } else if constexpr (OUT == kBf16) {
                bf16* out = static_cast<bf16*>(p.result) + r * p.ldr + col;
                const bool wide = reinterpret_cast<uintptr_t>(out) % 16 == 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float* x = f + 8 * j;
                    if (wide && col + 8 * j + 8 <= p.d) {
                        *reinterpret_cast<uint4*>(out + 8 * j) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (col + 8 * j + e < p.d) out[8 * j + e] = __float2bfloat16_rn(x[e]);
                    }
                }
            } else if constexpr (OUT == kWeights) {
                char* w = static_cast<char*>(p.result) + r * p.ldr * (p.w_bf16 ? 2 : 4);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (col + 4 * j >= p.d) break;
                    const float change[4] = {p.step * f[4 * j], p.step * f[4 * j + 1], p.step * f[4 * j + 2], p.step * f[4 * j + 3]};
                    update_weights(p.mask, static_cast<long long>(r) * p.d + col + 4 * j, p.w_bf16, w, col + 4 * j, p.d - col - 4 * j, p.decay, change);
                }
            }
        }
        meet(true);
    }
    if (issuer && *abort_flag) {  // loads and MMAs in flight, within a limit
        for (int b = 0; b < 2; ++b)
            if (loads[b]) wait(smem_u32(&loaded[b]), (loads[b] - 1) & 1, nullptr);
        drain_one(smem_u32(drained));
    }
    meet(false);
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256));
}

long long up(long long v, long long m) { return (v + m - 1) / m * m; }

struct Matrix {
    uint16_t* part[2];
    long long rows, cols, ld;
    int exp;
};
float power(int e) { return ldexpf(1.0f, e); }

int operand_maps(CUtensorMap (&maps)[2], const Matrix& x, bool mn) {
    int rc = TB_OK;
    for (int q = 0; q < 2 && !rc; ++q) rc = operand_map(&maps[q], x.part[q], x.rows, x.cols, x.ld, mn);
    return rc;
}
int out_maps(CUtensorMap (&maps)[2], const Matrix& x) {
    int rc = TB_OK;
    for (int q = 0; q < 2 && !rc; ++q) rc = make_out_map(&maps[q], x.part[q], true, x.cols, x.rows, 1, x.ld, x.ld * x.rows);
    return rc;
}

// out = scale A B^T (MN: scale A^T B), a symmetric matrix; plus beta C + diagonal I where C is given.
// With a second B and out, two products with the same A; with a factor (in device memory), that too.
template <bool MN>
int symmetric(const Matrix& a, const Matrix& b, const Matrix& out, float scale, const Matrix* c, float beta, float diagonal, const Matrix* b2, const Matrix* out2,
              int* failed, cudaStream_t st, const float* factor = nullptr) {
    Launch<Symmetric<MN>> L{};
    Params& p = L.p;
    p.m = p.n = static_cast<int>(out.rows);
    p.k = static_cast<int>(MN ? a.rows : a.cols);
    p.tiles_m = tiles(p.m, 256);
    p.products = b2 ? 2 : 1;
    p.ld = out.ld;
    int rc = operand_maps(L.a, a, MN);
    if (!rc) rc = operand_maps(L.b[0], b, MN);
    if (!rc) rc = out_maps(L.o[0], out);
    if (!rc && b2) rc = operand_maps(L.b[1], *b2, MN);
    if (!rc && b2) rc = out_maps(L.o[1], *out2);
    if (rc) return rc;
    p.factor = factor;
    p.failed = failed;
    p.alpha[0] = scale * power(out.exp - a.exp - b.exp);
    if (b2) p.alpha[1] = scale * power(out2->exp - a.exp - b2->exp);
    for (int q = 0; q < 2; ++q) {
        p.out[0][q] = out.part[q];
        if (b2) p.out[1][q] = out2->part[q];
        if (c) p.c[q] = c->part[q];
    }
    if (c) {
        p.beta = beta * power(out.exp - c->exp);
        p.diagonal = diagonal * power(out.exp);
    }
    const long long t = (p.m + 127) / 128, pairs = static_cast<long long>(p.tiles_m) * (p.tiles_m + 1) / 2 * p.products, units = t * (t + 1) / 2 * p.products;
    return launch_either(L, units, pairs, (p.k + 63) / 64, st);
}

struct Result {
    int* failed;
    void* out;
    long long ld;
    Mask mask;
    int w_bf16;
    float decay, step;
};
// X (Q X, tall: X Q) into `out`, or into the result.
template <bool BMN, int OUT>
int apply(const Matrix& q, const Matrix& x, const Matrix& out, const Result& res, const Factors* factors, cudaStream_t st) {
    pair::Launch<Apply<BMN, OUT>> L{};
    Params& p = L.p;
    p.m = static_cast<int>(x.rows);
    p.n = static_cast<int>(x.cols);
    p.k = static_cast<int>(q.rows);
    p.tiles_m = tiles(p.m, 256);
    p.tiles_n = tiles(p.n, 256);
    int rc = operand_maps(L.a, BMN ? q : x, false);
    if (!rc) rc = operand_maps(L.b[0], BMN ? x : q, BMN);
    if (!rc && OUT == kSplit) rc = out_maps(L.o[0], out);
    if (rc) return rc;
    p.factor = OUT == kSplit ? &factors->next : &factors->result;
    p.alpha[0] = power((OUT == kSplit ? out.exp : 0) - q.exp - x.exp);
    p.failed = res.failed;
    p.result = res.out;
    p.ldr = res.ld;
    p.mask = res.mask;
    p.w_bf16 = res.w_bf16;
    p.decay = res.decay;
    p.step = res.step;
    if (OUT == kSplit) {
        p.ld = out.ld;
        for (int q = 0; q < 2; ++q) p.out[0][q] = out.part[q];
    }
    const long long pairs = static_cast<long long>(p.tiles_m) * p.tiles_n, units = static_cast<long long>((p.m + 127) / 128) * ((p.n + 127) / 128);
    return launch_either(L, units, pairs, (p.k + 63) / 64, st);
}
template <int OUT>
int apply(bool tall, const Matrix& q, const Matrix& x, const Matrix& out, const Result& res, const Factors* factors, cudaStream_t st) {
    return tall ? apply<false, OUT>(q, x, out, res, factors, st) : apply<true, OUT>(q, x, out, res, factors, st);
}

template <int OUT>
int launch_short(const ShortMaps& maps, const ShortParams& p, int ctas, cudaStream_t st) {
    static std::mutex mu;
    static uint64_t prepared = 0;  // per device: the shared-memory limit
    int dev = 0;
    const int rc = require_device(&dev);
    if (rc) return rc;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 64 || !(prepared >> dev & 1)) {
            const cudaError_t e = cudaFuncSetAttribute(short_kernel<OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kShortSmem));
            if (e != cudaSuccess) return cuda_fail(e, "short_kernel setup");
            if (dev < 64) prepared |= 1ull << dev;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(kShortThreads);
    cfg.dynamicSmemBytes = kShortSmem;
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
    const cudaError_t e = cudaLaunchKernelEx(&cfg, short_kernel<OUT>, maps, p, ctas);
    return e == cudaSuccess ? check_launch("short_kernel") : cuda_fail(e, "short_kernel launch");
}
// Q of `steps` steps from A, for k up to 128.
int core(const Matrix& A, const Matrix& q, int steps, int* failed, cudaStream_t st) {
    ShortMaps maps{};
    const int rc = operand_maps(maps.x, A, false);
    if (rc) return rc;
    ShortParams p{};
    p.k = static_cast<int>(A.rows);
    p.steps = steps;
    p.segments = 1;
    p.core = 1;
    p.failed = failed;
    p.x[0] = q.part[0];
    p.x[1] = q.part[1];
    p.ld = q.ld;
    return launch_short<kSplit>(maps, p, 1, st);
}
// All of it.
template <int OUT>
int whole(const Matrix& x, bool tall, int steps, int segments, const Result& res, const Factors* factors, cudaStream_t st) {
    ShortMaps maps{};
    const int rc = operand_maps(maps.x, x, false);
    if (rc) return rc;
    ShortParams p{};
    p.r = static_cast<int>(x.rows);
    p.d = static_cast<int>(x.cols);
    p.tall = tall;
    p.k = std::min(p.r, p.d);
    p.chunks = tiles(std::max(p.r, p.d), 128);
    p.steps = steps;
    p.segments = segments;
    p.factors = factors;
    p.failed = res.failed;
    p.x[0] = x.part[0];
    p.x[1] = x.part[1];
    p.ld = x.ld;
    p.result = res.out;
    p.ldr = res.ld;
    p.mask = res.mask;
    p.w_bf16 = res.w_bf16;
    p.decay = res.decay;
    p.step = res.step;
    return launch_short<OUT>(maps, p, (p.chunks + 1) / 2, st);
}

// O(U) to the result.
template <int OUT>
int orthogonalize(const Source& s, int steps, float eps, Result res, cudaStream_t st) {
    const bool tall = s.r > s.d;
    const long long k = std::min(s.r, s.d), ldx = up(s.d, 8), ldk = up(k, 8);
    const size_t x_bytes = up(2ll * s.r * ldx, 256), k_bytes = up(2ll * k * ldk, 256);
    const int segments = (steps + kSegment - 1) / kSegment;
    void* base = nullptr;
    const size_t partial_bytes = up(sizeof(double) * kNormBlocks, 256), factor_bytes = up(sizeof(Factors) * kMostSegments + sizeof(int), 256);
    int rc = scratch_alloc(&base, partial_bytes + factor_bytes + (segments > 1 ? 4 : 2) * x_bytes + 12 * k_bytes, st);
    if (rc) return rc;
    char* at = static_cast<char*>(base);
    double* partial = reinterpret_cast<double*>(at);
    at += partial_bytes;
    Factors* factors = reinterpret_cast<Factors*>(at);
    int* failed = res.failed = reinterpret_cast<int*>(factors + kMostSegments);
    at += factor_bytes;
    auto matrix = [&](long long rows, long long cols, long long ld, size_t bytes, int exp) {
        Matrix x{{reinterpret_cast<uint16_t*>(at), reinterpret_cast<uint16_t*>(at + bytes)}, rows, cols, ld, exp};
        at += 2 * bytes;
        return x;
    };
    Matrix x = matrix(s.r, s.d, ldx, x_bytes, kExpX), x2 = x;
    if (segments > 1) x2 = matrix(s.r, s.d, ldx, x_bytes, kExpX);
    Matrix A = matrix(k, k, ldk, k_bytes, kExpK), T = matrix(k, k, ldk, k_bytes, kExpK);
    Matrix P[2] = {matrix(k, k, ldk, k_bytes, kExpK), matrix(k, k, ldk, k_bytes, kExpK)};
    Matrix Q[2] = {matrix(k, k, ldk, k_bytes, kExpQ), matrix(k, k, ldk, k_bytes, kExpQ)};

    const long long units = static_cast<long long>(s.r) * ((s.d + 3) / 4);
    const unsigned blocks = static_cast<unsigned>(std::min<long long>((units + 255) / 256, kNormBlocks));
    norm_kernel<<<blocks, 256, 0, st>>>(s, partial);
    rc = check_launch("norm_kernel");
    if (!rc) {
        const cudaError_t e = launch_pdl(scale_kernel, dim3(blocks), dim3(256), 0, st, s, partial, static_cast<int>(blocks), eps, x.part[0], x.part[1], ldx, factors, failed, segments);
        rc = e == cudaSuccess ? check_launch("scale_kernel") : cuda_fail(e, "scale_kernel launch");
    }
    const bool small = k <= 128;
    if (!rc && small && std::max(s.r, s.d) <= 128 * kShortChunks) {
        rc = whole<OUT>(x, tall, steps, segments, res, factors, st);
        scratch_free(base, st);
        return rc;
    }
    for (int seg = 0; seg < segments && !rc; ++seg) {
        const int n = steps * (seg + 1) / segments - steps * seg / segments;
        const float* gram = &factors[seg].gram;
        rc = tall ? symmetric<true>(x, x, A, 1.0f, nullptr, 0, 0, nullptr, nullptr, failed, st, gram) : symmetric<false>(x, x, A, 1.0f, nullptr, 0, 0, nullptr, nullptr, failed, st, gram);
        Matrix q = P[0];
        if (!rc && small) {
            if (n > 1) q = Q[0];
            rc = core(A, q, n, failed, st);
        }
        for (int i = 0; i < n && !rc && !small; ++i) {
            const Matrix& p = P[i & 1];
            rc = symmetric<false>(A, A, p, kC, &A, kB, kA, nullptr, nullptr, failed, st);
            const Matrix& next = Q[i & 1];
            const bool last = i == n - 1;
            if (!rc && !last) rc = i ? symmetric<false>(p, A, T, 1.0f, nullptr, 0, 0, &q, &next, failed, st) : symmetric<false>(p, A, T, 1.0f, nullptr, 0, 0, nullptr, nullptr, failed, st);
            if (!rc && !last) rc = symmetric<false>(p, T, A, 1.0f, nullptr, 0, 0, nullptr, nullptr, failed, st);
            if (!rc && last && i) rc = symmetric<false>(p, q, next, 1.0f, nullptr, 0, 0, nullptr, nullptr, failed, st);
            if (i) q = next;
        }
        if (rc) break;
        if (seg < segments - 1) {
            rc = apply<kSplit>(tall, q, x, x2, res, factors + seg, st);
            std::swap(x, x2);
        } else {
            rc = apply<OUT>(tall, q, x, x, res, factors + seg, st);
        }
    }
    scratch_free(base, st);
    return rc;
}

int shift_of(int m) { return m == 1 ? 0 : m == 2 ? 1 : m == 4 ? 2 : m == 8 ? 3 : -1; }

int check_shape(const char* who, int r, int d, int steps, float eps) {
    if (r <= 0 || d <= 0) return fail(TB_ERR_ZERO_SIZE, "%s: empty matrix", who);
    if (r > 0x7FFFFFFF - 256 || d > 0x7FFFFFFF - 256) return fail(TB_ERR_SHAPE, "%s: %d x %d", who, r, d);
    if (std::min(r, d) > 32768) return fail(TB_ERR_CAPACITY, "%s: %d x %d: the shorter side ends at 32768", who, r, d);
    if (static_cast<long long>((r + 255) / 256) * ((d + 255) / 256) > 0x3FFFFFFFll) return fail(TB_ERR_CAPACITY, "%s: %d x %d", who, r, d);
    if (steps < 1 || steps > 32) return fail(TB_ERR_CONFIG, "%s: %d steps", who, steps);
    if (!(eps >= 0.0f && eps < INFINITY)) return fail(TB_ERR_CONFIG, "%s: eps %g", who, eps);
    return TB_OK;
}
bool misaligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == TB_F32 ? 4 : 2) != 0; }

}  // namespace

int take_error(cudaStream_t st) {
    int h = 0, zero = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&h, g_muon_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_muon_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    return e == cudaSuccess ? h : -1;
}

}  // namespace muon
}  // namespace tb

using namespace tb;

extern "C" int tb_orthogonalize(const void* x, int x_dtype, int64_t ldx, int r, int d, void* out, int out_dtype, int64_t ldo, int steps, float eps,
                                void* stream) {
    constexpr const char* who = "tb_orthogonalize";
    if (x_dtype != TB_F32 && x_dtype != TB_BF16) return fail(x_dtype == TB_F16 ? TB_ERR_UNSUPPORTED : TB_ERR_ARG, "%s: x of dtype %d", who, x_dtype);
    if (out_dtype != TB_BF16) return fail(out_dtype == TB_F16 || out_dtype == TB_F32 ? TB_ERR_UNSUPPORTED : TB_ERR_ARG, "%s: out of dtype %d", who, out_dtype);
    int rc = muon::check_shape(who, r, d, steps, eps);
    if (rc) return rc;
    if (!x || !out || muon::misaligned(x, x_dtype) || muon::misaligned(out, out_dtype)) return fail(TB_ERR_ARG, "%s: null or misaligned pointer", who);
    if (ldx < d || ldo < d) return fail(TB_ERR_ARG, "%s: a row stride below d", who);
    if ((rc = require_device(nullptr))) return rc;
    muon::Source s{};
    s.r = r;
    s.d = d;
    s.g = x;
    s.g_bf16 = x_dtype == TB_BF16;
    s.ldg = ldx;
    muon::Result res{};
    res.out = out;
    res.ld = ldo;
    return muon::orthogonalize<muon::kBf16>(s, steps, eps, res, static_cast<cudaStream_t>(stream));
}

extern "C" int tb_muon_step(const tb_muon_args* p, void* stream) {
    constexpr const char* who = "tb_muon_step";
    if (!p || p->struct_size != sizeof(tb_muon_args)) return fail(TB_ERR_ARG, "%s: null args or bad struct_size", who);
    if (p->g_dtype != TB_F32 && p->g_dtype != TB_BF16) return fail(p->g_dtype == TB_F16 ? TB_ERR_UNSUPPORTED : TB_ERR_ARG, "%s: gradient of dtype %d", who, p->g_dtype);
    if (p->w_dtype != TB_F32 && p->w_dtype != TB_BF16) return fail(p->w_dtype == TB_F16 ? TB_ERR_UNSUPPORTED : TB_ERR_ARG, "%s: weights of dtype %d", who, p->w_dtype);
    int rc = muon::check_shape(who, p->r, p->d, p->steps, p->eps);
    if (rc) return rc;
    if (!p->grad || !p->w || muon::misaligned(p->grad, p->g_dtype) || muon::misaligned(p->w, p->w_dtype) || muon::misaligned(p->momentum, TB_F32))
        return fail(TB_ERR_ARG, "%s: null or misaligned pointer", who);
    const int64_t ldg = p->ldg ? p->ldg : p->d, ldm = p->ldm ? p->ldm : p->d, ldw = p->ldw ? p->ldw : p->d;
    if (ldg < p->d || ldm < p->d || ldw < p->d) return fail(TB_ERR_ARG, "%s: a row stride below d", who);
    if (p->mask) {
        if (p->nm_m < 1) return fail(TB_ERR_CONFIG, "%s: a mask of groups of %d", who, p->nm_m);
        if (p->nm_m > 8) return fail(TB_ERR_UNSUPPORTED, "%s: M=%d > 8: masks hold one byte per group", who, p->nm_m);
        if (static_cast<int64_t>(p->r) * p->d % p->nm_m) return fail(TB_ERR_SHAPE, "%s: %d x %d is not a multiple of %d", who, p->r, p->d, p->nm_m);
    }
    for (float v : {p->beta, p->lr, p->weight_decay, p->scale})
        if (!(v > -INFINITY && v < INFINITY)) return fail(TB_ERR_CONFIG, "%s: a factor that is not finite", who);
    if ((rc = require_device(nullptr))) return rc;
    muon::Source s{};
    s.r = p->r;
    s.d = p->d;
    s.g = p->grad;
    s.g_bf16 = p->g_dtype == TB_BF16;
    s.ldg = ldg;
    s.m = p->momentum;
    s.ldm = ldm;
    s.beta = p->beta;
    s.nesterov = p->nesterov;
    s.mask = {p->mask, p->nm_m, muon::shift_of(p->nm_m)};
    muon::Result res{};
    res.out = p->w;
    res.ld = ldw;
    res.mask = s.mask;
    res.w_bf16 = p->w_dtype == TB_BF16;
    res.decay = static_cast<float>(1.0 - static_cast<double>(p->lr) * p->weight_decay);
    res.step = static_cast<float>(static_cast<double>(p->lr) * p->scale);
    return muon::orthogonalize<muon::kWeights>(s, p->steps, p->eps, res, static_cast<cudaStream_t>(stream));
}
