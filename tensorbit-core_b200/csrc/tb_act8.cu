// 8-bit activation checkpoints and what a calibration pass makes of them:
// packing, reading back, weight gradients per sample, the Fisher EMA of those
// gradients, and X^T X for exact OBS (contract in include/tb_kernels.h).
#include <algorithm>

#include "tb_act8.cuh"
#include "tb_linear.cuh"
#include "tb_runtime.h"

namespace tb {
namespace act8 {

int check(const tb_act8* ck, const char* who, View* v) {
    if (!ck || ck->struct_size != sizeof(tb_act8)) return fail(TB_ERR_ARG, "%s: null checkpoint or bad struct_size", who);
    if (ck->d <= 0) return fail(TB_ERR_ZERO_SIZE, "%s: a checkpoint has at least one feature", who);
    if (ck->d > kMaxFeatures) return fail(TB_ERR_SHAPE, "%s: %d features", who, ck->d);
    if (ck->n < 0 || ck->n > 0x7FFFFFFFll - 64) return fail(TB_ERR_SHAPE, "%s: %lld tokens", who, static_cast<long long>(ck->n));
    if (ck->ldq < ck->d || ck->ldq % 16 || ck->lde < ck->d || ck->lde % 16)
        return fail(TB_ERR_ARG, "%s: ldq and lde must be multiples of 16 and at least d", who);
    if (ck->n > 0 && (!ck->codes || !ck->exps || reinterpret_cast<uintptr_t>(ck->codes) % 16 ||
                      reinterpret_cast<uintptr_t>(ck->exps) % 16))
        return fail(TB_ERR_ARG, "%s: codes and exps must be non-null and 16-byte aligned", who);
    *v = {ck->codes, ck->exps, ck->ldq, ck->lde, ck->n, ck->d};
    return TB_OK;
}

namespace {

// One block of 256 threads holds 128 tokens x 128 features in registers as they
// are stored, so X is read once: thread (row, col) has 8 consecutive features of
// 8 tokens.  16000 x 14336 BF16, a quarter of them padding that is not read: 113 us,
// 0.77 of the copy rate (126 us with the maxima a word each in shared memory, 138
// with five blocks an SM, which spills).  Bound by memory: the largest magnitudes are found on the values'
// own bits, and a code costs one multiply-add: x 2^(127-E) + 1.5 2^23 holds
// rint(x 2^(127-E)), ties to even, in its low bits, the first product being exact.
// (No padding, out of memory: BF16 113, F16 111, FP32 178 us, 0.93 to 0.98 of the copy
// rate; rows that do not start on 16 bytes, a value a load: 221, 221 and 246.)
constexpr int kFeat = 128, kRowsPass = 16, kPasses = kBlock / kRowsPass;

// Eight consecutive values as stored.
template <int DT>
struct Eight {
    uint32_t w[DT == TB_F32 ? 8 : 4];
    // value i's bits in FP32
    __device__ __forceinline__ float at(int i) const {
        if constexpr (DT == TB_F32) return __uint_as_float(w[i]);
        else if constexpr (DT == TB_BF16) return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
        else return __half2float(__ushort_as_half(static_cast<unsigned short>(w[i >> 1] >> (16 * (i & 1)))));
    }
};

template <int DT, bool VEC>
__device__ __forceinline__ Eight<DT> load8(const void* x, long long at, int valid) {
    Eight<DT> v{};
    if (VEC && valid >= 8) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(x) + at * (DT == TB_F32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < (DT == TB_F32 ? 2 : 1); ++i) {
            const uint4 q = __ldcs(p + i);
            v.w[4 * i] = q.x; v.w[4 * i + 1] = q.y; v.w[4 * i + 2] = q.z; v.w[4 * i + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= valid) continue;
            if constexpr (DT == TB_F32) v.w[i] = static_cast<const uint32_t*>(x)[at + i];
            else v.w[i >> 1] |= static_cast<uint32_t>(static_cast<const uint16_t*>(x)[at + i]) << (16 * (i & 1));
        }
    }
    return v;
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(256) pack_kernel(const View ck, const void* __restrict__ x, const long long ldx,
                                                   const uint8_t* __restrict__ keep) {
    constexpr int kWords = DT == TB_F32 ? 8 : 4;  // of eight values
    __shared__ alignas(16) uint32_t smax[kRowsPass][16 * kWords];
    __shared__ alignas(8) uint8_t exps[kFeat];
    const int col = threadIdx.x & 15, row = threadIdx.x >> 4;
    const int f0 = blockIdx.x * kFeat + col * 8;
    const int valid = ck.d - f0;  // features of this thread (may be <= 0 or > 8)
    const long long t0 = static_cast<long long>(blockIdx.y) * kBlock;
    bool kept[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const long long t = t0 + p * kRowsPass + row;
        kept[p] = t < ck.n && valid > 0 && (!keep || keep[t] != 0);
    }
    Eight<DT> v[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        v[p] = {};
        if (kept[p]) v[p] = load8<DT, VEC>(x, (t0 + p * kRowsPass + row) * ldx + f0, valid);
    }
    // (16-bit values: the magnitudes of two features to a word)
    uint32_t most[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
        most[i] = 0;
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            if constexpr (DT == TB_F32) most[i] = max(most[i], v[p].w[i] & 0x7FFFFFFFu);
            else most[i] = __vmaxu2(most[i], v[p].w[i] & 0x7FFF7FFFu);
        }
    }
#pragma unroll
    for (int i = 0; i < kWords; i += 4)
        *reinterpret_cast<uint4*>(&smax[row][col * kWords + i]) = make_uint4(most[i], most[i + 1], most[i + 2], most[i + 3]);
    __syncthreads();
    if (threadIdx.x < kFeat) {
        uint32_t m = 0;
        if constexpr (DT == TB_F32) {
#pragma unroll
            for (int r = 0; r < kRowsPass; ++r) m = max(m, smax[r][threadIdx.x]);
        } else {
#pragma unroll
            for (int r = 0; r < kRowsPass; ++r) m = __vmaxu2(m, smax[r][threadIdx.x >> 1]);
            m = threadIdx.x & 1 ? m >> 16 : m & 0xFFFFu;
            m = DT == TB_BF16 ? m << 16 : __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m)))) & 0x7FFFFFFFu;
        }
        const uint32_t e = exponent_of(m);
        const int f = blockIdx.x * kFeat + threadIdx.x;
        if (f < ck.d) ck.exps[blockIdx.y * ck.lde + f] = static_cast<uint8_t>(e);
        exps[threadIdx.x] = static_cast<uint8_t>(e);
    }
    __syncthreads();
    if (valid <= 0) return;
    float inv[8];
    const uint2 ew = *reinterpret_cast<const uint2*>(exps + col * 8);
    uint32_t dead = 0;  // bytes of features whose block holds a NaN or an infinity: codes 0
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t e = ((i < 4 ? ew.x : ew.y) >> (8 * (i & 3))) & 0xFFu;
        dead |= e == 255u ? 1u << i : 0u;
        inv[i] = e == 255u ? 0.0f : inverse_scale(e);
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const long long t = t0 + p * kRowsPass + row;
        if (t >= ck.n) break;
        uint32_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = __float_as_uint(fmaf(v[p].at(i), inv[i], 12582912.0f));
        if (dead) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (dead >> i & 1) c[i] = 0;
        }
        const uint32_t lo = prmt(prmt(c[0], c[1], 0x0040u), prmt(c[2], c[3], 0x0040u), 0x5410u);
        const uint32_t hi = prmt(prmt(c[4], c[5], 0x0040u), prmt(c[6], c[7], 0x0040u), 0x5410u);
        int8_t* out = ck.codes + t * ck.ldq + f0;
        if (valid >= 8) {
            *reinterpret_cast<uint2*>(out) = make_uint2(lo, hi);
        } else {
            for (int i = 0; i < valid; ++i) out[i] = static_cast<int8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
        }
    }
}

// The same tile; all codes are read before the first value is written.  (16000 x
// 14336 to BF16, behind the packing, part of the codes still in L2: 101 us, 1.03
// of the copy rate; 127 us row by row, 104 without the streaming stores.  Codes out of
// memory: BF16 and F16 113 us, 0.93 of the copy rate, FP32 233, 0.75; rows that do not
// start on 16 bytes are stored a value at a time: 633, 635 and 881 us, 0.17 to 0.20.)
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) unpack_kernel(const View ck, void* __restrict__ out, const long long ldo) {
    using T = typename Elem<DT>::T;
    const int col = threadIdx.x & 15, row = threadIdx.x >> 4;
    const int f0 = blockIdx.x * kFeat + col * 8;
    const int valid = ck.d - f0;
    if (valid <= 0) return;
    const long long t0 = static_cast<long long>(blockIdx.y) * kBlock;
    const uint2 ew = *reinterpret_cast<const uint2*>(ck.exps + blockIdx.y * ck.lde + f0);
    float s[8];
    uint32_t s2[4];
    scales8(ew, s2);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = scale_f32(((i < 4 ? ew.x : ew.y) >> (8 * (i & 3))) & 0xFFu);
    uint2 codes[kPasses];
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const long long t = t0 + p * kRowsPass + row;
        if (t < ck.n) codes[p] = __ldcs(reinterpret_cast<const uint2*>(ck.codes + t * ck.ldq + f0));
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
        const long long t = t0 + p * kRowsPass + row;
        if (t >= ck.n) break;
        const uint2 w = codes[p];
        alignas(16) T o[8];
        if constexpr (DT == TB_BF16) {
            *reinterpret_cast<uint4*>(o) = decode8(w, s2);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int q = static_cast<int8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
                o[i] = Elem<DT>::to(static_cast<float>(q) * s[i]);
            }
        }
        T* dst = static_cast<T*>(out) + t * ldo + f0;
        if (VEC && valid >= 8) {
            const uint4* src = reinterpret_cast<const uint4*>(o);
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) __stcs(reinterpret_cast<uint4*>(dst) + i, src[i]);
        } else {
            for (int i = 0; i < 8 && i < valid; ++i) dst[i] = o[i];
        }
    }
}

// dy as BF16 parts that add up to it exactly: the leading 8 bits, the next 8
// and the last (FP32: three, F16: two; BF16 is copied, to aligned rows).  The
// parts are cut off, not rounded, so the largest finite value stays finite.
// The last part of a value below 2^-110 can fall below BF16's smallest, 2^-133.
template <int DT, int PARTS>
__global__ void __launch_bounds__(256) split_kernel(const void* __restrict__ dy, const long long lddy, const long long n,
                                                    const int r, const bool vec, uint16_t* __restrict__ out,
                                                    const long long ldo) {
    const int groups = static_cast<int>(ldo / 4);
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n * groups; i += gridDim.x * 256ll) {
        const long long t = i / groups;
        const int c = static_cast<int>(i % groups) * 4;
        float v[4];
        if (vec && c + 4 <= r) {
            if constexpr (DT == TB_F32) {
                const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(dy) + t * lddy + c);
                v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(dy) + t * lddy + c);
                const uint16_t h[4] = {static_cast<uint16_t>(w.x), static_cast<uint16_t>(w.x >> 16), static_cast<uint16_t>(w.y), static_cast<uint16_t>(w.y >> 16)};
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = Elem<DT>::load(h, k);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = c + k < r ? Elem<DT>::load(dy, t * lddy + c + k) : 0.0f;
        }
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            uint16_t h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t bits = __float_as_uint(v[k]);
                h[k] = static_cast<uint16_t>(bits >> 16);
                if ((bits & 0x7FFFFFFFu) > 0x7F800000u) h[k] = 0x7FFFu;  // a NaN stays one
                v[k] = (bits & 0x7F800000u) == 0x7F800000u ? 0.0f : v[k] - __uint_as_float(bits & 0xFFFF0000u);
            }
            *reinterpret_cast<uint2*>(out + (p * n + t) * ldo + c) =
                make_uint2(h[0] | static_cast<uint32_t>(h[1]) << 16, h[2] | static_cast<uint32_t>(h[3]) << 16);
        }
    }
}

bool vectors(const void* p, long long ld, int esize) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld * esize) % 16 == 0;
}

int check_dy(const char* who, const void* dy, int dtype, int64_t lddy, int r, int64_t n, const int64_t* samples, int S) {
    if (dtype < TB_F32 || dtype > TB_BF16) return fail(TB_ERR_ARG, "%s: bad dy dtype %d", who, dtype);
    if (r <= 0) return fail(TB_ERR_ZERO_SIZE, "%s: r must be positive", who);
    if (r > kMaxFeatures) return fail(TB_ERR_SHAPE, "%s: %d rows of a gradient", who, r);
    if (S < 0 || S > 65535 || (!samples && S != 1))
        return fail(TB_ERR_ARG, "%s: S must be in 0..65535, and 1 where samples is NULL", who);
    if (n > 0 && S > 0 && (!dy || lddy < r)) return fail(TB_ERR_ARG, "%s: dy is null or lddy < r", who);
    return TB_OK;
}

// dy in the form that the tensor-core products read; *scratch is freed by the caller.
int prepare_dy(const View& ck, const void* dy, int dtype, int64_t lddy, int r, cudaStream_t st, linear::Parts* out,
               void** scratch) {
    *out = {dy, lddy, 1};
    if (ck.n == 0) return TB_OK;
    const bool vec16 = vectors(dy, lddy, dtype == TB_F32 ? 4 : 2);
    if (dtype == TB_BF16 && vec16) return TB_OK;
    const int parts = dtype == TB_F32 ? 3 : dtype == TB_F16 ? 2 : 1;
    const long long ld = (r + 7) / 8 * 8;
    int rc = scratch_alloc(scratch, static_cast<size_t>(parts) * ck.n * ld * 2, st);
    if (rc) return rc;
    uint16_t* p = static_cast<uint16_t*>(*scratch);
    *out = {p, ld, parts};
    const unsigned grid = static_cast<unsigned>(std::min<long long>((ck.n * (ld / 4) + 255) / 256, 148 * 16));
    if (dtype == TB_F32) split_kernel<TB_F32, 3><<<grid, 256, 0, st>>>(dy, lddy, ck.n, r, vec16, p, ld);
    else if (dtype == TB_F16) split_kernel<TB_F16, 2><<<grid, 256, 0, st>>>(dy, lddy, ck.n, r, vec16, p, ld);
    else split_kernel<TB_BF16, 1><<<grid, 256, 0, st>>>(dy, lddy, ck.n, r, vec16, p, ld);
    return check_launch("split_kernel");
}

}  // namespace

int unpack(const View& ck, void* out, int dtype, long long ldo, cudaStream_t st) {
    const long long blocks = (ck.n + kBlock - 1) / kBlock;
    for (long long b0 = 0; b0 < blocks; b0 += 65535) {
        const long long nb = std::min(blocks - b0, 65535ll), t0 = b0 * kBlock;
        const View v{ck.codes + t0 * ck.ldq, ck.exps + b0 * ck.lde, ck.ldq, ck.lde, ck.n - t0, ck.d};
        const dim3 grid((ck.d + kFeat - 1) / kFeat, static_cast<unsigned>(nb));
        void* op = static_cast<char*>(out) + t0 * ldo * (dtype == TB_F32 ? 4 : 2);
        const bool vec = vectors(out, ldo, dtype == TB_F32 ? 4 : 2);
        switch (dtype) {
        case TB_F32: vec ? unpack_kernel<TB_F32, true><<<grid, 256, 0, st>>>(v, op, ldo) : unpack_kernel<TB_F32, false><<<grid, 256, 0, st>>>(v, op, ldo); break;
        case TB_F16: vec ? unpack_kernel<TB_F16, true><<<grid, 256, 0, st>>>(v, op, ldo) : unpack_kernel<TB_F16, false><<<grid, 256, 0, st>>>(v, op, ldo); break;
        default: vec ? unpack_kernel<TB_BF16, true><<<grid, 256, 0, st>>>(v, op, ldo) : unpack_kernel<TB_BF16, false><<<grid, 256, 0, st>>>(v, op, ldo); break;
        }
    }
    return check_launch("unpack_kernel");
}

}  // namespace act8
}  // namespace tb

using namespace tb;
using namespace tb::act8;

extern "C" int tb_act8_pack(const tb_act8* ckp, const void* x, int dtype, int64_t ldx, const uint8_t* keep,
                            void* stream) {
    View ck;
    int rc = act8::check(ckp, "tb_act8_pack", &ck);
    if (rc) return rc;
    if (dtype < TB_F32 || dtype > TB_BF16) return fail(TB_ERR_ARG, "tb_act8_pack: bad dtype %d", dtype);
    if (ck.n == 0) return TB_OK;
    if (!x || ldx < ck.d) return fail(TB_ERR_ARG, "tb_act8_pack: x is null or ldx < d");
    if ((rc = require_device(nullptr))) return rc;
    const long long blocks = (ck.n + kBlock - 1) / kBlock;
    auto st = static_cast<cudaStream_t>(stream);
    // The grid's y extent ends at 65535 blocks of tokens: longer checkpoints take several launches.
    for (long long b0 = 0; b0 < blocks; b0 += 65535) {
        const long long nb = std::min(blocks - b0, 65535ll), t0 = b0 * kBlock;
        const View v{ck.codes + t0 * ck.ldq, ck.exps + b0 * ck.lde, ck.ldq, ck.lde, ck.n - t0, ck.d};
        const dim3 grid((ck.d + kFeat - 1) / kFeat, static_cast<unsigned>(nb));
        const void* xp = static_cast<const char*>(x) + t0 * ldx * (dtype == TB_F32 ? 4 : 2);
        const uint8_t* kp = keep ? keep + t0 : nullptr;
        const bool vec = vectors(x, ldx, dtype == TB_F32 ? 4 : 2);
        switch (dtype) {
        case TB_F32: vec ? pack_kernel<TB_F32, true><<<grid, 256, 0, st>>>(v, xp, ldx, kp) : pack_kernel<TB_F32, false><<<grid, 256, 0, st>>>(v, xp, ldx, kp); break;
        case TB_F16: vec ? pack_kernel<TB_F16, true><<<grid, 256, 0, st>>>(v, xp, ldx, kp) : pack_kernel<TB_F16, false><<<grid, 256, 0, st>>>(v, xp, ldx, kp); break;
        default: vec ? pack_kernel<TB_BF16, true><<<grid, 256, 0, st>>>(v, xp, ldx, kp) : pack_kernel<TB_BF16, false><<<grid, 256, 0, st>>>(v, xp, ldx, kp); break;
        }
    }
    return check_launch("pack_kernel");
}

extern "C" int tb_act8_unpack(const tb_act8* ckp, void* out, int dtype, int64_t ldo, void* stream) {
    View ck;
    int rc = act8::check(ckp, "tb_act8_unpack", &ck);
    if (rc) return rc;
    if (dtype < TB_F32 || dtype > TB_BF16) return fail(TB_ERR_ARG, "tb_act8_unpack: bad dtype %d", dtype);
    if (ck.n == 0) return TB_OK;
    if (!out || ldo < ck.d) return fail(TB_ERR_ARG, "tb_act8_unpack: out is null or ldo < d");
    if ((rc = require_device(nullptr))) return rc;
    return act8::unpack(ck, out, dtype, ldo, static_cast<cudaStream_t>(stream));
}

extern "C" int tb_act8_weight_grad(const tb_act8* ckp, const void* dy, int dy_dtype, int64_t lddy, int r,
                                   const int64_t* samples, int S, void* grads, int g_dtype, int64_t g_stride,
                                   void* stream) {
    View ck;
    int rc = act8::check(ckp, "tb_act8_weight_grad", &ck);
    if (!rc) rc = check_dy("tb_act8_weight_grad", dy, dy_dtype, lddy, r, ck.n, samples, S);
    if (rc) return rc;
    const long long rd = static_cast<long long>(r) * ck.d;
    if (g_dtype == TB_F16) return fail(TB_ERR_UNSUPPORTED, "tb_act8_weight_grad: gradients are TB_F32 or TB_BF16");
    if (g_dtype != TB_F32 && g_dtype != TB_BF16) return fail(TB_ERR_ARG, "tb_act8_weight_grad: bad gradient dtype %d", g_dtype);
    if (g_stride == 0) g_stride = rd;
    if (g_stride < rd) return fail(TB_ERR_SHAPE, "tb_act8_weight_grad: g_stride below r * d");
    if (S == 0) return TB_OK;
    if (!grads) return fail(TB_ERR_ARG, "tb_act8_weight_grad: null gradients");
    if ((rc = require_device(nullptr))) return rc;
    auto st = static_cast<cudaStream_t>(stream);
    linear::Parts parts{};
    void* scratch = nullptr;
    rc = prepare_dy(ck, dy, dy_dtype, lddy, r, st, &parts, &scratch);
    if (!rc) rc = linear::weight_grad(ck, parts, r, samples, S, grads, g_dtype, g_stride, st);
    scratch_free(scratch, st);
    return rc;
}

extern "C" int tb_act8_fisher(const tb_act8* ckp, const void* dy, int dy_dtype, int64_t lddy, int r,
                              const int64_t* samples, int S, double alpha, double beta, int first_step, float* fisher,
                              void* stream) {
    View ck;
    int rc = act8::check(ckp, "tb_act8_fisher", &ck);
    if (!rc) rc = check_dy("tb_act8_fisher", dy, dy_dtype, lddy, r, ck.n, samples, S);
    if (rc) return rc;
    if (S == 0) return TB_OK;
    if (!fisher) return fail(TB_ERR_ARG, "tb_act8_fisher: null Fisher state");
    if ((rc = require_device(nullptr))) return rc;
    auto st = static_cast<cudaStream_t>(stream);
    linear::Parts parts{};
    void* scratch = nullptr;
    rc = prepare_dy(ck, dy, dy_dtype, lddy, r, st, &parts, &scratch);
    if (!rc) rc = linear::fisher(ck, parts, r, samples, S, alpha, beta, first_step != 0, fisher, st);
    scratch_free(scratch, st);
    return rc;
}

extern "C" int tb_act8_hessian(const tb_act8* ckp, float scale, int accumulate, float* H, void* stream) {
    View ck;
    int rc = act8::check(ckp, "tb_act8_hessian", &ck);
    if (rc) return rc;
    if (!H) return fail(TB_ERR_ARG, "tb_act8_hessian: null H");
    // (The product's token indexes, rounded up to its K step of 128, are 32 bits wide.)
    if (ck.n > 0x7FFFFFFFll - 127) return fail(TB_ERR_SHAPE, "tb_act8_hessian: %lld tokens", static_cast<long long>(ck.n));
    if ((rc = require_device(nullptr))) return rc;
    return linear::hessian(ck, scale, accumulate != 0, H, static_cast<cudaStream_t>(stream));
}
