// Low-rank adapters of many requests beside a shared projection: forward and
// backward (contract in include/tb_kernels.h).
#include <algorithm>

#include "tb_act8.cuh"
#include "tb_runtime.h"
#include "tb_simple_gemm.cuh"

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
__device__ __forceinline__ float xhat(const View& ck, long long t, long long f) {
    return static_cast<float>(ck.codes[t * ck.ldq + f]) * act8::scale_f32(ck.exps[(t / act8::kBlock) * ck.lde + f]);
}

// u[t][k] = scale A x (mode 0), scale A xhat (mode 1) or scale B^T dy (mode 2); 0 without an adapter.
__global__ void skinny_kernel(const Args g, const int mode, float* __restrict__ u) {
    const long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    if (i >= g.n * g.rank) return;
    const long long t = i / g.rank;
    const int k = static_cast<int>(i % g.rank), a = adapter_of(g, t);
    float sum = 0.0f;
    if (a >= 0) {
        const bf16* A = g.a + (static_cast<long long>(a) * g.rank + k) * g.lda;
        const bf16* B = g.b + static_cast<long long>(a) * g.r * g.ldb + k;
        if (mode == 0) for (int c = 0; c < g.d; ++c) sum = fmaf(__bfloat162float(g.x[t * g.ldx + c]), __bfloat162float(A[c]), sum);
        if (mode == 1) for (int c = 0; c < g.d; ++c) sum = fmaf(xhat(g.x8, t, c), __bfloat162float(A[c]), sum);
        if (mode == 2) for (int o = 0; o < g.r; ++o) sum = fmaf(__bfloat162float(g.dy[t * g.lddy + o]), __bfloat162float(B[o * g.ldb]), sum);
        sum *= g.scale[a];
    }
    u[i] = sum;
}

struct ForwardOp {
    static constexpr bool kRowA = true, kRowB = false;
    Args g;
    const float* u;
    long long M, N;
    __device__ bool wanted(long long, long long) const { return true; }
    __device__ int first_unit(int) const { return 0; }
    __device__ int last_unit(int) const { return 1; }
    __device__ long long k_begin(int) const { return 0; }
    __device__ long long k_end(int) const { return g.d; }
    __device__ float a(long long m, long long k) const { return __bfloat162float(g.x[m * g.ldx + k]); }
    __device__ float b(long long k, long long n) const { return __bfloat162float(g.w[n * g.ldw + k]); }
    __device__ void store(int, long long t, long long o, float y) const {
        const int a = adapter_of(g, t);
        if (a >= 0)
            for (int k = 0; k < g.rank; ++k) y = fmaf(u[t * g.rank + k], __bfloat162float(g.b[(static_cast<long long>(a) * g.r + o) * g.ldb + k]), y);
        g.y[t * g.ldy + o] = __float2bfloat16_rn(y);
    }
};

struct InputGradOp {
    static constexpr bool kRowA = true, kRowB = true;
    Args g;
    const float* v;
    long long M, N;
    __device__ bool wanted(long long, long long) const { return true; }
    __device__ int first_unit(int) const { return 0; }
    __device__ int last_unit(int) const { return 1; }
    __device__ long long k_begin(int) const { return 0; }
    __device__ long long k_end(int) const { return g.r; }
    __device__ float a(long long m, long long k) const { return __bfloat162float(g.dy[m * g.lddy + k]); }
    __device__ float b(long long k, long long n) const { return __bfloat162float(g.w[k * g.ldw + n]); }
    __device__ void store(int, long long t, long long c, float x) const {
        const int a = adapter_of(g, t);
        if (a >= 0)
            for (int k = 0; k < g.rank; ++k) x = fmaf(v[t * g.rank + k], __bfloat162float(g.a[(static_cast<long long>(a) * g.rank + k) * g.lda + c]), x);
        g.dx[t * g.lddx + c] = __float2bfloat16_rn(x);
    }
};

// da[a][k][c] = sum v[t][k] xhat[t][c]  (blockIdx.z = a, blockIdx.y = k)
__global__ void grad_a_kernel(const Args g, const float* __restrict__ v) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x, k = blockIdx.y, a = blockIdx.z;
    if (c >= g.d) return;
    float sum = 0.0f;
    for (long long t = 0; t < g.n; ++t)
        if (adapter_of(g, t) == a) sum = fmaf(v[t * g.rank + k], xhat(g.x8, t, c), sum);
    g.da[(static_cast<long long>(a) * g.rank + k) * g.lda + c] = __float2bfloat16_rn(sum);
}
__global__ void grad_b_kernel(const Args g, const float* __restrict__ u) {
    const int o = blockIdx.x * blockDim.x + threadIdx.x, k = blockIdx.y, a = blockIdx.z;
    if (o >= g.r) return;
    float sum = 0.0f;
    for (long long t = 0; t < g.n; ++t)
        if (adapter_of(g, t) == a) sum = fmaf(u[t * g.rank + k], __bfloat162float(g.dy[t * g.lddy + o]), sum);
    g.db[(static_cast<long long>(a) * g.r + o) * g.ldb + k] = __float2bfloat16_rn(sum);
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
    float* u = nullptr;
    if (g.na) {
        if ((rc = scratch_alloc(reinterpret_cast<void**>(&u), g.n * g.rank * sizeof(float), st))) return rc;
        skinny_kernel<<<static_cast<unsigned>((g.n * g.rank + 255) / 256), 256, 0, st>>>(g, 0, u);
    }
    ForwardOp op{g, u, g.n, g.r};
    simple_gemm_kernel<<<dim3((g.r + 63) / 64, static_cast<unsigned>((g.n + 63) / 64)), 256, 0, st>>>(op);
    rc = check_launch("adapter forward");
    scratch_free(u, st);
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
    float *u = nullptr, *v = nullptr;
    if (g.na && g.n) {
        const size_t bytes = g.n * g.rank * sizeof(float);
        if ((rc = scratch_alloc(reinterpret_cast<void**>(&v), 2 * bytes, st))) return rc;
        u = v + g.n * g.rank;
        const unsigned grid = static_cast<unsigned>((g.n * g.rank + 255) / 256);
        skinny_kernel<<<grid, 256, 0, st>>>(g, 2, v);
        if (grads) skinny_kernel<<<grid, 256, 0, st>>>(g, 1, u);
    }
    if (g.dx && g.n) {
        InputGradOp op{g, v, g.n, g.d};
        simple_gemm_kernel<<<dim3((g.d + 63) / 64, static_cast<unsigned>((g.n + 63) / 64)), 256, 0, st>>>(op);
    }
    if (grads) {
        grad_a_kernel<<<dim3((g.d + 255) / 256, g.rank, g.na), 256, 0, st>>>(g, v);
        grad_b_kernel<<<dim3((g.r + 255) / 256, g.rank, g.na), 256, 0, st>>>(g, u);
    }
    rc = check_launch("adapter backward");
    scratch_free(v, st);
    return rc;
}
