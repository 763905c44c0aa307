// Low-rank adapters of many requests beside a shared projection: forward and
// backward (contract in include/tb_kernels.h).
#include <algorithm>

#include "tb_act8.cuh"
#include "tb_linear.cuh"
#include "tb_runtime.h"

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

// The adapters that occur among 256 tokens, in order of first occurrence: the
// count, then their numbers.
__global__ void __launch_bounds__(256) list_kernel(const Args g, int32_t* __restrict__ lists) {
    __shared__ int who[256], count[8];
    const int i = threadIdx.x, lane = i & 31, warp = i >> 5;
    const long long t = blockIdx.x * 256ll + i;
    who[i] = t < g.n ? adapter_of(g, t) : -1;
    __syncthreads();
    bool first = who[i] >= 0;
    for (int j = 0; j < i && first; ++j) first = who[j] != who[i];
    const unsigned m = __ballot_sync(~0u, first);
    if (lane == 0) count[warp] = __popc(m);
    __syncthreads();
    int at = __popc(m & ((1u << lane) - 1)), total = 0;
    for (int w = 0; w < 8; ++w) {
        if (w < warp) at += count[w];
        total += count[w];
    }
    int32_t* out = lists + static_cast<long long>(blockIdx.x) * linear::kListPitch;
    if (i == 0) out[0] = total;
    if (first) out[1 + at] = who[i];
}

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

// One piece of scratch: the lists, u and v (freed through `lists`).  Empty without adapters or tokens.
struct Scratch {
    int32_t* lists;
    float *u, *v;
};
int make_scratch(const Args& g, bool both, cudaStream_t st, Scratch* s) {
    if (!g.na || !g.n) return TB_OK;
    const size_t list = ((g.n + 255) / 256 * linear::kListPitch * sizeof(int32_t) + 255) / 256 * 256;
    const size_t vals = (g.n * g.rank * sizeof(float) + 255) / 256 * 256;
    void* p = nullptr;
    const int rc = scratch_alloc(&p, list + (both ? 2 : 1) * vals, st);
    if (rc) return rc;
    s->lists = static_cast<int32_t*>(p);
    s->v = reinterpret_cast<float*>(static_cast<char*>(p) + list);
    s->u = both ? reinterpret_cast<float*>(reinterpret_cast<char*>(s->v) + vals) : s->v;
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
        skinny_kernel<<<static_cast<unsigned>((g.n * g.rank + 255) / 256), 256, 0, st>>>(g, 0, s.u);
        list_kernel<<<static_cast<unsigned>((g.n + 255) / 256), 256, 0, st>>>(g, s.lists);
        rc = check_launch("adapter down projection");
    }
    if (!rc) rc = linear::adapter_forward({g.n, g.r, g.d, g.x, g.ldx, g.w, g.ldw, g.y, g.ldy, g.who, s.lists, s.u, g.b, g.ldb, g.rank, g.na}, st);
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
        const unsigned grid = static_cast<unsigned>((g.n * g.rank + 255) / 256);
        skinny_kernel<<<grid, 256, 0, st>>>(g, 2, s.v);
        if (grads) skinny_kernel<<<grid, 256, 0, st>>>(g, 1, s.u);
        list_kernel<<<static_cast<unsigned>((g.n + 255) / 256), 256, 0, st>>>(g, s.lists);
        rc = check_launch("adapter down projection");
    }
    if (!rc && g.dx && g.n)
        rc = linear::adapter_input_grad({g.n, g.d, g.r, g.dy, g.lddy, g.w, g.ldw, g.dx, g.lddx, g.who, s.lists, s.v, g.a, g.lda, g.rank, g.na}, st);
    if (!rc && grads) {
        grad_a_kernel<<<dim3((g.d + 255) / 256, g.rank, g.na), 256, 0, st>>>(g, s.v);
        grad_b_kernel<<<dim3((g.r + 255) / 256, g.rank, g.na), 256, 0, st>>>(g, s.u);
        rc = check_launch("adapter gradients");
    }
    scratch_free(s.lists, st);
    return rc;
}
