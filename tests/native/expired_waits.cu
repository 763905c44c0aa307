// Products of the tensor-core skeletons whose loading thread leaves its last slice out where it is told to:
// the wait for that slice runs out, within its limit, and nothing else is missing.
#include "tb_split_product.cuh"

namespace {
using namespace tb::pair;

__device__ int g_error;

struct Params {
    int* failed;
    float* out;     // [m][n]
    int n, slices;
    int left_out;   // rank of the cluster whose last slice is not loaded, or -1
};
// out = A B^T of BF16, rows of A and B along K.
struct Plain {
    static constexpr bool kAMn = false, kBMn = false, kF16 = false, kMirror = false;
    static constexpr int kParts = 1, kGroup = 4;
    using Params = ::Params;
    static __device__ __forceinline__ int* error() { return &g_error; }
    static __device__ __forceinline__ int items(const Params& p) { return p.n / 256; }
    static __device__ __forceinline__ Work work(const Params& p, int item) {
        Work w{0, item, 0, p.slices, 0, -1};
        if (static_cast<int>(threadIdx.x >> 5) == kLoadWarp && static_cast<int>(cluster_rank()) == p.left_out) --w.slices;
        return w;
    }
    static __device__ __forceinline__ void finish(const Launch<Plain>& L, const Work& w, float (&acc)[128], uint8_t* buf, int row_in, int half, int lane) {
        const int col = w.tn * 256 + half * 128;
        store_rows<false>(buf, acc, L.p.out + static_cast<long long>(row_in) * L.p.n + col, L.p.n, 32, 128, lane);
    }
    // by clusters of four: every CTA has slices / 4, the told one's loading warp one fewer
    static __device__ __forceinline__ Work split_work(const Params& p, int tile) {
        Work w{0, tile, 0, p.slices, 0, -1};
        if (static_cast<int>(threadIdx.x >> 5) == 4 && static_cast<int>(cluster_rank()) == p.left_out) w.slices -= 4;
        return w;
    }
    static __device__ __forceinline__ uint4 fetch_quad(const Launch<Plain>&, int, int) { return make_uint4(0, 0, 0, 0); }
    static __device__ __forceinline__ void finish_quad(const Launch<Plain>& L, const Work&, int row, int col, const float4& v, const uint4&, uint4&) {
        *reinterpret_cast<float4*>(L.p.out + static_cast<long long>(row) * L.p.n + col) = v;
    }
};
}  // namespace

// a [256][64 slices], b [n][64 slices], out [256][n] (by clusters: [128][n]); n a multiple of 256, slices of 4.
extern "C" int expired_product(const void* a, const void* b, float* out, int* failed, int n, int slices, int clusters, int left_out, void* stream) {
    Launch<Plain> L{};
    L.p = {failed, out, n, slices, left_out};
    int rc = operand_map(&L.a[0], a, 256, 64ll * slices, 64ll * slices, false);
    if (!rc) rc = operand_map(&L.b[0][0], b, n, 64ll * slices, 64ll * slices, false);
    if (rc) return rc;
    const auto st = static_cast<cudaStream_t>(stream);
    if (!clusters) return launch_product(L, n / 256, st);
    SplitClusters known{};
    rc = split_setup<Plain>(&known);
    return rc ? rc : launch_split(L, n / 128, 4, st);
}
extern "C" int expired_error(int* out) {
    const int zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(out, g_error, sizeof(int));
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
    return static_cast<int>(e);
}
