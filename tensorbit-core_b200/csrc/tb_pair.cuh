// Building blocks of the persistent kernels whose CTA pairs (cta_group::2) own
// 256 x 256 output tiles: waits, operand descriptors, the ring of stages, reads of
// accumulators, and the way of results to memory through shared memory.
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "tb_runtime.h"
#include "tb_tcgen05.cuh"

namespace tb {
namespace pair {

using namespace tb::umma;

// Waits for the barrier phase `parity`, at most about two seconds of SM cycles.
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
constexpr long long kWaitCycles = 4000000000ll;
// A role that passes over work which needs nothing of it waits at once for the next
// that does.  Its limit grows with what lies between: so much for each slice (of
// about 2^10 cycles).  The TMA warp beside it, which takes every slice,
// has the plain limit and ends that wait if it gives up.
constexpr long long kPassedCycles = 1 << 14;
// False once that is over, or as soon as another role of the CTA has given up.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, long long passed = 0) {
    if (try_wait(bar, parity)) return true;
    const long long t0 = clock64(), limit = kWaitCycles + passed * kPassedCycles;
    while (clock64() - t0 < limit) {
        if (try_wait(bar, parity)) return true;
        if (abort_flag && *abort_flag) return false;
    }
    return false;
}

// Tells the roles of both CTAs that one of them has given up.
__device__ __forceinline__ void abort_pair(volatile int* abort_flag) {
    *abort_flag = 1;
    asm volatile(
        "{\n\t.reg .b32 a;\n\t"
        "mapa.shared::cluster.u32 a, %0, 0;\n\tst.shared::cluster.u32 [a], %1;\n\t"
        "mapa.shared::cluster.u32 a, %0, 1;\n\tst.shared::cluster.u32 [a], %1;\n\t}" ::"r"(smem_u32(const_cast<int*>(abort_flag))), "r"(1)
        : "memory");
}
// The issuing thread's way out: its MMAs are done when this returns, so that TMEM and their operands' places may be given
// back.  `bar` is for this alone: one that results wait for would pass an unfinished sum off as a finished one.
__device__ __forceinline__ void drain_pair(uint32_t bar) {
    commit_pair(bar);
    wait(bar, 0, nullptr);
}
__device__ __forceinline__ void drain_one(uint32_t bar) {
    mma_commit(bar);
    wait(bar, 0, nullptr);
}

// (An explicit .release.cluster here cost about 0.4 us per slice: 1235 against
// 675 us for the 7000 x 4096 x 14336 forward.)
__device__ __forceinline__ void arrive_even(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar & kPeerMask) : "memory");
}

// 128-byte-swizzle operand descriptors.  K-major: rows of M or N are 128 bytes of
// K, 8-row atoms 1024 bytes apart.  MN-major: rows of K are 128 bytes of M or N,
// 8-row atoms 1024 bytes apart along K, the next 128 bytes of M or N `kMnChunk`
// further.
constexpr int kMnChunk = 64 * 128;
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn) {
    const uint64_t lbo = mn ? kMnChunk >> 4 : 1;
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (lbo << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// Sixteen accumulator columns of this lane's row: the read, and the wait for all reads under way.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// Two lanes of a += v in packed FP32 (round to nearest).
__device__ __forceinline__ void add2(float& a0, float& a1, uint32_t v0, uint32_t v1) {
    asm("{\n\t.reg .b64 A, V;\n\tmov.b64 A, {%0, %1};\n\tmov.b64 V, {%2, %3};\n\t"
        "add.rn.f32x2 A, A, V;\n\tmov.b64 {%0, %1}, A;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "r"(v0), "r"(v1));
}

// A load that counts on the even CTA's barrier.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t even_bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(even_bar)
        : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A place in the ring of stages: its index and the parity of its current phase.
template <int STAGES>
struct Ring {
    int s = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++s == STAGES) {
            s = 0;
            phase ^= 1;
        }
    }
};

// ---- results: a lane holds COLS columns of its row, memory wants rows --------------
// They pass through shared memory in pieces of 32 rows x 128 bytes (32 FP32 or 64
// BF16 columns) with 128-byte swizzle: written by 16-byte units of a row a lane,
// read without conflicts by rows.  A piece leaves by TMA (gradients whose rows
// start on 16 bytes), as 16-byte units of whole rows, or, where rows do not start
// on 16 bytes or a piece is not whole, element by element, consecutive ones a
// store.  rows, cols: how many of the warp's rows, of a piece's columns, exist.
// (26 gradients of 14282 x 743, rows not on 16 bytes: 2417 us stored a row a lane, 320 so.)
constexpr int kPieceBytes = 4096;
template <bool BF16>
struct Piece {
    static constexpr int kCols = BF16 ? 64 : 32, kSize = BF16 ? 2 : 4;
};
template <bool BF16, int COLS>
__device__ __forceinline__ void fill_piece(uint8_t* buf, const float (&v)[COLS], int c, int lane) {
    uint8_t* row = buf + lane * 128;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        uint4 w;
        const float* x = v + c * Piece<BF16>::kCols + j * (Piece<BF16>::kCols / 8);
        if constexpr (BF16) w = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
        else w = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
        *reinterpret_cast<uint4*>(row + ((j ^ (lane & 7)) << 4)) = w;
    }
}
// Byte `at` of row r.
__device__ __forceinline__ int piece_at(int r, int at) { return r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15); }

template <bool BF16>
__device__ __noinline__ void store_piece(const uint8_t* buf, void* out, long long ld, int rows, int cols, int lane) {
    constexpr int kSize = Piece<BF16>::kSize;
    char* p = static_cast<char*>(out);
    const long long pitch = ld * kSize;
    const unsigned align = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p) | pitch);
    if (cols >= Piece<BF16>::kCols && align % 16 == 0) {
        const int sub = lane >> 3, unit = (lane & 7) * 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + sub;
            const uint4 w = *reinterpret_cast<const uint4*>(buf + piece_at(r, unit));
            if (r < rows) *reinterpret_cast<uint4*>(p + r * pitch + unit) = w;
        }
    } else if (!BF16 || align % 4 == 0) {  // a word a lane; a last odd BF16 column by itself
        const int at = 4 * lane, left = cols * kSize - at;
        if (left >= 4) {
#pragma unroll 16
            for (int r = 0; r < 32; ++r) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(buf + piece_at(r, at));
                if (r < rows) *reinterpret_cast<uint32_t*>(p + r * pitch + at) = w;
            }
        } else if (left == 2) {
#pragma unroll 1
            for (int r = 0; r < rows; ++r) *reinterpret_cast<uint16_t*>(p + r * pitch + at) = *reinterpret_cast<const uint16_t*>(buf + piece_at(r, at));
        }
    } else {
#pragma unroll 1
        for (int at = 2 * lane; at < 2 * min(cols, Piece<BF16>::kCols); at += 64) {  // (`cols` may go on behind the piece)
#pragma unroll 16
            for (int r = 0; r < 32; ++r) {
                const uint16_t w = *reinterpret_cast<const uint16_t*>(buf + piece_at(r, at));
                if (r < rows) *reinterpret_cast<uint16_t*>(p + r * pitch + at) = w;
            }
        }
    }
}
// All of the warp's pieces; `out` is its first row and column.  (A piece's store is a function of its
// own: inlined for every piece and kind of result, it cost the other roles 6 to 8 %.)
template <bool BF16, int COLS>
__device__ __forceinline__ void store_rows(uint8_t* buf, const float (&v)[COLS], void* out, long long ld, int rows, int cols, int lane) {
    if (rows <= 0) return;
#pragma unroll
    for (int c = 0; c < COLS / Piece<BF16>::kCols; ++c) {
        if (c * Piece<BF16>::kCols >= cols) break;
        __syncwarp();
        fill_piece<BF16>(buf, v, c, lane);
        __syncwarp();
        store_piece<BF16>(buf, static_cast<char*>(out) + c * 128, ld, rows, cols - c * Piece<BF16>::kCols, lane);
    }
}
// The same by TMA, as many pieces in flight as there are buffers, stored or (FP32) added to what is
// there: sixteen 4096 x 4096 gradients in 336 us, where straight from registers, 32 bytes of a row a
// lane, they took 400.
template <bool BF16, int PIECES, int COLS>
__device__ __forceinline__ void store_tma(const CUtensorMap* map, uint8_t* buf, const float (&v)[COLS], int col, int row0, int s, int N,
                                          bool add, int lane) {
#pragma unroll
    for (int c = 0; c < COLS / Piece<BF16>::kCols; ++c) {
        uint8_t* piece = buf + c % PIECES * kPieceBytes;
        asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PIECES - 1) : "memory");  // the buffer's last piece has left it
        __syncwarp();
        fill_piece<BF16>(piece, v, c, lane);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            const int x = col + c * Piece<BF16>::kCols;
            if (x < N && add)
                asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(reinterpret_cast<uint64_t>(map)),
                             "r"(x), "r"(row0), "r"(s), "r"(smem_u32(piece))
                             : "memory");
            else if (x < N)
                asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(reinterpret_cast<uint64_t>(map)),
                             "r"(x), "r"(row0), "r"(s), "r"(smem_u32(piece))
                             : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
}
// Reads a piece of FP32 rows: 32 columns of the lane's row.
__device__ __forceinline__ void load_piece(uint8_t* buf, float* v, const float* p, long long ld, int rows, int cols, int lane) {
    __syncwarp();
#pragma unroll 16
    for (int r = 0; r < 32; ++r) *reinterpret_cast<float*>(buf + piece_at(r, 4 * lane)) = r < rows && lane < cols ? p[r * ld + lane] : 0.0f;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 w = *reinterpret_cast<const float4*>(buf + piece_at(lane, 16 * j));
        v[4 * j] = w.x; v[4 * j + 1] = w.y; v[4 * j + 2] = w.z; v[4 * j + 3] = w.w;
    }
}

// f(c, x) for each 16 columns x of this lane's row of a finished accumulator, the
// next read under way meanwhile; the accumulator is given back before the last.
template <int COLS, class F>
__device__ __forceinline__ void read_accumulator(uint32_t from, uint32_t accempty, int lane, F&& f) {
    fence_after();
    uint32_t v[2][16];
    tmem_ld16(from, v[0]);
#pragma unroll
    for (int c = 0; c < COLS / 16; ++c) {
        tmem_wait16(v[c & 1]);
        if (c + 1 < COLS / 16) {
            tmem_ld16(from + static_cast<uint32_t>(16 * (c + 1)), v[(c + 1) & 1]);
        } else {
            fence_before();
            __syncwarp();
            if (lane == 0) arrive_even(accempty);
        }
        f(c, v[c & 1]);
    }
}

// Row-major [rows][cols] of `esize`-byte elements, boxes of box_cols x box_rows (128-byte swizzle or none).
inline int make_map(CUtensorMap* map, const void* base, int esize, long long cols, long long rows, long long ld, int box_cols,
             int box_rows, bool swizzle) {
    EncodeFn enc = encode_fn();
    if (!enc) return fail(TB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * esize};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = encode_tiled(enc, map, esize == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
                           const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? TB_OK : fail(TB_ERR_ARG, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
}

constexpr long long kPairs = 74;  // one CTA on each of the 148 SMs

// Results [samples][rows][cols] in rows of ld, as boxes of 32 rows x 128 bytes.
inline int make_out_map(CUtensorMap* map, void* base, bool bf16_out, long long cols, long long rows, long long samples, long long ld, long long stride) {
    EncodeFn enc = encode_fn();
    if (!enc) return fail(TB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const int esize = bf16_out ? 2 : 4;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(samples)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * esize, static_cast<cuuint64_t>(stride) * esize};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(128 / esize), 32, 1}, estr[3] = {1, 1, 1};
    const CUresult e = encode_tiled(enc, map, bf16_out ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, base, dims,
                           strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return e == CUDA_SUCCESS ? TB_OK : fail(TB_ERR_ARG, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(e));
}

inline int tiles(long long v, int t) { return static_cast<int>((v + t - 1) / t); }

}  // namespace pair
}  // namespace tb
