// Products of the calibration operators on tcgen05 tensor cores (sm_100a).
//
// One persistent kernel skeleton, instantiated per mode.  A pair of CTAs
// (cta_group::2) owns a 256 x NB output tile: each CTA holds its 128 rows of A
// and NB/2 of the B columns of a K slice in shared memory, and its 128 x NB
// half of the accumulator in TMEM.  Roles of a CTA's 16 warps:
//   warp 12      TMA loads of K slices into a ring of stages;
//   warps 8-11   (and 14-15) "prepare" stages that do not arrive as operands: decode int8
//                codes to BF16, zero what lies behind a sample's end, or build
//                the operands of an adapter; then tell the even CTA;
//   warp 13      (even CTA) issues tcgen05.mma for both CTAs;
//   warps 0-7    take finished accumulators out of TMEM and store results.
// The accumulator is double buffered, so the next sums run while a tile is
// stored.  The tensor core's own additions truncate: the modes with FP32
// results accumulate short groups of K in TMEM and add those into FP32
// registers with round to nearest.  That needs 128 accumulators a thread, so
// these modes move registers from the other roles to the epilogue's warps.
//
// Modes:
//   kGrad    G_s = dY_s^T Xhat_s: A = dY (M-major by TMA), B = decoded codes
//   kFisher  the same with the Fisher state in registers: a sum of the samples' g^2
//            with the factors that the EMA's steps give them, in order
//   kGradX, kFisherX  the same two with B = Xhat in BF16, decoded beforehand
//   kHess    Xhat^T Xhat on int8 tensor cores: the codes of a block of 128
//            tokens multiply exactly into int32, and the block's two
//            power-of-two scales enter when its sum is added in FP32
//   kFwd     X W^T, kDx: dY W, with one extra K slice of 64 for every 32 ranks
//            of an adapter present in the tile: [u_hi | u_lo] of its tokens
//            (zero for the others) times [E | E]
// Every wait is bounded; on expiry the kernel records an error and leaves.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "tb_device.cuh"
#include "tb_linear.cuh"
#include "tb_runtime.h"
#include "tb_tcgen05.cuh"

namespace tb {
namespace linear {
namespace {

using namespace tb::umma;
using bf16 = __nv_bfloat16;

enum Mode { kGrad = 0, kFisher = 1, kHess = 2, kFwd = 3, kDx = 4, kGradX = 5, kFisherX = 6 };
__host__ __device__ constexpr int kind(int mode) { return mode == kGradX ? kGrad : mode == kFisherX ? kFisher : mode; }

__device__ int g_linear_error;

constexpr int kThreads = 512;
constexpr int kEpiWarps = 8, kPrepWarp = 8, kTmaWarp = 12, kMmaWarp = 13;
// Codes are decoded by six warps (8-11, 14, 15).  (All six a slice: 313 us for
// sixteen gradients of a q_proj, where two groups of three, every second slice
// each, took 332.  Groups that skip a barrier's phases may not wait on its parity
// in any case: TMA loads can complete out of order.)
constexpr int kDecodeWarps = 6;

constexpr int kGradGroup = 8;  // slices that kGrad sums in TMEM

template <int MODE>
struct Cfg {
    static constexpr bool kCodes = MODE == kGrad || MODE == kFisher;   // B decoded from codes here
    static constexpr bool kTails = MODE == kGradX || MODE == kFisherX; // B in BF16; a sample's last slice is cut off in shared memory
    static constexpr bool kSamples = kCodes || kTails;
    static constexpr bool kAdapter = MODE == kFwd || MODE == kDx;
    static constexpr bool kPromote = !kAdapter;
    static constexpr int NB = 256;                                     // columns of a pair's tile
    static constexpr int kAcc = 512 / NB;                              // accumulators in TMEM
    static constexpr int kCols = NB / 2;                               // columns of an epilogue warp, and of a CTA's B
    // K slices summed in TMEM before they are added in FP32: 512 tokens (kGrad), one block of codes
    // (kHess), all (16-bit results).  kFisher: see kDirect.
    static constexpr int kGroup = kind(MODE) == kGrad ? kGradGroup : kind(MODE) == kFisher ? 4 : MODE == kHess ? 1 : 1 << 30;
    static constexpr int kA = 16384;                                   // 128 rows x 128 bytes of K (or 128 int8 tokens)
    static constexpr int kB = kCols * 128;
    static constexpr int kRaw = kCodes ? 64 * kCols : 0;               // codes of the slice
    static constexpr int kExps = kCodes ? kCols : 0;                   // exponents of its block
    static constexpr int kStage = kA + kB + kRaw;
    // Arrivals that make a stage ready: the decoding warps of each CTA (codes), the even CTA's
    // TMA thread (bytes of both CTAs), or either (an adapter's or a sample's last slice is the prepare warps')
    static constexpr int kReady = kCodes ? 2 * kDecodeWarps : kAdapter || kTails ? 9 : 1;
    static constexpr int kStages = kCodes ? 4 : MODE == kFisherX ? 5 : 6;
    // Behind the stages: pieces of results on their way out, the exponents of each stage
    static constexpr int kPieces = MODE == kGrad ? 2 : 1, kOutWarp = kPieces * 4096;
    static constexpr int kOut = kEpiWarps * kOutWarp;
    static constexpr int kFactors = kind(MODE) == kFisher ? 1024 : 0;        // samples whose factor is held in shared memory
    static constexpr int kExtra = kOut + kStages * kExps + kFactors * 4;
    static constexpr size_t kSmem = static_cast<size_t>(kStages) * kStage + kExtra + 1024 + 512;
    static_assert(kSmem <= 232448, "shared memory of a block");
};

struct Params {
    long long M, N;
    int K, n;  // K of the adapter products; tokens
    int tiles_m, tiles_n, items;
    // checkpoint and samples
    const uint8_t* exps;
    long long lde;
    const int64_t* samples;
    int S, parts;
    // results
    void* out;
    long long ldo, out_stride;
    int out_bf16, out_tma;
    double alpha, beta;
    float scale, decay;  // decay: beta^S
    int first, accumulate;
    AdapterProduct ad;
    // The first `whole` units are items of their own; each of the `tail` units behind them is `splits` items,
    // shares of its K (kFisher: of its samples), whose sums go to `part`, [splits][tail][256][256] FP32.
    int whole, tail, splits;
    float* part;
};
constexpr int kPartTile = 256 * 256;

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
__device__ __forceinline__ void give_up(volatile int* abort_flag) {
    *abort_flag = 1;
    atomicExch(&g_linear_error, 1);
}
// (An explicit .release.cluster here cost about 0.4 us per slice: 1235 against
// 675 us for the 7000 x 4096 x 14336 forward.)
__device__ __forceinline__ void arrive_even(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar & kPeerMask) : "memory");
}
// Sets bits of a word of both CTAs, before what this warp tells anyone next.
__device__ __forceinline__ void set_pair(uint32_t* word, uint32_t bits) {
    asm volatile(
        "{\n\t.reg .b32 a;\n\t"
        "mapa.shared::cluster.u32 a, %0, 0;\n\tred.relaxed.cluster.shared::cluster.or.b32 [a], %1;\n\t"
        "mapa.shared::cluster.u32 a, %0, 1;\n\tred.relaxed.cluster.shared::cluster.or.b32 [a], %1;\n\t"
        "fence.acq_rel.cluster;\n\t}" ::"r"(smem_u32(word)), "r"(bits)
        : "memory");
}
template <int MODE>
__device__ __forceinline__ void mma_step(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (MODE == kHess)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}"
            ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u));
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}"
            ::"r"(tmem), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u));
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
// Eight columns of each of two accumulators, waited for.
__device__ __forceinline__ void tmem_ld8x2(uint32_t from0, uint32_t from1, uint32_t (&x)[8], uint32_t (&y)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=&r"(x[0]), "=&r"(x[1]), "=&r"(x[2]), "=&r"(x[3]), "=&r"(x[4]), "=&r"(x[5]), "=&r"(x[6]), "=&r"(x[7]),
          "=&r"(y[0]), "=&r"(y[1]), "=&r"(y[2]), "=&r"(y[3]), "=&r"(y[4]), "=&r"(y[5]), "=&r"(y[6]), "=&r"(y[7])
        : "r"(from0), "r"(from1)
        : "memory");
}
// Two lanes of a += v, and of a += (m * row + base) * col, in packed FP32 (round to nearest).
__device__ __forceinline__ void add2(float& a0, float& a1, uint32_t v0, uint32_t v1) {
    asm("{\n\t.reg .b64 A, V;\n\tmov.b64 A, {%0, %1};\n\tmov.b64 V, {%2, %3};\n\t"
        "add.rn.f32x2 A, A, V;\n\tmov.b64 {%0, %1}, A;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "r"(v0), "r"(v1));
}
__device__ __forceinline__ void scale_add2(float& a0, float& a1, uint32_t m0, uint32_t m1, float row, float base, float c0, float c1) {
    asm("{\n\t.reg .b64 A, M, R, B, C;\n\tmov.b64 A, {%0, %1};\n\tmov.b64 M, {%2, %3};\n\t"
        "mov.b64 R, {%4, %4};\n\tmov.b64 B, {%5, %5};\n\tmov.b64 C, {%6, %7};\n\t"
        "fma.rn.f32x2 M, M, R, B;\n\tfma.rn.f32x2 A, M, C, A;\n\tmov.b64 {%0, %1}, A;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "r"(m0), "r"(m1), "f"(row), "f"(base), "f"(c0), "f"(c1));
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

// kFisher has the Fisher state in the registers that would add a sample's groups
// up.  A sample of at most kDirect slices over all parts comes out of TMEM whole:
// one sum where that is at most kGradGroup slices of tokens, as in a group of kGrad,
// else (more than 512 tokens of BF16 dy) two, in both accumulators, added as they are
// read.  Each of a slice's four steps cuts off less than 2^-23 of the sum so far; the
// parts before the leading one count little.  (Of g^2, 2-norm against float64, 1000
// tokens with terms of one sign: 1.5e-6 in one sum, 5e-7 in two, 2e-7 where signs
// are mixed.)  For a longer one the state waits in its place in memory, once, while
// groups of 256 tokens are added in FP32.
constexpr int kDirect = 16;

// ---- the walk over work items, units (one sum each) and K slices that every role shares ----
struct Tile {
    int tm, tn;
    int s;              // sample
    int q, splits;      // share
    int slot;           // its place in `part`, or -1
};
struct Unit {
    int lo, hi;         // K range (samples: lo rounded down to a whole slice,
    int begin;          // begin the first token)
    int slices;         // K slices of one part
    int first, total;   // the share's slices, counted over the parts
    int group;          // slices summed in one accumulator
    int extra;          // adapters: slices behind those of K,
    int rslices;        // so many for each adapter
    const int32_t* list;
};

template <int MODE>
__device__ __forceinline__ Tile tile_of(const Params& P, int item) {
    Tile t{0, 0, 0, 0, 1, -1};
    int unit = item;
    if (item >= P.whole) {
        t.slot = item - P.whole;
        t.q = t.slot / P.tail;
        t.splits = P.splits;
        unit = P.whole + t.slot % P.tail;
    }
    if constexpr (MODE == kHess) {  // tiles on or below the diagonal, row by row
        int tm = static_cast<int>((sqrtf(8.0f * static_cast<float>(unit) + 1.0f) - 1.0f) * 0.5f);
        while (tm * (tm + 1) / 2 > unit) --tm;
        while ((tm + 1) * (tm + 2) / 2 <= unit) ++tm;
        t.tm = tm;
        t.tn = unit - tm * (tm + 1) / 2;
    } else {
        const int tiles = P.tiles_m * P.tiles_n, i = kind(MODE) == kGrad ? unit % tiles : unit;
        if constexpr (kind(MODE) == kGrad) t.s = unit / tiles;
        // bands of 8 tile rows, column by column inside, so that concurrent tiles share operands in L2
        const int band = i / (8 * P.tiles_n), in = i % (8 * P.tiles_n);
        const int rows = min(8, P.tiles_m - 8 * band);
        t.tm = 8 * band + in % rows;
        t.tn = in / rows;
    }
    return t;
}

// The share `q` of `all` slices.
__device__ __forceinline__ int share_begin(int all, int q, int splits) {
    return static_cast<int>(static_cast<unsigned long long>(all) * static_cast<unsigned>(q) / static_cast<unsigned>(splits));
}
template <int MODE>
__device__ __forceinline__ Unit unit_of(const Params& P, const Tile& t, int s) {
    Unit u{0, P.K, 0, 0, 0, 0, Cfg<MODE>::kGroup, 0, 1, nullptr};
    if constexpr (Cfg<MODE>::kSamples) {
        u.hi = P.n;
        if (P.samples) {
            const long long b = __ldg(P.samples + 2 * s), e = __ldg(P.samples + 2 * s + 1);
            u.begin = static_cast<int>(min(max(b, 0ll), static_cast<long long>(P.n)));
            u.hi = static_cast<int>(max(min(e, static_cast<long long>(P.n)), static_cast<long long>(u.begin)));
            u.lo = Cfg<MODE>::kCodes ? u.begin & ~63 : u.begin;  // (codes: a slice then lies in one block)
        }
        u.slices = u.hi > u.begin ? (u.hi - u.lo + 63) / 64 : 0;
        u.total = u.slices * P.parts;
        if (kind(MODE) == kFisher && u.total <= kDirect) u.group = u.slices <= kGradGroup ? kDirect : kGradGroup;
        if (kind(MODE) != kFisher && t.splits > 1) {
            u.first = share_begin(u.slices * P.parts, t.q, t.splits);
            u.total = share_begin(u.slices * P.parts, t.q + 1, t.splits) - u.first;
        }
    } else {  // a share begins at its own `lo`
        constexpr int kStep = MODE == kHess ? 128 : 64;
        u.total = u.slices = ((MODE == kHess ? P.n : P.K) + kStep - 1) / kStep;
        if (t.splits > 1) {
            const int all = u.slices, first = share_begin(all, t.q, t.splits);
            u.lo = first * kStep;
            u.total = u.slices = share_begin(all, t.q + 1, t.splits) - first;
        }
        if constexpr (Cfg<MODE>::kAdapter) {
            if (P.ad.lists && t.q == t.splits - 1) {
                u.list = P.ad.lists + static_cast<long long>(t.tm) * kListPitch;
                u.rslices = (P.ad.rank + 31) / 32;
                u.extra = __ldg(u.list) * u.rslices;
            }
        }
    }
    return u;
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

// Calls f(tile, unit) for every unit of this pair's items until it returns false.
template <int MODE, class F>
__device__ __forceinline__ bool for_units(const Params& P, F&& f) {
    for (int item = blockIdx.x >> 1; item < P.items; item += gridDim.x >> 1) {
        const Tile t = tile_of<MODE>(P, item);
        if constexpr (kind(MODE) == kFisher) {
            for (int s = share_begin(P.S, t.q, t.splits), end = share_begin(P.S, t.q + 1, t.splits); s < end; ++s)
                if (!f(t, unit_of<MODE>(P, t, s))) return false;
        } else {
            if (!f(t, unit_of<MODE>(P, t, t.s))) return false;
        }
    }
    return true;
}
// Calls f(part, i, count) for the unit's runs of slices i .. i + count - 1 of one
// part of K until it returns false.
template <class F>
__device__ __forceinline__ bool for_runs(const Unit& u, F&& f) {
    int part = 0, i = 0;
    if (u.first) {
        part = u.first / u.slices;
        i = u.first % u.slices;
    }
    for (int left = u.total; left > 0; ++part, i = 0) {
        const int run = min(left, u.slices - i);
        if (!f(part, i, run)) return false;
        left -= run;
    }
    return true;
}

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

// An adapter's second factor enters the product for all tokens of a tile, times
// zero for those of other adapters; zero times an infinity or a NaN is not zero.
// Such values are ones of their sign in the operand, which notes their adapter, and
// the epilogue adds their own terms to the results of the adapter's own tokens.
// (Beside those a one's does not count; an infinity of the token, which with a zero
// would be a NaN, keeps its sign.)
__device__ __forceinline__ uint32_t finite_pair(uint32_t w, bool& odd) {
    if ((w & 0x7F80u) == 0x7F80u) {
        w = (w & 0xFFFF8000u) | 0x3F80u;
        odd = true;
    }
    if ((w & 0x7F800000u) == 0x7F800000u) {
        w = (w & 0x8000FFFFu) | 0x3F800000u;
        odd = true;
    }
    return w;
}
// The bit that stands for adapter a among those noted (for others too, whose factors then are looked through).
__device__ __forceinline__ uint32_t odd_bit(int a) { return 1u << (a & 31); }

// Result i of this lane's token, feature o + i, is at v[32 i].  A lane looks one
// feature's ranks through for all tokens of an adapter.  (8000 x 4096 x 4096 forward,
// four adapters of rank 64, 268 us: with one value an infinity 10991 looked through
// token by token and 365 so, with a whole adapter NaN 12089 and 437.)
template <int MODE>
__device__ __noinline__ void add_odd_columns(const AdapterProduct& p, const uint32_t* noted, float* v, long long row0, int rows, long long o,
                                             int cols, int lane) {
    const long long t = row0 + lane;
    int own = lane < rows ? __ldg(p.who + t) : -1;  // this lane's adapter if it is one of those noted, else -1
    if (own < 0 || own >= p.na || !(*const_cast<const volatile uint32_t*>(noted) & odd_bit(own))) own = -1;
    const long long step = MODE == kFwd ? 1 : p.lde;  // from rank to rank
    for (unsigned left = __ballot_sync(~0u, own >= 0); left;) {
        const int a = __shfl_sync(~0u, own, __ffs(left) - 1);
        left &= ~__ballot_sync(~0u, own == a);
        const uint16_t* e = reinterpret_cast<const uint16_t*>(p.e) +
                            (MODE == kFwd ? (static_cast<long long>(a) * p.N + o) * p.lde : static_cast<long long>(a) * p.rank * p.lde + o);
        bool nan = false, inf = false;
        if (lane < cols) {
            const uint16_t* mine = e + (MODE == kFwd ? lane * p.lde : lane);
#pragma unroll 8
            for (int j = 0; j < p.rank; ++j) {
                const uint32_t magnitude = __ldg(mine + j * step) & 0x7FFFu;
                nan |= magnitude > 0x7F80u;
                inf |= magnitude == 0x7F80u;
            }
        }
        const unsigned nans = __ballot_sync(~0u, nan), infs = __ballot_sync(~0u, inf) & ~nans;
        if (own != a) continue;
        for (unsigned m = nans; m; m &= m - 1) v[32 * (__ffs(m) - 1)] = __uint_as_float(0x7FFFFFFFu);
        for (unsigned m = infs; m; m &= m - 1) {
            const int i = __ffs(m) - 1;
            float s = v[32 * i];
            for (int j = 0; j < p.rank && s == s; ++j) {
                const uint32_t x = __ldg(e + (MODE == kFwd ? i * p.lde : i) + j * step);
                if ((x & 0x7FFFu) == 0x7F80u) s = fmaf(p.u[t * p.rank + j], __uint_as_float(x << 16), s);
            }
            v[32 * i] = s;
        }
    }
}
template <int MODE>
__device__ __forceinline__ void add_odd_terms(const AdapterProduct& p, const uint32_t* noted, uint8_t* buf, float (&v)[64], long long row0,
                                              long long col, int rows, int cols, int lane) {
    float* x = reinterpret_cast<float*>(buf) + lane;  // column i of this lane's row at 32 i
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 32; ++i) x[32 * i] = v[32 * h + i];
        add_odd_columns<MODE>(p, noted, x, row0, rows, col + 32 * h, min(32, cols - 32 * h), lane);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[32 * h + i] = x[32 * i];
    }
    __syncwarp();
}

// Ranks r0.. of adapter `a` as one K slice of 64 (thread pt of 128): A is the
// tile's tokens' u as two BF16 parts, zero unless the adapter is their own; B is
// the adapter's second factor, twice, as finite_pair has it.  What it needs is fetched
// ahead: into registers before the stage is free.  (7000 x 4096 x 14336 forward
// with one adapter in most tiles: 584 us fetched once the stage was free, 560 so.)
template <int MODE>
struct AdapterSlice {
    int nr;          // ranks
    float u[32];     // of this thread's token
    uint4 e[4];      // kFwd: a row of b; kDx: 8 features of every eighth rank's row of a

    __device__ __forceinline__ void fetch(const AdapterProduct& p, int own, int a, int r0, long long m0, int n0, int pt) {
        nr = min(32, p.rank - r0);
        const bool mine = own == a;
        const float* up = p.u + (m0 + pt) * p.rank + r0;
        if (p.rank % 4 == 0) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float4 f = mine && 4 * q < nr ? *reinterpret_cast<const float4*>(up + 4 * q) : make_float4(0, 0, 0, 0);
                u[4 * q] = f.x; u[4 * q + 1] = f.y; u[4 * q + 2] = f.z; u[4 * q + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] = mine && j < nr ? up[j] : 0.0f;
        }
        const int c = pt & 15, f = n0 + 8 * c;
        const long long o = n0 + pt;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = (pt >> 4) + 8 * i;
            e[i] = make_uint4(0, 0, 0, 0);
            if constexpr (MODE == kFwd) {
                if (o < p.N && 8 * i < nr) e[i] = __ldg(reinterpret_cast<const uint4*>(p.e + (static_cast<long long>(a) * p.N + o) * p.lde + r0 + 8 * i));
            } else {
                if (f < p.N && k < nr) e[i] = __ldg(reinterpret_cast<const uint4*>(p.e + (static_cast<long long>(a) * p.rank + r0 + k) * p.lde + f));
            }
        }
    }
    // True if the factor has values that are not finite.
    __device__ __forceinline__ bool build(uint8_t* sa, uint8_t* sb, int pt) const {
        bool odd = false;
        uint8_t* arow = sa + pt * 128;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split_pair(u[8 * q + 2 * i], u[8 * q + 2 * i + 1], hi[i], lo[i]);
            *reinterpret_cast<uint4*>(arow + ((q ^ (pt & 7)) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(arow + (((q + 4) ^ (pt & 7)) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        const int c = pt & 15;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[4] = {e[i].x, e[i].y, e[i].z, e[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = 8 * i + 2 * j;
                if (MODE == kFwd) w[j] = k + 1 < nr ? w[j] : k < nr ? w[j] & 0xFFFFu : 0u;
                w[j] = finite_pair(w[j], odd);
            }
            const uint4 v = make_uint4(w[0], w[1], w[2], w[3]);
            if constexpr (MODE == kFwd) {  // ranks 8 i .. of the output column's row
                uint8_t* brow = sb + pt * 128;
                *reinterpret_cast<uint4*>(brow + ((i ^ (pt & 7)) << 4)) = v;
                *reinterpret_cast<uint4*>(brow + (((i + 4) ^ (pt & 7)) << 4)) = v;
            } else {  // the ranks along K
                const int k = (pt >> 4) + 8 * i, unit = ((c & 7) ^ (k & 7)) << 4;
                uint8_t* dst = sb + (c >> 3) * kMnChunk;
                *reinterpret_cast<uint4*>(dst + k * 128 + unit) = v;
                *reinterpret_cast<uint4*>(dst + (k + 32) * 128 + unit) = v;
            }
        }
        return odd;
    }
};

// What the square of sample s's gradient counts for in the state after all S steps
// F <- beta F + alpha (1 - beta) g^2, the first of which, on no state, is alpha g^2.
__device__ __forceinline__ float fisher_factor(const Params& P, int s) {
    return static_cast<float>(P.alpha * (P.first && s == 0 ? 1.0 : 1.0 - P.beta) * pow(P.beta, static_cast<double>(P.S - 1 - s)));
}
// Two lanes of F += (w g) g in packed FP32.
__device__ __forceinline__ void square_add2(float& f0, float& f1, uint64_t w2, float g0, float g1) {
    asm("{\n\t.reg .b64 F, G, T;\n\tmov.b64 F, {%0, %1};\n\tmov.b64 G, {%3, %4};\n\t"
        "mul.rn.f32x2 T, %2, G;\n\tfma.rn.f32x2 F, T, G, F;\n\tmov.b64 {%0, %1}, F;\n\t}"
        : "+f"(f0), "+f"(f1)
        : "l"(w2), "f"(g0), "f"(g1));
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

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
linear_kernel(const __grid_constant__ CUtensorMap tA, const __grid_constant__ CUtensorMap tB,
              const __grid_constant__ CUtensorMap tE, const __grid_constant__ CUtensorMap tO,
              const __grid_constant__ CUtensorMap tP, const __grid_constant__ Params P) {
    using C = Cfg<MODE>;
    constexpr int NB = C::NB, kStages = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    // (by offset, so that the compiler still knows it for shared memory)
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* out_buf = smem + kStages * C::kStage;
    uint8_t* exps_buf = out_buf + C::kOut;
    float* factors = reinterpret_cast<float*>(exps_buf + kStages * C::kExps);
    uint64_t* full = reinterpret_cast<uint64_t*>(out_buf + C::kExtra);
    uint64_t* ready = full + kStages;     // (even CTA) stage prepared by both CTAs
    uint64_t* empty = ready + kStages;    // stage read by the MMAs
    uint64_t* accfull = empty + kStages;      // [kAcc] accumulator finished
    uint64_t* accempty = accfull + C::kAcc;   // [kAcc] (even CTA) accumulator taken by both CTAs
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accempty + C::kAcc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    uint32_t* odd_flag = tmem_slot + 2;  // a bit for each adapter whose factor had values that are not finite (set in both CTAs, never reset)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank());

    if (threadIdx.x == kTmaWarp * 32 && P.n > 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tA)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tB)) : "memory");
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&ready[s]), C::kReady);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        for (int b = 0; b < C::kAcc; ++b) {
            mbar_init(smem_u32(&accfull[b]), 1);
            mbar_init(smem_u32(&accempty[b]), 2 * kEpiWarps);
        }
        *abort_flag = 0;
        *odd_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if constexpr (kind(MODE) == kFisher)
        for (int s = threadIdx.x; s < min(P.S, C::kFactors); s += kThreads) factors[s] = fisher_factor(P, s);
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    fence_before();
    cluster_sync_all();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    auto stage_a = [&](int s) { return smem_u32(smem + s * C::kStage); };
    auto stage_b = [&](int s) { return smem_u32(smem + s * C::kStage + C::kA); };

    // Register shares of the promoting modes: 8 warps x 200 + 8 warps x 56 = the launch's 16 x 128.
    if (warp < kEpiWarps) {
        if constexpr (C::kPromote) asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        constexpr int COLS = C::kCols;
        const int quad = warp & 3, half = warp >> 2;
        const int row_in = rank * 128 + quad * 32;
        uint8_t* buf = out_buf + warp * C::kOutWarp;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(quad * 32) << 16) + static_cast<uint32_t>(half * COLS);
        bool ok = true;
        Ring<C::kAcc> ac;
        for (int item = blockIdx.x >> 1; item < P.items && ok; item += gridDim.x >> 1) {
            const Tile t = tile_of<MODE>(P, item);
            const long long row0 = static_cast<long long>(t.tm) * 256 + row_in, row = row0 + lane;
            const long long col = static_cast<long long>(t.tn) * NB + half * COLS;
            const int rows = static_cast<int>(min(32ll, P.M - row0)), cols = static_cast<int>(min(static_cast<long long>(COLS), P.N - col));
            if constexpr (C::kAdapter) {
                const int b = ac.s;
                if (!wait(smem_u32(&accfull[b]), ac.phase, abort_flag)) { ok = false; break; }
                fence_after();
                ac.next();
                // (the adapters' slices are the last share's)
                const bool odd = P.ad.lists && t.q == t.splits - 1 && __any_sync(~0u, *const_cast<volatile uint32_t*>(odd_flag));
#pragma unroll 1
                for (int c = 0; c < COLS && c < cols; c += 64) {
                    float v[64];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x[32];
                        tmem_ld32(lane_base + static_cast<uint32_t>(b * NB + c + 32 * h), x);
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[32 * h + i] = x[i];
                    }
                    const int left = cols - c;
                    if (odd) add_odd_terms<MODE>(P.ad, odd_flag, buf, v, row0, col + c, rows, left, lane);
                    if (t.slot >= 0) {
                        store_rows<false>(buf, v, P.part + static_cast<long long>(t.slot) * kPartTile + row_in * 256 + half * COLS + c, 256, rows, left, lane);
                        continue;
                    }
                    store_rows<true>(buf, v, static_cast<bf16*>(P.out) + row0 * P.ldo + col + c, P.ldo, rows, left, lane);
                }
                fence_before();
                __syncwarp();
                if (lane == 0) arrive_even(smem_u32(&accempty[b]));
            } else if constexpr (kind(MODE) == kFisher) {
                // A share is a state of its own, begun at 0.
                float* out = t.slot < 0 ? static_cast<float*>(P.out) + row0 * P.ldo + col
                                        : P.part + static_cast<long long>(t.slot) * kPartTile + row_in * 256 + half * COLS;
                const int ld = t.slot < 0 ? static_cast<int>(P.ldo) : 256;
                float F[COLS];
                if (P.first || t.slot >= 0) {
#pragma unroll
                    for (int i = 0; i < COLS; ++i) F[i] = 0.0f;
                } else {
#pragma unroll
                    for (int c = 0; c < COLS / 32; ++c) load_piece(buf, F + 32 * c, out + 32 * c, ld, rows, cols - 32 * c, lane);
#pragma unroll
                    for (int i = 0; i < COLS; ++i) F[i] *= P.decay;
                }
                const int s_end = share_begin(P.S, t.q + 1, t.splits);
                for (int s = share_begin(P.S, t.q, t.splits); s < s_end && ok; ++s) {
                    const Unit u = unit_of<MODE>(P, t, s);
                    if (u.total == 0) continue;  // no tokens: g = 0
                    const float factor = s < C::kFactors ? factors[s] : fisher_factor(P, s);
                    const uint64_t factor2 = pack2(factor, factor);
                    if (u.total > kDirect) {
                        store_rows<false>(buf, F, out, ld, rows, cols, lane);
#pragma unroll
                        for (int i = 0; i < COLS; ++i) F[i] = 0.0f;
                        for (int left = u.total; left > 0 && ok; left -= u.group) {
                            const int b = ac.s;
                            if (!wait(smem_u32(&accfull[b]), ac.phase, abort_flag)) { ok = false; break; }
                            ac.next();
                            read_accumulator<COLS>(lane_base + static_cast<uint32_t>(b * NB), smem_u32(&accempty[b]), lane, [&](int c, uint32_t (&x)[16]) {
#pragma unroll
                                for (int i = 0; i < 16; i += 2) add2(F[c * 16 + i], F[c * 16 + i + 1], x[i], x[i + 1]);
                            });
                        }
#pragma unroll
                        for (int c = 0; c < COLS / 32; ++c) {
                            float old[32];
                            load_piece(buf, old, out + 32 * c, ld, rows, cols - 32 * c, lane);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                square_add2(old[i], old[i + 1], factor2, F[32 * c + i], F[32 * c + i + 1]);
                                F[32 * c + i] = old[i];
                                F[32 * c + i + 1] = old[i + 1];
                            }
                        }
                    } else if (u.total > u.group) {  // two sums, one in each accumulator
                        const int b = ac.s;
                        if (!wait(smem_u32(&accfull[b]), ac.phase, abort_flag)) { ok = false; break; }
                        ac.next();
                        if (!wait(smem_u32(&accfull[b ^ 1]), ac.phase, abort_flag)) { ok = false; break; }
                        ac.next();
                        fence_after();
#pragma unroll
                        for (int c = 0; c < COLS / 8; ++c) {
                            uint32_t x[8], y[8];
                            tmem_ld8x2(lane_base + static_cast<uint32_t>(b * NB + 8 * c), lane_base + static_cast<uint32_t>((b ^ 1) * NB + 8 * c), x, y);
                            if (c + 1 == COLS / 8) {
                                fence_before();
                                __syncwarp();
                                if (lane == 0) {
                                    arrive_even(smem_u32(&accempty[0]));
                                    arrive_even(smem_u32(&accempty[1]));
                                }
                            }
#pragma unroll
                            for (int i = 0; i < 8; i += 2) {
                                float g0 = __uint_as_float(x[i]), g1 = __uint_as_float(x[i + 1]);
                                add2(g0, g1, y[i], y[i + 1]);
                                square_add2(F[c * 8 + i], F[c * 8 + i + 1], factor2, g0, g1);
                            }
                        }
                    } else {
                        const int b = ac.s;
                        if (!wait(smem_u32(&accfull[b]), ac.phase, abort_flag)) { ok = false; break; }
                        ac.next();
                        read_accumulator<COLS>(lane_base + static_cast<uint32_t>(b * NB), smem_u32(&accempty[b]), lane, [&](int c, uint32_t (&x)[16]) {
#pragma unroll
                            for (int i = 0; i < 16; i += 2)
                                square_add2(F[c * 16 + i], F[c * 16 + i + 1], factor2, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                        });
                    }
                }
                if (ok) {
                    store_rows<false>(buf, F, out, ld, rows, cols, lane);
                }
            } else {
                {
                    const int s = t.s;
                    const Unit u = unit_of<MODE>(P, t, s);
                    const int groups = (u.total + u.group - 1) / u.group;
                    float acc[COLS];
#pragma unroll
                    for (int i = 0; i < COLS; ++i) acc[i] = 0.0f;
                    float* scol = reinterpret_cast<float*>(buf);  // kHess: the columns' scales of two groups, until results leave
                    // kHess: exponent bytes of this lane's row and of four of the warp's columns, fetched one
                    // group ahead and not touched before (bytes behind the last column go to columns not stored)
                    uint8_t er = 0;
                    uint32_t ec = 0;
                    auto load_exps = [&](int g) {
                        if constexpr (MODE == kHess) {
                            const uint8_t* e = P.exps + (u.lo / 128 + g) * P.lde;
                            if (row < P.M) er = __ldg(e + row);
                            if (col + 4 * lane < P.N) ec = __ldg(reinterpret_cast<const uint32_t*>(e + col + 4 * lane));
                        }
                    };
                    if (groups > 0) load_exps(0);
                    if constexpr (MODE == kHess) {  // the last results have left `scol`
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __syncwarp();
                    }
                    for (int g = 0; g < groups; ++g) {
                        float srow = 0.0f;
                        if constexpr (MODE == kHess) {
                            srow = act8::scale_f32(er);
                            const float4 f = make_float4(act8::scale_f32(ec & 0xFF), act8::scale_f32((ec >> 8) & 0xFF),
                                                         act8::scale_f32((ec >> 16) & 0xFF), act8::scale_f32(ec >> 24));
                            __syncwarp();
                            *reinterpret_cast<float4*>(scol + (g & 1) * COLS + 4 * lane) = f;
                            __syncwarp();
                            if (g + 1 < groups) load_exps(g + 1);
                        }
                        const int b = ac.s;
                        if (!wait(smem_u32(&accfull[b]), ac.phase, abort_flag)) { ok = false; break; }
                        ac.next();
                        read_accumulator<COLS>(lane_base + static_cast<uint32_t>(b * NB), smem_u32(&accempty[b]), lane, [&](int c, uint32_t (&x)[16]) {
                            if constexpr (MODE == kHess) {
                                // |block sum| <= 128 * 127^2 < 2^22: as the low bits of 1.5 * 2^23 it is an
                                // exact FP32 value, and subtracting that base times the row's power of two too
                                const float base = -12582912.0f * srow;
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    const float4 sc = *reinterpret_cast<const float4*>(scol + (g & 1) * COLS + c * 16 + 4 * q);
                                    float* to = acc + c * 16 + 4 * q;
                                    scale_add2(to[0], to[1], 0x4B400000u + x[4 * q], 0x4B400000u + x[4 * q + 1], srow, base, sc.x, sc.y);
                                    scale_add2(to[2], to[3], 0x4B400000u + x[4 * q + 2], 0x4B400000u + x[4 * q + 3], srow, base, sc.z, sc.w);
                                }
                            } else {
#pragma unroll
                                for (int i = 0; i < 16; i += 2) add2(acc[c * 16 + i], acc[c * 16 + i + 1], x[i], x[i + 1]);
                            }
                        });
                    }
                    if (!ok) break;
                    {
                        if constexpr (MODE == kHess) {
#pragma unroll
                            for (int i = 0; i < COLS; ++i) acc[i] *= P.scale;
                        }
                        // kHess: only 128 x 128 tiles on or below the diagonal
                        const bool wanted = rows > 0 && cols > 0 && (kind(MODE) == kGrad || col / 128 <= row0 / 128);
                        if (t.slot >= 0) {
                            if (wanted) store_tma<false, C::kPieces>(&tP, buf, acc, half * COLS, row_in, t.slot, 256, false, lane);
                        } else if (MODE == kHess || P.out_tma) {
                            if (!wanted) continue;
                            if (kind(MODE) == kGrad && P.out_bf16) store_tma<true, C::kPieces>(&tO, buf, acc, static_cast<int>(col), static_cast<int>(row0), t.s, static_cast<int>(P.N), false, lane);
                            else store_tma<false, C::kPieces>(&tO, buf, acc, static_cast<int>(col), static_cast<int>(row0), t.s, static_cast<int>(P.N), MODE == kHess && P.accumulate, lane);
                        } else if constexpr (kind(MODE) == kGrad) {
                            const long long at = t.s * P.out_stride + row0 * P.ldo + col;
                            if (P.out_bf16) store_rows<true>(buf, acc, static_cast<bf16*>(P.out) + at, P.ldo, rows, cols, lane);
                            else store_rows<false>(buf, acc, static_cast<float*>(P.out) + at, P.ldo, rows, cols, lane);
                        }
                    }
                }
            }
        }
        if constexpr (kind(MODE) == kGrad || MODE == kHess) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if (!ok) give_up(abort_flag);
    } else {
        if constexpr (C::kPromote) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == kTmaWarp) {
            if (lane == 0) {
                // (This loop and the MMA warp's bound the products: 60 cycles more a slice are 5 % of their time.)
                Ring<kStages> at;
                uint32_t tails = 0, tailed = 0;  // a bit per stage: parity of its cut slices, whether it had any
                const uint32_t full0 = smem_u32(full), ready0 = smem_u32(ready) & kPeerMask, empty0 = smem_u32(empty);
                const bool done = for_units<MODE>(P, [&](const Tile& t, const Unit& u) {
                    const int m0 = t.tm * 256 + rank * 128, n0 = t.tn * NB + rank * C::kCols;
                    const bool ok = for_runs(u, [&](int part, int i, int count) {
                        constexpr int kStep = MODE == kHess ? 128 : 64;
                        int k = u.lo + i * kStep;
                        // parts with fewer leading bits first: the large ones are then truncated least often
                        const int above = C::kSamples ? (P.parts - 1 - part) * P.n : 0;
#pragma unroll 1
                        for (; count > 0; --count, k += kStep, at.next()) {
                            const uint32_t a = stage_a(0) + at.s * C::kStage, b = a + C::kA;
                            if (!wait(empty0 + 8 * at.s, at.phase ^ 1, abort_flag)) return false;  // (the first round passes at once)
                            if constexpr (C::kCodes) {
                                const uint32_t bar = full0 + 8 * at.s;
                                mbar_expect_tx(bar, C::kA + C::kRaw + C::kExps);
                                tma_load_2d(a, &tA, m0, above + k, bar);
                                tma_load_2d(a + kMnChunk, &tA, m0 + 64, above + k, bar);
                                tma_load_2d(b + C::kB, &tB, n0, k, bar);
                                tma_load_2d(smem_u32(exps_buf) + at.s * C::kExps, &tE, n0, k >> 7, bar);
                            } else if (C::kTails && k + 64 > u.hi) {  // the sample ends in this slice: the prepare warps cut it off
                                const uint32_t bar = full0 + 8 * at.s;
                                if (rank == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(ready0 + 8 * at.s) : "memory");
                                mbar_expect_tx(bar, C::kA + C::kB);
                                tma_load_2d(a, &tA, m0, above + k, bar);
                                tma_load_2d(a + kMnChunk, &tA, m0 + 64, above + k, bar);
                                tma_load_2d(b, &tB, n0, k, bar);
                                tma_load_2d(b + kMnChunk, &tB, n0 + 64, k, bar);
                                tails ^= 1u << at.s;
                                tailed |= 1u << at.s;
                            } else {
                                const uint32_t bar = ready0 + 8 * at.s;
                                if (rank == 0) {
                                    if (C::kAdapter || C::kTails) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 8;" ::"r"(bar) : "memory");
                                    mbar_expect_tx(bar, 2 * (C::kA + C::kB));
                                }
                                if constexpr (MODE == kHess) {
                                    tma_load_pair(a, &tA, m0, k, bar);
                                } else if constexpr (C::kTails) {
                                    tma_load_pair(a, &tA, m0, above + k, bar);
                                    tma_load_pair(a + kMnChunk, &tA, m0 + 64, above + k, bar);
                                } else {
                                    tma_load_pair(a, &tA, k, m0, bar);
                                }
                                if constexpr (MODE == kFwd) {
                                    tma_load_pair(b, &tB, k, n0, bar);
                                } else {
                                    tma_load_pair(b, &tB, n0, k, bar);
                                    if constexpr (MODE == kDx || C::kTails) tma_load_pair(b + kMnChunk, &tB, n0 + 64, k, bar);
                                }
                            }
                        }
                        return true;
                    });
                    if (!ok) return false;
                    for (int x = 0; C::kAdapter && x < u.extra; ++x, at.next()) {  // the prepare warps fill these stages
                        if (!wait(empty0 + 8 * at.s, at.phase ^ 1, abort_flag)) return false;
                        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(full0 + 8 * at.s) : "memory");
                        if (rank == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(ready0 + 8 * at.s) : "memory");
                    }
                    return true;
                });
                if (!done) {
                    give_up(abort_flag);
                    // Loads in flight, each stage's last phase waited for within a limit (the odd CTA's may count
                    // on the even one's barrier).  A stage never used answers at once.
                    for (int i = 0; i < kStages && (C::kCodes || rank == 0); ++i) {
                        const bool used = i < at.s || at.phase;
                        if (used) wait(smem_u32(C::kCodes ? &full[i] : &ready[i]), i < at.s ? at.phase : at.phase ^ 1, nullptr);
                    }
                    for (int i = 0; C::kTails && i < kStages; ++i)
                        if (tailed >> i & 1) wait(smem_u32(&full[i]), (tails >> i & 1) ^ 1, nullptr);
                }
            }
            __syncwarp();
        } else if (warp == kMmaWarp) {
            if (lane == 0 && rank == 0) {
                constexpr bool kAmn = !C::kAdapter, kBmn = MODE != kFwd;
                constexpr uint32_t kIdesc = ((MODE == kHess ? 2u : 1u) << 4) | (1u << 7) | (1u << 10) |
                                            (kAmn ? 1u << 15 : 0u) | (kBmn ? 1u << 16 : 0u) | ((NB >> 3) << 17) | (16u << 24);
                // descriptor steps of one MMA: K-major 32 bytes along a row; MN-major 16 (int8: 32) rows
                constexpr uint64_t kStepMn = (MODE == kHess ? 32 : 16) * 128 >> 4;
                constexpr uint64_t kStepA = kAmn ? kStepMn : 2, kStepB = kBmn ? kStepMn : 2;
                Ring<kStages> at;
                Ring<C::kAcc> ac;
                const uint64_t a_desc = operand_desc(stage_a(0), kAmn), b_desc = operand_desc(stage_b(0), kBmn);
                const uint32_t ready0 = smem_u32(ready), empty0 = smem_u32(empty);
                const bool done = for_units<MODE>(P, [&](const Tile&, const Unit& u) {
                    for (int left = u.total + u.extra; left > 0;) {  // a group of slices sums in one accumulator
                        const uint32_t d = tmem + static_cast<uint32_t>(ac.s * NB);
                        int n = min(left, u.group);
                        left -= n;
                        if (!wait(smem_u32(&accempty[ac.s]), ac.phase ^ 1, abort_flag)) return false;
                        uint32_t more = 0;
#pragma unroll 1
                        for (; n > 0; --n, at.next()) {
                            const uint64_t a0 = a_desc + at.s * (C::kStage >> 4), b0 = b_desc + at.s * (C::kStage >> 4);
                            if (!wait(ready0 + 8 * at.s, at.phase, abort_flag)) return false;
                            fence_after();
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) {
                                mma_step<MODE>(d, a0 + kk * kStepA, b0 + kk * kStepB, kIdesc, more);
                                more = 1;
                            }
                            commit_pair(empty0 + 8 * at.s);
                        }
                        commit_pair(smem_u32(&accfull[ac.s]));
                        ac.next();
                    }
                    return true;
                });
                if (!done) {
                    give_up(abort_flag);
                    for (int b = 0; b < C::kAcc; ++b) commit_pair(smem_u32(&accfull[b]));  // releases the waiting epilogues
                }
            }
            __syncwarp();
        } else if (C::kCodes) {
            // 8 consecutive features (one 16-byte unit of the operand) of every kRowStep-th token
            constexpr int kUnits = C::kCols / 8, kRowStep = 32 * kDecodeWarps / kUnits, kSteps = (64 + kRowStep - 1) / kRowStep;
            const int pt = (warp < kTmaWarp ? warp - kPrepWarp : warp - kMmaWarp + 3) * 32 + lane, pc = pt % kUnits, pr = pt / kUnits;
            Ring<kStages> at;
            auto slice = [&](const Unit& u, int i, int s, uint32_t phase) {
                // the slice's tokens first .. last - 1 are the sample's
                const int k0 = u.lo + i * 64, first = max(0, u.begin - k0), last = min(64, u.hi - k0);
                if (!wait(smem_u32(&full[s]), phase, abort_flag)) return false;
                uint8_t* stage = smem + s * C::kStage;
                const uint8_t* raw = stage + C::kA + C::kB;
                uint32_t scale[4];
                act8::scales8(*reinterpret_cast<const uint2*>(exps_buf + s * C::kExps + pc * 8), scale);
                uint8_t* dst = stage + C::kA + (pc >> 3) * kMnChunk;
                uint2 w[kSteps];
#pragma unroll
                for (int q = 0; q < kSteps; ++q)
                    if (pr + q * kRowStep < 64) w[q] = *reinterpret_cast<const uint2*>(raw + (pr + q * kRowStep) * C::kCols + pc * 8);
                if (first > 0 || last < 64) {
#pragma unroll
                    for (int q = 0; q < kSteps; ++q)
                        if (pr + q * kRowStep < first || pr + q * kRowStep >= last) w[q] = make_uint2(0, 0);
                }
#pragma unroll
                for (int q = 0; q < kSteps; ++q) {
                    const int k = pr + q * kRowStep;
                    if (k < 64) *reinterpret_cast<uint4*>(dst + k * 128 + (((pc & 7) ^ (k & 7)) << 4)) = act8::decode8(w[q], scale);
                }
                // the other tokens: dY may hold anything there.  (Their codes are zero now; a block that holds a
                // NaN is infinitely scaled, but then it is NaN for the sample's tokens in it too.)
                for (int q = pt; q < (first + 64 - last) * 16; q += 32 * kDecodeWarps) {
                    const int r = q >> 4, k = r < first ? r : last + r - first;
                    *reinterpret_cast<uint4*>(stage + (q & 1) * kMnChunk + k * 128 + ((q >> 1) & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive_even(smem_u32(&ready[s]));
                return true;
            };
            const bool done = for_units<MODE>(P, [&](const Tile&, const Unit& u) {
                return for_runs(u, [&](int, int i, int count) {
#pragma unroll 1
                    for (; count > 0; --count, ++i, at.next())
                        if (!slice(u, i, at.s, at.phase)) return false;
                    return true;
                });
            });
            if (!done) give_up(abort_flag);
        } else if (C::kTails && warp >= kPrepWarp && warp < kTmaWarp) {
            // Zeros for the tokens behind the sample's end in both operands (either may hold anything there).
            const int pt = threadIdx.x - kPrepWarp * 32;
            int it = 0, waited = 0;  // slices so far, and at the last wait
            uint32_t phase = 0;  // a bit per stage, for its cut slices only
            const bool done = for_units<MODE>(P, [&](const Tile&, const Unit& u) {
                return for_runs(u, [&](int, int i, int count) {
                    it += count;
                    const int last = u.hi - u.lo - (u.slices - 1) * 64;
                    if (i + count < u.slices || last == 64) return true;
                    const int s = (it - 1) % kStages;
                    if (!wait(smem_u32(&full[s]), (phase >> s) & 1, abort_flag, it - waited)) return false;
                    waited = it;
                    phase ^= 1u << s;
                    uint8_t* stage = smem + s * C::kStage;  // two chunks of A, two of B, rows of 128 bytes
                    for (int q = pt; q < (64 - last) * 32; q += 128)
                        *reinterpret_cast<uint4*>(stage + (q & 3) * kMnChunk + (last + (q >> 5)) * 128 + ((q >> 2) & 7) * 16) = make_uint4(0, 0, 0, 0);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) arrive_even(smem_u32(&ready[s]));
                    return true;
                });
            });
            if (!done) give_up(abort_flag);
        } else if (C::kAdapter && warp >= kPrepWarp && warp < kTmaWarp) {
            // The TMA warp passes a free stage on through full[s]; every use of a stage for an adapter is one
            // phase of that barrier.  (empty[s] cannot be waited on here: its parity says nothing to a waiter
            // that skips phases.)
            const int pt = threadIdx.x - kPrepWarp * 32;
            int it = 0, waited = 0;  // slices so far, and at the last wait
            uint32_t phase = 0;  // a bit per stage
            bool ok = true;
            for (int item = blockIdx.x >> 1; item < P.items && ok; item += gridDim.x >> 1) {
                const Tile t = tile_of<MODE>(P, item);
                const Unit u = unit_of<MODE>(P, t, 0);
                it += u.total;
                if (!u.extra) continue;
                const long long m0 = static_cast<long long>(t.tm) * 256 + rank * 128;
                const int n0 = t.tn * NB + rank * C::kCols, own = m0 + pt < P.ad.n ? __ldg(P.ad.who + m0 + pt) : -1;
                AdapterSlice<MODE> slice;
                int a = __ldg(u.list + 1);
                slice.fetch(P.ad, own, a, 0, m0, n0, pt);
                for (int x = 0; x < u.extra; ++x, ++it) {
                    const int s = it % kStages, next = x + 1;
                    const int following = next < u.extra ? __ldg(u.list + 1 + next / u.rslices) : 0;
                    if (!wait(smem_u32(&full[s]), (phase >> s) & 1, abort_flag, it - waited)) { ok = false; break; }
                    waited = it;
                    phase ^= 1u << s;
                    const bool odd = slice.build(smem + s * C::kStage, smem + s * C::kStage + C::kA, pt);
                    if (odd) set_pair(odd_flag, odd_bit(a));
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) arrive_even(smem_u32(&ready[s]));
                    a = following;
                    if (next < u.extra) slice.fetch(P.ad, own, a, next % u.rslices * 32, m0, n0, pt);
                }
            }
            if (!ok) give_up(abort_flag);
        }
    }
    fence_before();
    cluster_sync_all();
    if (warp == 0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Joins the shares of the units behind the whole ones, in order: four consecutive columns per thread.
template <int MODE>
__global__ void __launch_bounds__(256) join_splits_kernel(const __grid_constant__ Params P, const int from) {
    const int unit = from + blockIdx.y;
    const Tile t = tile_of<MODE>(P, P.whole + unit);
    const int at_tile = (blockIdx.x * 256 + threadIdx.x) * 4;
    const long long row = t.tm * 256ll + at_tile / 256, col = t.tn * 256ll + at_tile % 256;
    if (row >= P.M || col >= P.N || (MODE == kHess && col / 128 > row / 128)) return;
    const float* part = P.part + static_cast<long long>(unit) * kPartTile + at_tile;
    float v[4] = {};
#pragma unroll 4
    for (int q = 0; q < P.splits; ++q) {
        const float4 f = *reinterpret_cast<const float4*>(part + static_cast<long long>(q) * P.tail * kPartTile);
        v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
    }
    const long long at = (kind(MODE) == kGrad ? t.s * P.out_stride : 0) + row * P.ldo + col;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (col + e >= P.N) break;
        float* to = static_cast<float*>(P.out) + at + e;
        if constexpr (MODE == kHess) *to = P.accumulate ? *to + v[e] : v[e];
        else if constexpr (kind(MODE) == kFisher) *to = P.first ? v[e] : fmaf(P.decay, *to, v[e]);
        else if (Cfg<MODE>::kAdapter || P.out_bf16) static_cast<bf16*>(P.out)[at + e] = __float2bfloat16_rn(v[e]);
        else *to = v[e];
    }
}

// Row-major [rows][cols] of `esize`-byte elements, boxes of box_cols x box_rows (128-byte swizzle or none).
int make_map(CUtensorMap* map, const void* base, int esize, long long cols, long long rows, long long ld, int box_cols,
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

template <int MODE>
int launch(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& e, const CUtensorMap& o, const CUtensorMap& part, const Params& P, cudaStream_t st) {
    using C = Cfg<MODE>;
    // Per device: the shared-memory limit, and that the launch has the registers that the roles' shares add up to.
    static std::mutex mu;
    static uint64_t prepared = 0;
    int dev = 0;
    int rc = require_device(&dev);
    if (rc) return rc;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 64 || !(prepared >> dev & 1)) {
            cudaFuncAttributes fa{};
            cudaError_t e = cudaFuncGetAttributes(&fa, linear_kernel<MODE>);
            if (e == cudaSuccess && C::kPromote && fa.numRegs != 128)
                return fail(TB_ERR_CUDA, "linear_kernel<%d> has %d registers a thread, not 128", MODE, fa.numRegs);
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(linear_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::kSmem));
            if (e != cudaSuccess) return cuda_fail(e, "linear_kernel setup");
            if (dev < 64) prepared |= 1ull << dev;
        }
    }
    const int pairs = static_cast<int>(std::min<long long>(P.items, kPairs));
    linear_kernel<MODE><<<2 * pairs, kThreads, C::kSmem, st>>>(a, b, e, o, part, P);
    return check_launch("linear_kernel");
}

// Results [samples][rows][cols] in rows of ld, as boxes of 32 rows x 128 bytes.
int make_out_map(CUtensorMap* map, void* base, bool bf16_out, long long cols, long long rows, long long samples, long long ld, long long stride) {
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

// launch() of `units` sums of about `slices` K slices each, in waves of one a pair
// of SMs.  The units of a last wave that is not full, or of an only one, are
// shared out where that is sooner: s shares of at most `shares` parts, two waves
// of them at most, s chosen for the fewest slices one after another, the second
// kernel that joins them counted as ten and an eighth for each share's tile (a
// slice takes 0.25 us, the join 2.5).  (64 tokens' forward, 4096 x 4096, 16
// units: 33.6 us with one share, 19.3 with four.)  The Hessian goes by way of
// `part` too where its rows do not start on 16 bytes, as TMA wants them.
template <int MODE>
int launch_shared(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& e, Params& P, long long units, long long slices,
                  long long shares, const char* who, cudaStream_t st) {
    constexpr bool kTma = kind(MODE) == kGrad || MODE == kHess;
    if (units > 0x3FFFFFFFll) return fail(TB_ERR_CAPACITY, "%s: %lld output tiles", who, units);
    const int esize = P.out_bf16 ? 2 : 4;
    P.out_tma = kTma && reinterpret_cast<uintptr_t>(P.out) % 16 == 0 && P.ldo * esize % 16 == 0 && P.out_stride * esize % 16 == 0;
    const long long tail = units % kPairs;
    long long best = slices, splits = 1;
    for (long long s = 2; tail && s <= shares && tail * s <= 2 * kPairs; ++s) {
        const long long cost = (tail * s + kPairs - 1) / kPairs * ((slices + s - 1) / s) + 10 + tail * s / 8;
        if (cost < best) best = cost, splits = s;
    }
    P.tail = static_cast<int>(MODE == kHess && !P.out_tma ? units : splits > 1 ? tail : 0);
    P.splits = static_cast<int>(P.tail == tail ? splits : 1);
    P.whole = static_cast<int>(units - P.tail);
    P.items = P.whole + P.tail * P.splits;
    CUtensorMap o{}, parts{};
    if (P.out_tma && P.whole) {
        const int rc = make_out_map(&o, P.out, P.out_bf16, P.N, P.M, std::max(1, P.S), P.ldo, P.out_stride);
        if (rc) return rc;
    }
    if (!P.tail) return launch<MODE>(a, b, e, o, parts, P, st);
    void* part = nullptr;
    const long long slots = static_cast<long long>(P.tail) * P.splits;
    int rc = scratch_alloc(&part, sizeof(float) * slots * kPartTile, st);
    if (rc) return rc;
    P.part = static_cast<float*>(part);
    if (kTma) rc = make_out_map(&parts, part, false, 256, 256, slots, 256, kPartTile);
    if (!rc) rc = launch<MODE>(a, b, e, o, parts, P, st);
    for (int u = 0; !rc && u < P.tail; u += 65535) {  // (a grid's y extent)
        join_splits_kernel<MODE><<<dim3(64, std::min(P.tail - u, 65535)), 256, 0, st>>>(P, u);
        rc = check_launch("join_splits_kernel");
    }
    scratch_free(part, st);
    return rc;
}

int tiles(long long v, int t) { return static_cast<int>((v + t - 1) / t); }

// Gradients and Fisher decode their codes once for each tile of rows and part of
// dY.  Where that is five times or more, the values are written out as BF16 first,
// to scratch, and the products read them without a decode between TMA and MMA; not
// where a pair of SMs has fewer than 32 slices, for which one launch more is not
// worth it.  (Kernels, 4096 features, decoded in the product against written out:
// 16 gradients of 4096 rows 313 and 248 + 17 us; 2048 rows, with all launches, 157
// and 145; 1024 rows 87 and 87; 512 rows 53 and 59.  One gradient of 500 tokens and
// 2048 rows 16.0 and 17.4.  64 samples' Fisher of 4096 rows 752 and 561 + 37.  Between
// and for other types, 16 gradients, calls: BF16 of 1280 rows, five uses, 135 and 123;
// F16 of 512 rows, four, 105 and 103, of 768, six, 147 and 137; FP32 of 256, three, 88
// and 89, of 512, six, 140 and 128.  16 samples' Fisher: BF16 of 1280 rows 110 and 110,
// F16 of 768 180 and 165, FP32 of 512 187 and 178.  One FP32 gradient of 509 tokens and
// 1024 rows 29 and 31.)
constexpr long long kValuesMax = 1ll << 31;  // bytes of them at most

template <int MODE, int VALUES>
int from_codes(const act8::View& ck, const Parts& dy, int r, Params& P, long long samples, const char* who, cudaStream_t st) {
    if (ck.n * dy.parts > 0x7FFFFFFFll - 64) return fail(TB_ERR_CAPACITY, "%s: %lld tokens in %d parts", who, ck.n, dy.parts);
    P.M = r;
    P.N = ck.d;
    P.tiles_m = tiles(r, 256);
    P.tiles_n = tiles(ck.d, 256);
    P.exps = ck.exps;
    P.lde = ck.lde;
    P.n = static_cast<int>(ck.n);
    P.parts = dy.parts;
    P.ldo = ck.d;
    int rc = TB_OK;
    CUtensorMap a{}, b{}, e{};
    const long long ld = (ck.d + 7) / 8 * 8;
    const long long units = static_cast<long long>(P.tiles_m) * P.tiles_n * samples;
    // (The samples' lengths are on the device: as if they were even.)  A unit of the Fisher mode has all samples.
    const long long each = (ck.n / std::max(1, P.S) + 63) / 64 * dy.parts, slices = MODE == kFisher ? P.S * each : each;
    const long long shares = MODE == kFisher ? P.S : slices;
    const bool values = static_cast<long long>(P.tiles_m) * P.parts >= 5 && units * slices >= 32 * kPairs && 2 * ck.n * ld <= kValuesMax;
    void* x = nullptr;
    if (values) {
        rc = scratch_alloc(&x, static_cast<size_t>(2 * ck.n * ld), st);
        if (!rc) rc = act8::unpack(ck, x, TB_BF16, ld, st);
    }
    if (!rc && ck.n > 0) rc = make_map(&a, dy.base, 2, r, ck.n * dy.parts, dy.ld, 64, 64, true);
    if (!rc && values) rc = make_map(&b, x, 2, ck.d, ck.n, ld, 64, 64, true);
    if (!rc && ck.n > 0 && !values) rc = make_map(&b, ck.codes, 1, ck.d, ck.n, ck.ldq, Cfg<MODE>::kCols, 64, false);
    if (!rc && ck.n > 0 && !values) rc = make_map(&e, ck.exps, 1, ck.d, (ck.n + 127) / 128, ck.lde, Cfg<MODE>::kCols, 1, false);
    if (!rc) rc = values ? launch_shared<VALUES>(a, b, b, P, units, slices, shares, who, st) : launch_shared<MODE>(a, b, e, P, units, slices, shares, who, st);
    scratch_free(x, st);
    return rc;
}

}  // namespace

int weight_grad(const act8::View& ck, const Parts& dy, int r, const int64_t* samples, int S, void* grads, int g_dtype,
                long long g_stride, cudaStream_t st) {
    Params P{};
    P.samples = samples;
    P.S = S;
    P.out = grads;
    P.out_bf16 = g_dtype == TB_BF16;
    P.out_stride = g_stride;
    return from_codes<kGrad, kGradX>(ck, dy, r, P, S, "tb_act8_weight_grad", st);
}

int fisher(const act8::View& ck, const Parts& dy, int r, const int64_t* samples, int S, double alpha, double beta, bool first,
           float* F, cudaStream_t st) {
    Params P{};
    P.samples = samples;
    P.S = S;
    P.out = F;
    P.alpha = alpha;
    P.beta = beta;
    P.first = first;
    P.decay = static_cast<float>(pow(beta, static_cast<double>(S)));
    return from_codes<kFisher, kFisherX>(ck, dy, r, P, 1, "tb_act8_fisher", st);
}

int hessian(const act8::View& ck, float scale, bool accumulate, float* H, cudaStream_t st) {
    Params P{};
    P.M = P.N = ck.d;
    P.tiles_m = tiles(ck.d, 256);
    P.exps = ck.exps;
    P.lde = ck.lde;
    P.n = static_cast<int>(ck.n);
    P.out = H;
    P.ldo = ck.d;
    P.scale = scale;
    P.accumulate = accumulate;
    if (ck.n == 0 && accumulate) return TB_OK;
    if (P.tiles_m > 46000) return fail(TB_ERR_CAPACITY, "tb_act8_hessian: %d features", ck.d);  // tiles are counted in 31 bits
    int rc = TB_OK;
    CUtensorMap a{};
    if (ck.n > 0) rc = make_map(&a, ck.codes, 1, ck.d, ck.n, ck.ldq, 128, 128, true);
    P.out_stride = static_cast<long long>(ck.d) * ck.d;
    const long long units = static_cast<long long>(P.tiles_m) * (P.tiles_m + 1) / 2;
    return rc ? rc : launch_shared<kHess>(a, a, a, P, units, (ck.n + 127) / 128, (ck.n + 127) / 128, "tb_act8_hessian", st);
}

template <int MODE>
static int adapter_product(const AdapterProduct& p, const char* who, cudaStream_t st) {
    Params P{};
    P.M = p.n;
    P.N = p.N;
    P.K = p.K;
    P.n = static_cast<int>(p.n);
    P.tiles_m = tiles(p.n, 256);
    P.tiles_n = tiles(p.N, 256);
    P.out = p.out;
    P.ldo = p.ldout;
    P.ad = p;
    int rc = TB_OK;
    CUtensorMap a{}, b{};
    if (!rc) rc = make_map(&a, p.in, 2, p.K, p.n, p.ldin, 64, 128, true);
    if (!rc) rc = MODE == kFwd ? make_map(&b, p.w, 2, p.K, p.N, p.ldw, 64, 128, true)
                               : make_map(&b, p.w, 2, p.N, p.K, p.ldw, 64, 64, true);
    if (!rc) rc = launch_shared<MODE>(a, b, b, P, static_cast<long long>(P.tiles_m) * P.tiles_n, (p.K + 63) / 64, (p.K + 63) / 64, who, st);
    return rc;
}

int adapter_forward(const AdapterProduct& p, cudaStream_t st) { return adapter_product<kFwd>(p, "tb_adapter_forward", st); }
int adapter_input_grad(const AdapterProduct& p, cudaStream_t st) { return adapter_product<kDx>(p, "tb_adapter_backward", st); }

int take_error(cudaStream_t st) {
    int h = 0, zero = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&h, g_linear_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaMemcpyToSymbolAsync(g_linear_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    return e == cudaSuccess ? h : -1;
}

}  // namespace linear
}  // namespace tb
