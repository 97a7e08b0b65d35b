// Attention over packed prompts on the tensor cores:
//
//   S = scale Q K^T (masked)   P = exp(S - lse)   O = P V          lse = log sum exp S, row by row
//   delta = rowsum(O * dO)     dV = P^T dO        dS = P * (dO V^T - delta)
//   dQ = scale dS K            dK = scale dS^T Q  (dK and dV summed over the query heads of a group)
//
// Three kernels of one shape: a TMA warp, a warp whose elected lane issues every tcgen05.mma, and eight (forward) or
// sixteen warps that turn scores into probabilities.  Tiles are 128 rows of 64 (dim <= 64) or 128 elements in
// 128-byte-swizzled shared memory; a dimension in between is filled up with zeros by TMA, and the products run over
// the multiple of 16 that covers it.  P and dS are the products' left operands straight from TMEM, as 16-bit pairs:
// they never pass through shared memory.
// That rounding to 16 bits is the one the operands of the tensor cores ask for; sums, maxima, lse, delta and the
// accumulators are float32.
//
// Rows of other sequences.  The tile at a sequence's end also holds rows of the next one or of padding.  Scores of
// such keys are replaced, not added to; but a probability of zero times a NaN in such a row would reach the sum, so
// the rows that a product sums over are zeroed in shared memory behind the sequence's end.
//
// Backward without atomics: dQ in a kernel of its own (one tile of queries, all keys) beside dK and dV (one tile of
// keys, all queries of all heads of the group).  S and dO V^T are formed twice, seven products instead of five, and
// in return no float32 sums of dQ go through memory and the same bits come out every time.
#include "attention.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "f32x2.cuh"
#include "gemm_device.cuh"
#include "launch_count.h"

namespace mgk {
namespace attn {

namespace {

using namespace mgk::ptx;

constexpr int TILE = 128;
constexpr int CHUNK_BYTES = TILE * 128;  // 128 rows of 64 elements
constexpr float LOG2E = 1.4426950408889634f;
constexpr int POLY = 1, POLY_OF = 4;  // of so many pairs of exponentials, so many by polynomial
constexpr uint64_t WAIT_NS = 4000000000ull;
constexpr float FAR = 0x1p20f;  // scores times scale log2 e from which on exponents are formed from differences

struct Params {
    const int* cu;
    int seqs, tokens, heads, kv_heads, dim;
    int causal;
    float scale;
    int* error_flag;
    // outputs and row statistics
    uint16_t *out0, *out1;
    int64_t row0, head0, row1, head1;
    float* lse;
    const float* delta;
    int tiles_per_cta;  // forward: tiles of queries
    int splits;         // dK and dV: CTAs that share the queries of one tile of keys
    float* part;        // their partial sums, [dK, dV][splits][tokens][kv_heads][dim], when splits > 1
};

// ---------------------------------------------------------------- PTX beyond ptx_sm100.cuh
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
            "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
            : "memory");
}
// Products of one CTA with 128 rows.  Operands in shared memory are given by the low word of their descriptor; the
// high one (8-row groups 1024 bytes apart, 128-byte swizzle) is the same for all.  A in TMEM: lane = row, a 32-bit
// column holds two neighbours along K.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
            "{\n"
            " .reg .pred p;\n"
            " .reg .b64 da, db;\n"
            " mov.b64 da, {%1, %5};\n"
            " mov.b64 db, {%2, %5};\n"
            " setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n"
            "}\n" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(DESC_HI)
            : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
            "{\n"
            " .reg .pred p;\n"
            " .reg .b64 db;\n"
            " mov.b64 db, {%2, %5};\n"
            " setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n"
            "}\n" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(DESC_HI)
            : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
            "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
            "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
            "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
            "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
            "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
            "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
            : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
            "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
            "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
            "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
            : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Moves registers from warps that need few to those that hold scores; the sums may not pass what the threads of the
// block started with
template <int N>
__device__ __forceinline__ void set_registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void set_registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// Programmatic launches: the next kernel of the stream may start once all CTAs of this one have said so (or ended);
// it waits where it needs this one's end.
__device__ __forceinline__ void next_kernel_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
using f32x2::both;
using f32x2::max3_nan;
using f32x2::Pair;

// 2^x for x <= 126 without the special-function unit: x = n + f with n the nearest whole number (it is left in the low
// bits of x + 1.5 2^23) and |f| <= 1/2, a polynomial of degree 4 for 2^f that is 1 at 0 (the least largest relative
// error, found by linear programming: 2.9e-6 in float32, a 700th of half a bf16 step), times 2^n.  At 2^-127 and
// below the result is zero, exactly: masked scores are -infinity.  A NaN stays one.
__device__ __forceinline__ Pair ex2_poly(Pair x) {
    const float magic = 12582912.f;
    x.x = max3_nan(x.x, -127.f, -127.f);
    x.y = max3_nan(x.y, -127.f, -127.f);
    const Pair t = f32x2::add(x, both(magic)), f = f32x2::add(x, f32x2::fma(t, both(-1.f), both(magic)));
    Pair p = f32x2::fma(both(0.009582852944731712f), f, both(0.055906426161527634f));
    p = f32x2::fma(p, f, both(0.24024099111557007f));
    p = f32x2::fma(p, f, both(0.6931241750717163f));
    p = f32x2::fma(p, f, both(1.f));
    return f32x2::mul(p, {__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                          __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u)});
}
// 2^x of a pair by one way or the other
template <bool POLY>
__device__ __forceinline__ Pair ex2_pair(Pair x) {
    if (POLY)
        return ex2_poly(x);
    return {ex2(x.x), ex2(x.y)};
}
template <bool FP16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (FP16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool FP16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if (FP16)
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// M = 128, both operands f16 or both bf16, float32 accumulator
template <bool FP16>
__device__ __forceinline__ uint32_t idesc_for(int n, bool b_mn) {
    const uint32_t f = FP16 ? 0u : 1u;
    return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(TILE >> 4) << 24);
}
// Tile [128 rows, dim] as an operand whose K axis is dim, or whose K axis is the rows: low word of the descriptor,
// and what a step of 16 elements or rows adds to it
__device__ __forceinline__ uint32_t desc_k(uint32_t tile) { return ((tile & 0x3FFFF) >> 4) | (1u << 16); }
__device__ __forceinline__ constexpr uint32_t step_k(int kk) { return ((kk >> 2) * CHUNK_BYTES + (kk & 3) * 32) >> 4; }
__device__ __forceinline__ uint32_t desc_mn(uint32_t tile) {
    return ((tile & 0x3FFFF) >> 4) | (static_cast<uint32_t>(CHUNK_BYTES >> 4) << 16);
}
__device__ __forceinline__ constexpr uint32_t step_mn(int kk) { return kk * 2048 >> 4; }

// The two kinds of products.  Everything an instruction needs is an addition away: the one thread that issues them
// was what the kernels waited for when each built its descriptors (75 cycles an instruction that takes 64).
// [128, 128] (+)= tile tile^T over `ksteps` x 16 elements of the dimension
template <int DP>
__device__ __forceinline__ void multiply_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int ksteps) {
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
        if (kk < ksteps)
            umma_ss(d, a + step_k(kk), b + step_k(kk), idesc, kk != 0);
}
// [128, dim] (+)= P tile over the tile's 128 rows
__device__ __forceinline__ void multiply_scores(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
#pragma unroll
    for (int kk = 0; kk < TILE / 16; ++kk)
        umma_ts(d, a + 8 * kk, b + step_mn(kk), idesc, kk != 0 || accumulate);
}
// A wait of the thread that issues products: it polls a while before it sleeps, which wakes it sooner
__device__ __forceinline__ bool issue_wait(uint32_t bar, uint32_t parity, const WaitCtx& w) {
    for (int i = 0; i < 256; ++i)
        if (mbar_test_wait(bar, parity))
            return true;
    return mbar_wait(bar, parity, w);
}

// ---------------------------------------------------------------- which sequence a tile belongs to
struct Where {
    int start, len, local;  // first row and length of the sequence, the tile's number in it; len = 0: no such tile
    int tiles;              // tiles of the sequence
};
// Tiles are numbered so that a sequence's first one follows from its own offset alone: tile cu[s] / rows + s.  (A sequence
// of L rows takes at most L / rows + 1 numbers, and the next one begins no earlier.)  So the sequence of a tile is found
// by a search, 32 offsets a step, whatever the number of sequences; numbers in between belong to no tile.  By one
// whole warp.  Offsets are forced into order and range, so that no access leaves the tensors whatever they hold.
__device__ __forceinline__ Where find_tile(const Params& p, int rows, int index) {
    Where w{0, 0, 0, 0};
    if (p.cu == nullptr) {
        w.tiles = (p.tokens + rows - 1) / rows;
        if (index < w.tiles)
            w = {0, p.tokens, index, w.tiles};
        return w;
    }
    const int lane = threadIdx.x & 31;
    auto offset = [&](int s) { return min(max(p.cu[s], 0), p.tokens); };
    int lo = 0, hi = p.seqs;  // the last sequence that begins at or before the tile lies in [lo, hi)
    do {
        const int step = (hi - lo + 31) / 32, s = lo + lane * step;
        const unsigned before = __ballot_sync(0xffffffffu, s < hi && offset(s) / rows + s <= index);
        if (before == 0)
            return w;
        lo += (31 - __clz(before)) * step;
        hi = min(hi, lo + step);
    } while (hi - lo > 1);
    const int start = offset(lo), len = max(offset(lo + 1) - start, 0);
    w.tiles = (len + rows - 1) / rows;
    w.local = index - (start / rows + lo);
    if (w.local >= 0 && w.local < w.tiles) {
        w.start = start;
        w.len = len;
    }
    return w;
}

// Loads rows [row, row + 128) of one head; `bar` counts the bytes (chunks past the dimension are not loaded)
template <int DP>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int head, int row) {
    mbar_expect_tx(bar, DP / 64 * CHUNK_BYTES);
#pragma unroll
    for (int c = 0; c < DP / 64; ++c)
        tma_load_3d(dst + c * CHUNK_BYTES, map, bar, c * 64, head, row);
}
// Zeroes rows [from, 128) of a tile (by a whole warp) for the asynchronous reads that follow
template <int DP>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from) {
    const int lane = threadIdx.x & 31;
    for (int c = 0; c < DP / 64; ++c)
        for (int i = from * 8 + lane; i < TILE * 8; i += 32)
            reinterpret_cast<uint4*>(tile + c * CHUNK_BYTES)[i] = make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
    __syncwarp();
}
// One tile into ring slot `dst` by a whole warp.  If the sequence ends inside, the rows behind are zeroed before
// the slot's barrier completes: the copy then arrives on `side` first.
template <int DP>
__device__ __forceinline__ bool feed(uint8_t* dst, const CUtensorMap* map, uint32_t full, uint32_t side, uint32_t& side_phase,
                                     int head, int row, int live, const WaitCtx& wc) {
    const bool cut = live < TILE;
    if (elect_one())
        load_tile<DP>(smem_u32(dst), map, cut ? side : full, head, row);
    __syncwarp();
    if (cut) {
        const bool ok = mbar_wait(side, side_phase, wc);
        side_phase ^= 1;
        if (!__all_sync(0xffffffffu, ok))
            return false;
        zero_rows<DP>(dst, live);
        if (elect_one())
            mbar_arrive(full);
        __syncwarp();
    }
    return true;
}

__device__ __forceinline__ uint8_t* align_1024(uint8_t* p) {
    return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~static_cast<uintptr_t>(1023));
}

// After a wait that ran out: copies and products may still be under way into memory that this CTA is about to give
// back.  They depend on nothing that this CTA still does; about a millisecond is left to them to end.
__device__ __forceinline__ void settle(const volatile int* abort_flag) {
    if (*abort_flag)
        for (int i = 0; i < 100; ++i)
            poll_pause(10000);
}

// Swizzled tiles start at multiples of 1024 bytes.  Dynamic shared memory does, and the backward kernels have no room
// for shifting it: if it ever does not, the error flag is set and nothing is done.
__device__ __forceinline__ bool unaligned(const uint8_t* smem, const Params& p) {
    if ((smem_u32(smem) & 1023) == 0)
        return false;
    if (threadIdx.x == 0 && p.error_flag != nullptr)
        *p.error_flag = 1;
    return true;
}

// Writes columns [from, to) of one row of float32 TMEM columns times `f`, rounded, to global memory; `from` is a
// multiple of 32
template <bool FP16>
__device__ __forceinline__ void store_row(uint32_t taddr, int from, int to, float f, uint16_t* row, bool write) {
    for (int c = from; c < to; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(taddr + c, r);
        tmem_ld_wait(r);
        if (!write)
            continue;
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            if (c + i < to) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = pack2<FP16>(__uint_as_float(r[i + 2 * k]) * f, __uint_as_float(r[i + 2 * k + 1]) * f);
                *reinterpret_cast<uint4*>(row + c + i) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

// The same as float32
__device__ __forceinline__ void store_sums(uint32_t taddr, int from, int to, float* row, bool write) {
    for (int c = from; c < to; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(taddr + c, r);
        tmem_ld_wait(r);
#pragma unroll
        for (int i = 0; i < 32; i += 4)
            if (write && c + i < to)
                *reinterpret_cast<uint4*>(row + c + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
    }
}

// ================================================================ forward
//
// A CTA takes two tiles of 128 queries of one head and walks over the keys once; while one warpgroup works on the
// scores of its tile, a row a thread, the tensor cores work for the other tile.  P lies over the scores that it comes
// from.  Bound by that chain: 3400 cycles for two tiles whose products take 2230.  (16384 tokens, 8 heads of 128,
// causal: 451 us, 1.22 PFLOP/s, in a short run at full clocks; 503 us at the power limit.)
// The running maximum is that of the first block until a later one is more than 2^32 larger (2^8 for float16, whose
// numbers end at 2^16): P may then be that large, which changes nothing in its relative precision.  So a block's
// exponentials do not wait for its maximum, which is found beside them; only if it did rise that far they are taken
// again, and the threads that own its rows rescale the accumulator in TMEM.
constexpr int FWD_ROW_WARPS = 8, FWD_MMA = 8, FWD_TMA = 9;  // (and two warps that idle)
constexpr int FWD_THREADS = 32 * (FWD_ROW_WARPS + 4);
constexpr int FWD_STAGES = 4;

template <int DP>
constexpr int tile_bytes() { return DP / 64 * CHUNK_BYTES; }
template <int DP>
constexpr int fwd_smem() { return (2 + FWD_STAGES) * tile_bytes<DP>() + 1024 + 512; }

template <int DP, bool FP16>
__global__ void __launch_bounds__(FWD_THREADS, 1)
        forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const Params p) {
    constexpr int TB = tile_bytes<DP>();
    // the last tiles of a sequence, which have the most keys, come first
    const int rows = p.tiles_per_cta * TILE;
    auto first_row = [&](const Where& w) { return (w.tiles - 1 - w.local) * rows; };
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align_1024(smem_raw);
    uint8_t* ring = smem + 2 * TB;
    uint64_t* bars = reinterpret_cast<uint64_t*>(ring + FWD_STAGES * TB);
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * FWD_STAGES;
    const uint32_t q_full = empty0 + 8 * FWD_STAGES;          // one per tile
    const uint32_t s_full = q_full + 16, p_ready = s_full + 16, o_full = p_ready + 16, side = o_full + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * FWD_STAGES + 9);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    Where* where = reinterpret_cast<Where*>(tmem_slot + 2);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const int head = static_cast<int>(blockIdx.x % p.heads);
    const int kv_head = head / (p.heads / p.kv_heads);
    if (warp == FWD_TMA) {
        if (lane == 0) {
            *abort_flag = 0;
            for (int s = 0; s < 2 * FWD_STAGES; ++s)
                mbar_init(full0 + 8 * s, 1);
            for (int t = 0; t < 2; ++t) {
                mbar_init(q_full + 8 * t, 1);
                mbar_init(s_full + 8 * t, 1);
                mbar_init(p_ready + 8 * t, FWD_ROW_WARPS / 2);
                mbar_init(o_full + 8 * t, 1);
            }
            mbar_init(side, 1);
            mbar_fence_init();
            fence_proxy_async_smem();
        }
        const Where found = find_tile(p, rows, static_cast<int>(blockIdx.x / p.heads));
        __syncwarp();
        if (elect_one()) {
            *where = found;
            if (found.len > 0) {  // the first copies are under way while the rest is set up
                const int first = first_row(found);
                load_tile<DP>(smem_u32(smem), &map_q, q_full, head, found.start + first);
                load_tile<DP>(smem_u32(ring), &map_k, full0, kv_head, found.start);
                if (rows > TILE && first + TILE < found.len)
                    load_tile<DP>(smem_u32(smem) + TB, &map_q, q_full + 8, head, found.start + first + TILE);
            }
        }
        __syncwarp();
    } else if (warp == FWD_MMA) {
        tmem_alloc_cg1(smem_u32(tmem_slot), 512);
        tmem_relinquish_cg1();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const Where w = *where;
    const uint32_t tmem = *tmem_slot;
    if (w.len == 0) {  // no such tile
        if (warp == FWD_MMA)
            tmem_dealloc_cg1(tmem, 512);
        return;
    }
    const uint32_t t_s = tmem, t_o = tmem + 2 * TILE;  // S of tile t at t_s + 128 t, O at t_o + 128 t

    const int r0 = first_row(w);
    int n_blocks[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int first = r0 + t * TILE;
        const int keys = p.causal ? min(w.len, first + TILE) : w.len;
        n_blocks[t] = t < p.tiles_per_cta && first < w.len ? (keys + TILE - 1) / TILE : 0;
    }
    const int n = max(n_blocks[0], n_blocks[1]);
    WaitCtx wc{abort_flag, WAIT_NS};

    if (warp == FWD_TMA) {
        set_registers_down<72>();  // 256 x 216 + 128 x 72 = 384 x 168
        uint32_t side_phase = 0;
        for (int it = 1; it < 2 * n; ++it) {  // (0 is on its way)
            const int s = it % FWD_STAGES;
            if (!__all_sync(0xffffffffu, mbar_wait(empty0 + 8 * s, ((it / FWD_STAGES) & 1) ^ 1, wc)))
                break;
            const int k0 = (it >> 1) * TILE;
            // keys behind the end are masked where their scores are used; values are summed over
            const int live = (it & 1) ? w.len - k0 : TILE;
            if (!feed<DP>(ring + s * TB, (it & 1) ? &map_v : &map_k, full0 + 8 * s, side, side_phase, kv_head, w.start + k0,
                          live, wc))
                break;
        }
    } else if (warp == FWD_MMA) {
        set_registers_down<72>();  // 256 x 216 + 128 x 72 = 384 x 168
        if (elect_one()) {
            const int ksteps = (p.dim + 15) / 16;
            const uint32_t id_s = idesc_for<FP16>(TILE, false), id_o = idesc_for<FP16>(ksteps * 16, true);
            const uint32_t q_desc = desc_k(smem_u32(smem)), ring0 = smem_u32(ring);
            auto scores = [&](int t, uint32_t k) {
                multiply_rows<DP>(t_s + t * TILE, q_desc + t * (TB >> 4), k, id_s, ksteps);
                umma_commit_cg1(s_full + 8 * t);
            };
            bool ok = issue_wait(q_full, 0, wc) && issue_wait(full0, 0, wc);
            if (ok) {
                tc_fence_after();
                scores(0, desc_k(ring0));
                if (n_blocks[1] > 0) {
                    ok = issue_wait(q_full + 8, 0, wc);
                    if (ok)
                        scores(1, desc_k(ring0));
                }
                if (n > 2)  // the slot is used again
                    umma_commit_cg1(empty0);
            }
            int sv = 1, sk = 2;       // slots of this block's values and of the next one's keys
            uint32_t pv = 0, pk = 0;  // and the parities of their barriers
            bool v_here = false, k_here = false;
            for (int j = 0; ok && j < n; ++j) {
                const uint32_t v = desc_mn(ring0 + sv * TB), k = desc_k(ring0 + sk * TB);
                bool next = false;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (!ok || j >= n_blocks[t])
                        continue;
                    ok = (v_here || issue_wait(full0 + 8 * sv, pv, wc)) && issue_wait(p_ready + 8 * t, j & 1, wc);
                    if (!ok)
                        continue;
                    v_here = true;
                    tc_fence_after();
                    const bool last = j + 1 == n_blocks[t];
                    if (!last && !k_here)  // (asked for early: its answer comes while the products are issued)
                        k_here = mbar_test_wait(full0 + 8 * sk, pk);
                    multiply_scores(t_o + t * TILE, t_s + t * TILE, v, id_o, j != 0);
                    if (last) {
                        umma_commit_cg1(o_full + 8 * t);
                    } else {
                        ok = k_here || issue_wait(full0 + 8 * sk, pk, wc);
                        k_here = true;
                        next = true;
                        if (ok) {
                            tc_fence_after();
                            scores(t, k);  // over P of this block: products of one thread run in order
                        }
                    }
                }
                if (next) {  // (behind the last block nobody waits for a free slot)
                    umma_commit_cg1(empty0 + 8 * sv);
                    umma_commit_cg1(empty0 + 8 * sk);
                }
                v_here = k_here = false;
                sv += 2;
                if (sv >= FWD_STAGES) {
                    sv -= FWD_STAGES;
                    pv ^= 1;
                }
                sk += 2;
                if (sk >= FWD_STAGES) {
                    sk -= FWD_STAGES;
                    pk ^= 1;
                }
            }
        }
        __syncwarp();
    } else if (warp < FWD_ROW_WARPS) {
        set_registers_up<216>();
        const int t = warp >> 2;
        const int row = (threadIdx.x & 127) + r0 + t * TILE;  // in the sequence
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = t_s + t * TILE + lanes, o_at = t_o + t * TILE + lanes;
        const float c = p.scale * LOG2E;
        const int limit = p.causal ? min(w.len, row + 1) : w.len;  // keys that this row sees
        float m = 0.f, l = 0.f;
        bool ok = true;
        // 32 scores of this row, masked
        auto chunk = [&](uint32_t (&s)[32], int i, int k0, bool masked) {
            tmem_ld_wait(s);
            if (masked) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (k0 + 32 * i + e >= limit)
                        s[e] = 0xff800000u;
            }
        };
        for (int j = 0; j < n_blocks[t]; ++j) {
            ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * t, j & 1, wc));
            if (!ok)
                break;
            tc_fence_after();
            const int k0 = j * TILE;
            const bool masked = k0 + TILE > w.len || (p.causal && k0 + TILE > r0 + t * TILE);
            uint32_t s[2][32], pk[2][32];
            Pair sum[2];
            // P with the maximum as it is, the block's own maximum beside it; a chunk is loaded while one is worked on
            auto exponentials = [&](auto far) {
                constexpr bool FAR_ROWS = decltype(far)::value;
                // (where all scores so far were -infinity their exponentials are zero)
                const float base = m == -INFINITY ? 0.f : m;
                // a row is far or not by itself, so that all its blocks have one reference
                const bool apart = FAR_ROWS && fabsf(base * c) >= FAR;
                const Pair cc = both(c), mc = both(apart ? 0.f : -base * c), off = both(apart ? -base : 0.f);
                float top[2] = {-INFINITY, -INFINITY};
                sum[0] = sum[1] = both(0.f);
                tmem_ld_32x32b_x32(s_at, s[0]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    chunk(s[i & 1], i, k0, masked);
                    if (i < 3)
                        tmem_ld_32x32b_x32(s_at + 32 * (i + 1), s[(i + 1) & 1]);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float a = __uint_as_float(s[i & 1][2 * e]), b = __uint_as_float(s[i & 1][2 * e + 1]);
                        Pair x = f32x2::fma(FAR_ROWS ? f32x2::add({a, b}, off) : Pair{a, b}, cc, mc);
                        x = e % POLY_OF < POLY ? ex2_pair<true>(x) : ex2_pair<false>(x);
                        top[e & 1] = max3_nan(top[e & 1], a, b);
                        sum[e & 1] = f32x2::add(sum[e & 1], x);
                        pk[i / 2][16 * (i & 1) + e] = pack2<FP16>(x.x, x.y);
                    }
                }
                return max3_nan(top[0], top[1], top[1]);
            };
            if (j == 0) {
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    tmem_ld_32x32b_x32(s_at + 32 * i, s[0]);
                    chunk(s[0], i, k0, masked);
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
                        top = max3_nan(top, __uint_as_float(s[0][e]), __uint_as_float(s[0][e + 1]));
                }
                m = top;
                exponentials(std::false_type{});
            } else {
                const float mx = exponentials(std::false_type{});
                // each row goes by its own maximum (also where a score is NaN: the row becomes NaN)
                const bool rises = !((mx - m) * c <= (FP16 ? 8.f : 32.f)) && mx != -INFINITY && row < w.len;
                if (__any_sync(0xffffffffu, rises)) {
                    // the product that last added to O has retired: the scores' barrier came after it
                    // (a row that does not rise is left alone: its maximum may be -infinity still)
                    const float to = rises ? max3_nan(m, mx, mx) : m, f = rises ? ex2((m - to) * c) : 1.f;
                    m = to;
                    l *= f;
                    for (int d = 0; d < p.dim; d += 32) {
                        tmem_ld_32x32b_x32(o_at + d, s[0]);
                        tmem_ld_wait(s[0]);
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            s[0][e] = __float_as_uint(__uint_as_float(s[0][e]) * f);
                        tmem_st_x32(o_at + d, s[0]);
                    }
                    exponentials(std::false_type{});
                }
            }
            // Far from zero the rounding of m c alone is a whole exponent: there the difference comes first
            if (__any_sync(0xffffffffu, fabsf(m * c) >= FAR && fabsf(m) != INFINITY && row < w.len))
                exponentials(std::true_type{});
            tmem_st_x32(s_at, pk[0]);
            tmem_st_x32(s_at + 32, pk[1]);
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(p_ready + 8 * t);
        }
        if (ok && n_blocks[t] > 0 && __all_sync(0xffffffffu, mbar_wait(o_full + 8 * t, 0, wc))) {
            tc_fence_after();
            const bool write = row < w.len;
            const int64_t at = w.start + row;
            store_row<FP16>(o_at, 0, p.dim, 1.f / l, p.out0 + at * p.row0 + head * p.head0, write);
            if (write)
                p.lse[static_cast<int64_t>(head) * p.tokens + at] = m * p.scale + logf(l);
        }
    } else {
        set_registers_down<72>();  // 256 x 216 + 128 x 72 = 384 x 168
    }
    settle(abort_flag);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == FWD_MMA)
        tmem_dealloc_cg1(tmem, 512);
    if (threadIdx.x == 0 && *abort_flag && p.error_flag != nullptr)
        *p.error_flag = 1;
}

// ================================================================ backward: delta
// Half a warp a row and head: sums of out * dout.  Bound by reading both.
template <bool FP16>
__global__ void __launch_bounds__(256) delta_kernel(const uint16_t* __restrict__ out, int64_t o_row, int64_t o_head,
                                                    const uint16_t* __restrict__ dout, int64_t d_row, int64_t d_head, int tokens,
                                                    int heads, int dim, float* __restrict__ delta) {
    next_kernel_may_start();
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);  // half a warp a row
    const int sub = threadIdx.x & 15;
    const int64_t row = i / heads, head = i % heads;
    float sum = 0.f;
    if (row < tokens && sub * 8 < dim) {
        const uint4 a = *reinterpret_cast<const uint4*>(out + row * o_row + head * o_head + sub * 8);
        const uint4 b = *reinterpret_cast<const uint4*>(dout + row * d_row + head * d_head + sub * 8);
        const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 x = unpack2<FP16>(aw[k]), y = unpack2<FP16>(bw[k]);
            sum += x.x * y.x + x.y * y.y;
        }
    }
    for (int o = 8; o > 0; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (row < tokens && sub == 0)
        delta[head * tokens + row] = sum;
}

// ================================================================ backward: dQ
//
// A CTA takes 128 queries of one head.  All row warps work on every tile of scores, a thread on a quarter of a row.
// Each has its own region of TMEM, which is free again as soon as its reader holds it in registers:
//   tensor cores:  S(j+1), dP(j+1) = dO V^T, dQ += dS(j) K, ...
//   row warps:     P(j) from S(j), dS(j) from dP(j), ...
constexpr int ROW_WARPS = 16, MMA_WARP = 16, TMA_WARP = 17, STAT_WARP = 18;  // (and a warp that idles)
constexpr int BWD_THREADS = 32 * (ROW_WARPS + 4);  // 512 x 104 + 128 x 64 = 640 x 96 registers

// Ring slots: the operand that both the scores and the last product of an iteration read (K, or Q) is held for one
// and a half iterations and needs three for the next to arrive in time, the other two.  (Two each: the tensor cores
// waited 1400 of 4600 cycles an iteration for Q.)
constexpr int LONG_STAGES = 3, SHORT_STAGES = 2;

template <int DP>
constexpr int bwd_smem() { return (2 + LONG_STAGES + SHORT_STAGES) * tile_bytes<DP>() + SHORT_STAGES * 2 * TILE * 4 + 256; }

// A quarter of a row (32 columns)
__device__ __forceinline__ void load_quarter(uint32_t at, float (&x)[32]) {
    uint32_t r[32];
    tmem_ld_32x32b_x32(at, r);
    tmem_ld_wait(r);
#pragma unroll
    for (int e = 0; e < 32; ++e)
        x[e] = __uint_as_float(r[e]);
}

template <int DP, bool FP16>
__global__ void __launch_bounds__(BWD_THREADS, 1)
        dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, const Params p) {
    constexpr int TB = tile_bytes<DP>();
    // the last tiles of a sequence, which have the most keys, come first
    auto first_row = [](const Where& w) { return (w.tiles - 1 - w.local) * TILE; };
    extern __shared__ __align__(1024) uint8_t smem[];  // Q, dO, then K slots, then V slots
    if (unaligned(smem, p)) {
        wait_for_last_kernel();
        return;
    }
    uint8_t *ring_k = smem + 2 * TB, *ring_v = ring_k + LONG_STAGES * TB;
    uint64_t* bars = reinterpret_cast<uint64_t*>(ring_v + SHORT_STAGES * TB);
    const uint32_t k_full = smem_u32(bars), k_empty = k_full + 8 * LONG_STAGES, v_full = k_empty + 8 * LONG_STAGES,
                   v_empty = v_full + 8 * SHORT_STAGES;
    const uint32_t q_full = v_empty + 8 * SHORT_STAGES, s_full = q_full + 8, s_free = s_full + 8, dp_full = s_free + 8, dp_free = dp_full + 8,
                   ds_ready = dp_free + 8, dq_done = ds_ready + 8, done = dq_done + 8, side = done + 8;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * (LONG_STAGES + SHORT_STAGES) + 9);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    Where* where = reinterpret_cast<Where*>(tmem_slot + 2);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const int head = static_cast<int>(blockIdx.x % p.heads);
    const int kv_head = head / (p.heads / p.kv_heads);
    if (warp == TMA_WARP) {
        if (lane == 0) {
            *abort_flag = 0;
            for (int s = 0; s < 2 * (LONG_STAGES + SHORT_STAGES); ++s)
                mbar_init(k_full + 8 * s, 1);
            mbar_init(q_full, 2);
            mbar_init(s_full, 1);
            mbar_init(s_free, ROW_WARPS);
            mbar_init(dp_full, 1);
            mbar_init(dp_free, ROW_WARPS);
            mbar_init(dq_done, 1);
            mbar_init(ds_ready, ROW_WARPS);
            mbar_init(done, 1);
            mbar_init(side, 1);
            mbar_fence_init();
            fence_proxy_async_smem();
        }
        const Where found = find_tile(p, TILE, static_cast<int>(blockIdx.x / p.heads));
        __syncwarp();
        if (elect_one()) {
            *where = found;
            if (found.len > 0) {  // the first copies are under way while the rest is set up
                load_tile<DP>(smem_u32(smem), &map_q, q_full, head, found.start + first_row(found));
                load_tile<DP>(smem_u32(smem) + TB, &map_do, q_full, head, found.start + first_row(found));
            }
        }
        __syncwarp();
    } else if (warp == MMA_WARP) {
        tmem_alloc_cg1(smem_u32(tmem_slot), 512);
        tmem_relinquish_cg1();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const Where w = *where;
    // The kernel before, dK and dV, need not have ended for this one to work, which fills the processors that it leaves
    // idle towards its end; but what comes after this one relies on both: its last CTA waits.
    const bool ends_last = blockIdx.x == gridDim.x - 1;
    const uint32_t tmem = *tmem_slot;
    if (w.len == 0) {  // no such tile
        if (warp == MMA_WARP)
            tmem_dealloc_cg1(tmem, 512);
        if (ends_last)
            wait_for_last_kernel();
        return;
    }
    const uint32_t t_s = tmem, t_dp = tmem + TILE, t_dq = tmem + 2 * TILE, t_ds = tmem + 3 * TILE;
    const int r0 = first_row(w);
    const int keys = p.causal ? min(w.len, r0 + TILE) : w.len;
    const int n = (keys + TILE - 1) / TILE;
    WaitCtx wc{abort_flag, WAIT_NS};

    if (warp == TMA_WARP) {
        set_registers_down<64>();
        uint32_t side_phase = 0;
        for (int j = 0; j < n; ++j) {
            const int s = j % LONG_STAGES, sv = j % SHORT_STAGES, live = w.len - j * TILE;
            if (!__all_sync(0xffffffffu, mbar_wait(k_empty + 8 * s, ((j / LONG_STAGES) & 1) ^ 1, wc)) ||
                !feed<DP>(ring_k + s * TB, &map_k, k_full + 8 * s, side, side_phase, kv_head, w.start + j * TILE, live, wc))
                break;
            if (!__all_sync(0xffffffffu, mbar_wait(v_empty + 8 * sv, ((j / SHORT_STAGES) & 1) ^ 1, wc)) ||
                !feed<DP>(ring_v + sv * TB, &map_v, v_full + 8 * sv, side, side_phase, kv_head, w.start + j * TILE, live, wc))
                break;
        }
    } else if (warp == MMA_WARP) {
        set_registers_down<64>();
        if (elect_one()) {
            const int ksteps = (p.dim + 15) / 16;
            const uint32_t id_s = idesc_for<FP16>(TILE, false), id_d = idesc_for<FP16>(ksteps * 16, true);
            const uint32_t q = desc_k(smem_u32(smem)), d_o = q + (TB >> 4), k0 = smem_u32(ring_k), v0 = smem_u32(ring_v);
            auto scores = [&](int j, bool here) {
                const int s = j % LONG_STAGES;
                if (!here && !issue_wait(k_full + 8 * s, (j / LONG_STAGES) & 1, wc))
                    return false;
                tc_fence_after();
                multiply_rows<DP>(t_s, q, desc_k(k0 + s * TB), id_s, ksteps);
                umma_commit_cg1(s_full);
                return true;
            };
            auto grads = [&](int j, bool here) {
                const int s = j % SHORT_STAGES;
                if (!here && !issue_wait(v_full + 8 * s, (j / SHORT_STAGES) & 1, wc))
                    return false;
                tc_fence_after();
                multiply_rows<DP>(t_dp, d_o, desc_k(v0 + s * TB), id_s, ksteps);
                umma_commit_cg1(dp_full);
                umma_commit_cg1(v_empty + 8 * s);
                return true;
            };
            auto k_here = [&](int j) { return mbar_test_wait(k_full + 8 * (j % LONG_STAGES), (j / LONG_STAGES) & 1); };
            auto v_here = [&](int j) { return mbar_test_wait(v_full + 8 * (j % SHORT_STAGES), (j / SHORT_STAGES) & 1); };
            bool ok = issue_wait(q_full, 0, wc) && scores(0, false) && grads(0, false);
            for (int j = 0; ok && j < n; ++j) {
                const bool more = j + 1 < n, k_now = more && k_here(j + 1);
                if (more)
                    ok = issue_wait(s_free, j & 1, wc) && scores(j + 1, k_now);
                const bool v_now = more && v_here(j + 1);
                ok = ok && issue_wait(dp_free, j & 1, wc);
                const bool ds_now = ok && mbar_test_wait(ds_ready, j & 1);
                if (ok && more)
                    ok = grads(j + 1, v_now);
                ok = ok && (ds_now || issue_wait(ds_ready, j & 1, wc));
                if (!ok)
                    break;
                tc_fence_after();
                multiply_scores(t_dq, t_ds, desc_mn(k0 + j % LONG_STAGES * TB), id_d, j != 0);
                umma_commit_cg1(k_empty + 8 * (j % LONG_STAGES));
                umma_commit_cg1(dq_done);
            }
            if (ok)
                umma_commit_cg1(done);
        }
        __syncwarp();
    } else if (warp < ROW_WARPS) {
        set_registers_up<104>();
        const int part = warp >> 2;  // 32 columns of every tile
        const int row = (threadIdx.x & 127) + r0;
        const bool live = row < w.len;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const float c = p.scale * LOG2E;
        const int limit = p.causal ? min(w.len, row + 1) : w.len;
        const int64_t at = static_cast<int64_t>(head) * p.tokens + w.start + row;
        const float lse2 = live ? p.lse[at] * LOG2E : 0.f, delta = live ? p.delta[at] : 0.f;
        bool ok = true;
        for (int j = 0; j < n; ++j) {
            const int k0 = j * TILE + part * 32;
            float pr[32], dp[32];
            ok = __all_sync(0xffffffffu, mbar_wait(s_full, j & 1, wc));
            if (!ok)
                break;
            tc_fence_after();
            load_quarter(t_s + part * 32 + lanes, pr);
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(s_free);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                Pair x = f32x2::fma({pr[e], pr[e + 1]}, both(c), both(-lse2));
                x = e / 2 % POLY_OF < POLY ? ex2_pair<true>(x) : ex2_pair<false>(x);
                pr[e] = x.x;
                pr[e + 1] = x.y;
            }
            if (j * TILE + TILE > w.len || (p.causal && j * TILE + TILE > r0)) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (k0 + e >= limit)
                        pr[e] = 0.f;
            }
            ok = __all_sync(0xffffffffu, mbar_wait(dp_full, j & 1, wc));
            if (!ok)
                break;
            tc_fence_after();
            load_quarter(t_dp + part * 32 + lanes, dp);
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(dp_free);
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                const Pair x = f32x2::mul({pr[e], pr[e + 1]}, f32x2::add({dp[e], dp[e + 1]}, both(-delta)));
                pk[e / 2] = pack2<FP16>(x.x, x.y);
            }
            if (j > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(dq_done, (j - 1) & 1, wc));
                if (!ok)
                    break;
                tc_fence_after();
            }
            tmem_st_x16(t_ds + part * 16 + lanes, pk);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(ds_ready);
        }
        if (ok && __all_sync(0xffffffffu, mbar_wait(done, 0, wc))) {
            tc_fence_after();
            store_row<FP16>(t_dq + lanes, part * 32, min(p.dim, part * 32 + 32), p.scale,
                            p.out0 + (w.start + static_cast<int64_t>(row)) * p.row0 + head * p.head0, live);
        }
    } else {
        set_registers_down<64>();
    }
    settle(abort_flag);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA_WARP)
        tmem_dealloc_cg1(tmem, 512);
    if (threadIdx.x == 0 && *abort_flag && p.error_flag != nullptr)
        *p.error_flag = 1;
    if (ends_last)
        wait_for_last_kernel();
}

// ================================================================ backward: dK and dV
//
// A CTA takes 128 keys of one key / value head and walks over the queries of every head of its group; rows of the
// score tiles are keys, so P^T and dS^T are left operands as they stand.  Where there are few tiles of keys, several CTAs
// share the queries of one and leave float32 sums that a last kernel adds up in order.
// Scores and their gradients take turns in one region of TMEM, A; probabilities and score gradients as 16-bit operands
// lie in another, B, so that neither waits for the product that reads the other:
//   tensor cores:  dV += P^T(i-1) dO, A = dP^T(i), dK += dS^T(i-1) Q, A = S^T(i+1), ...
//   row warps:     P(i) from S(i) (in registers: A is free at once)    dS(i) from dP(i)
// (P written over S and dS over dP, so that S(i+1) waited for dV: 3180 cycles an iteration; the products take 2048.)
// The compiler keeps 24 bytes of a thread of this kernel in local memory.
template <int DP, bool FP16>
__global__ void __launch_bounds__(BWD_THREADS, 1)
        dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, const Params p) {
    constexpr int TB = tile_bytes<DP>();
    // K, V, then Q slots, then dO slots, then -lse log2 e and -delta of the rows of two blocks
    extern __shared__ __align__(1024) uint8_t smem[];
    // dQ's last CTA waits for this kernel alone, and what comes after dQ relies on delta's end too: also where no CTA
    // has a tile (empty sequences only), the last one waits for delta.
    const bool ends_last = blockIdx.x == gridDim.x - 1;
    if (unaligned(smem, p)) {
        wait_for_last_kernel();
        return;
    }
    uint8_t *ring_q = smem + 2 * TB, *ring_do = ring_q + LONG_STAGES * TB;
    float* stats = reinterpret_cast<float*>(ring_do + SHORT_STAGES * TB);
    uint64_t* bars = reinterpret_cast<uint64_t*>(stats + SHORT_STAGES * 2 * TILE);
    const uint32_t q_full = smem_u32(bars), q_empty = q_full + 8 * LONG_STAGES, o_full = q_empty + 8 * LONG_STAGES,
                   o_empty = o_full + 8 * SHORT_STAGES;
    const uint32_t st_full = o_empty + 8 * SHORT_STAGES, st_empty = st_full + 8 * SHORT_STAGES;
    const uint32_t kv_full = st_empty + 8 * SHORT_STAGES, s_full = kv_full + 8, s_free = s_full + 8, dp_full = s_free + 8,
                   dp_free = dp_full + 8, ds_ready = dp_free + 8, dk_done = ds_ready + 8,
                   done = dk_done + 8, side = done + 8;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * LONG_STAGES + 4 * SHORT_STAGES + 9);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    Where* where = reinterpret_cast<Where*>(tmem_slot + 2);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const int split = static_cast<int>(blockIdx.x % p.splits), kv_head = static_cast<int>(blockIdx.x / p.splits % p.kv_heads);
    const int group = p.heads / p.kv_heads;
    if (warp == TMA_WARP) {
        if (lane == 0) {
            *abort_flag = 0;
            for (int s = 0; s < 2 * (LONG_STAGES + SHORT_STAGES); ++s)
                mbar_init(q_full + 8 * s, 1);
            for (int s = 0; s < SHORT_STAGES; ++s) {
                mbar_init(st_full + 8 * s, 1);
                mbar_init(st_empty + 8 * s, ROW_WARPS);
            }
            mbar_init(kv_full, 2);
            mbar_init(s_full, 1);
            mbar_init(s_free, ROW_WARPS);
            mbar_init(dp_full, 1);
            mbar_init(dp_free, ROW_WARPS);
            mbar_init(ds_ready, ROW_WARPS);
            mbar_init(dk_done, 1);
            mbar_init(done, 1);
            mbar_init(side, 1);
            mbar_fence_init();
            fence_proxy_async_smem();
        }
        const Where found = find_tile(p, TILE, static_cast<int>(blockIdx.x / p.splits / p.kv_heads));
        __syncwarp();
        if (elect_one()) {
            *where = found;
            if (found.len > 0) {  // the first copies are under way while the rest is set up
                load_tile<DP>(smem_u32(smem), &map_k, kv_full, kv_head, found.start + found.local * TILE);
                load_tile<DP>(smem_u32(smem) + TB, &map_v, kv_full, kv_head, found.start + found.local * TILE);
            }
        }
        __syncwarp();
    } else if (warp == MMA_WARP) {
        tmem_alloc_cg1(smem_u32(tmem_slot), 512);
        tmem_relinquish_cg1();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const Where w = *where;
    const uint32_t tmem = *tmem_slot;
    if (w.len == 0) {  // no such tile
        if (warp == MMA_WARP)
            tmem_dealloc_cg1(tmem, 512);
        if (ends_last)
            wait_for_last_kernel();
        return;
    }
    const uint32_t t_a = tmem, t_p = tmem + TILE, t_ds = t_p + 64, t_dv = tmem + 2 * TILE, t_dk = tmem + 3 * TILE;
    const int k0 = w.local * TILE;               // the first keys, which the most queries see, come first
    const int i0 = p.causal ? w.local : 0;       // first block of queries that sees them
    const int per_head = w.tiles - i0;
    // this CTA's share of the blocks of queries of all heads of the group
    const int all = group * per_head;
    const int first = static_cast<int>(static_cast<int64_t>(all) * split / p.splits);
    const int n = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / p.splits) - first;
    WaitCtx wc{abort_flag, WAIT_NS};

    if (warp == TMA_WARP) {
        set_registers_down<64>();
        uint32_t side_phase = 0;
        for (int it = 0; it < n; ++it) {
            const int s = it % LONG_STAGES, so = it % SHORT_STAGES, head = kv_head * group + (first + it) / per_head;
            const int q0 = (i0 + (first + it) % per_head) * TILE;
            if (!__all_sync(0xffffffffu, mbar_wait(q_empty + 8 * s, ((it / LONG_STAGES) & 1) ^ 1, wc)) ||
                !feed<DP>(ring_q + s * TB, &map_q, q_full + 8 * s, side, side_phase, head, w.start + q0, w.len - q0, wc))
                break;
            if (!__all_sync(0xffffffffu, mbar_wait(o_empty + 8 * so, ((it / SHORT_STAGES) & 1) ^ 1, wc)) ||
                !feed<DP>(ring_do + so * TB, &map_do, o_full + 8 * so, side, side_phase, head, w.start + q0, w.len - q0, wc))
                break;
        }
    } else if (warp == STAT_WARP) {
        set_registers_down<64>();
        // delta has to be complete; and only then may dQ start, which relies on that
        wait_for_last_kernel();
        next_kernel_may_start();
        // -lse log2 e and -delta of every block's rows; a row behind the end has probabilities of zero
        for (int it = 0; it < n; ++it) {
            const int s = it % SHORT_STAGES, head = kv_head * group + (first + it) / per_head, q0 = (i0 + (first + it) % per_head) * TILE;
            if (!__all_sync(0xffffffffu, mbar_wait(st_empty + 8 * s, ((it / SHORT_STAGES) & 1) ^ 1, wc)))
                break;
            float* to = stats + s * 2 * TILE;
            const int64_t at = static_cast<int64_t>(head) * p.tokens + w.start + q0;
            float z[TILE / 32], d[TILE / 32];
#pragma unroll
            for (int i = 0; i < TILE / 32; ++i) {
                const int r = lane + 32 * i;
                const bool live = q0 + r < w.len;
                z[i] = live ? p.lse[at + r] : INFINITY;
                d[i] = live ? p.delta[at + r] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < TILE / 32; ++i) {
                to[lane + 32 * i] = z[i] * -LOG2E;
                to[TILE + lane + 32 * i] = -d[i];
            }
            __syncwarp();
            if (lane == 0)
                mbar_arrive(st_full + 8 * s);
        }
    } else if (warp == MMA_WARP) {
        set_registers_down<64>();
        if (elect_one()) {
            const int ksteps = (p.dim + 15) / 16;
            const uint32_t id_s = idesc_for<FP16>(TILE, false), id_d = idesc_for<FP16>(ksteps * 16, true);
            const uint32_t k = desc_k(smem_u32(smem)), v = k + (TB >> 4), rq = smem_u32(ring_q), ro = smem_u32(ring_do);
            auto q_here = [&](int it) { return mbar_test_wait(q_full + 8 * (it % LONG_STAGES), (it / LONG_STAGES) & 1); };
            auto o_here = [&](int it) { return mbar_test_wait(o_full + 8 * (it % SHORT_STAGES), (it / SHORT_STAGES) & 1); };
            auto scores = [&](int it, bool here) {
                const int s = it % LONG_STAGES;
                if (!here && !issue_wait(q_full + 8 * s, (it / LONG_STAGES) & 1, wc))
                    return false;
                tc_fence_after();
                multiply_rows<DP>(t_a, k, desc_k(rq + s * TB), id_s, ksteps);
                umma_commit_cg1(s_full);
                return true;
            };
            auto grads = [&](int it, bool here) {
                const int s = it % SHORT_STAGES;
                if (!here && !issue_wait(o_full + 8 * s, (it / SHORT_STAGES) & 1, wc))
                    return false;
                tc_fence_after();
                multiply_rows<DP>(t_a, v, desc_k(ro + s * TB), id_s, ksteps);
                umma_commit_cg1(dp_full);
                return true;
            };
            // (P is in place when dP has been read: both are told by one barrier)
            auto add_dv = [&](int it) {
                const int s = it % SHORT_STAGES;
                multiply_scores(t_dv, t_p, desc_mn(ro + s * TB), id_d, it != 0);
                umma_commit_cg1(o_empty + 8 * s);
            };
            auto add_dk = [&](int it, bool here) {
                const int s = it % LONG_STAGES;
                if (!here && !issue_wait(ds_ready, it & 1, wc))
                    return false;
                tc_fence_after();
                multiply_scores(t_dk, t_ds, desc_mn(rq + s * TB), id_d, it != 0);
                umma_commit_cg1(q_empty + 8 * s);
                umma_commit_cg1(dk_done);
                return true;
            };
            // barriers are asked ahead of the products before which they are needed, so that the answers come while
            // others are issued
            bool ok = issue_wait(kv_full, 0, wc) && n > 0 && scores(0, false);  // (the copies are waited for in any case)
            for (int it = 0; ok && it < n; ++it) {
                const bool o_now = o_here(it);
                if (it > 0)
                    add_dv(it - 1);
                ok = issue_wait(s_free, it & 1, wc);
                if (!ok)
                    break;
                const bool ds_now = it > 0 && mbar_test_wait(ds_ready, (it - 1) & 1);
                ok = grads(it, o_now);
                const bool q_now = it + 1 < n && q_here(it + 1);
                ok = ok && (it == 0 || add_dk(it - 1, ds_now)) && issue_wait(dp_free, it & 1, wc);
                if (ok && it + 1 < n)
                    ok = scores(it + 1, q_now);
            }
            if (ok) {
                tc_fence_after();
                add_dv(n - 1);
                ok = add_dk(n - 1, false);
            }
            if (ok)
                umma_commit_cg1(done);
        }
        __syncwarp();
    } else if (warp < ROW_WARPS) {
        set_registers_up<104>();
        const int part = warp >> 2;  // 32 columns (queries) of every tile
        const int key = (threadIdx.x & 127) + k0;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const float c = p.scale * LOG2E;
        bool ok = true;
        for (int it = 0; it < n; ++it) {
            const int s = it % SHORT_STAGES, q0 = (i0 + (first + it) % per_head) * TILE + part * 32;
            const float4* minus_lse = reinterpret_cast<const float4*>(stats + s * 2 * TILE + part * 32);
            const float4* minus_delta = minus_lse + TILE / 4;
            float pr[32], dp[32];
            uint32_t pk[16];
            ok = __all_sync(0xffffffffu, mbar_wait(st_full + 8 * s, (it / SHORT_STAGES) & 1, wc) && mbar_wait(s_full, it & 1, wc));
            if (!ok)
                break;
            tc_fence_after();
            load_quarter(t_a + part * 32 + lanes, pr);
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(s_free);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                const float4 z = minus_lse[e / 4];
                Pair a = f32x2::fma({pr[e], pr[e + 1]}, both(c), {z.x, z.y});
                Pair b = f32x2::fma({pr[e + 2], pr[e + 3]}, both(c), {z.z, z.w});
                a = e / 2 % POLY_OF < POLY ? ex2_pair<true>(a) : ex2_pair<false>(a);
                b = (e / 2 + 1) % POLY_OF < POLY ? ex2_pair<true>(b) : ex2_pair<false>(b);
                pr[e] = a.x;
                pr[e + 1] = a.y;
                pr[e + 2] = b.x;
                pr[e + 3] = b.y;
            }
            if (p.causal && (first + it) % per_head == 0) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (q0 + e < key)
                        pr[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e)
                pk[e] = pack2<FP16>(pr[2 * e], pr[2 * e + 1]);
            // (dV of the block before, which reads the last P, came before dP)
            ok = __all_sync(0xffffffffu, mbar_wait(dp_full, it & 1, wc));
            if (!ok)
                break;
            tc_fence_after();
            tmem_st_x16(t_p + part * 16 + lanes, pk);
            load_quarter(t_a + part * 32 + lanes, dp);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(dp_free);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                const float4 d = minus_delta[e / 4];
                const Pair a = f32x2::mul({pr[e], pr[e + 1]}, f32x2::add({dp[e], dp[e + 1]}, {d.x, d.y}));
                const Pair b = f32x2::mul({pr[e + 2], pr[e + 3]}, f32x2::add({dp[e + 2], dp[e + 3]}, {d.z, d.w}));
                pk[e / 2] = pack2<FP16>(a.x, a.y);
                pk[e / 2 + 1] = pack2<FP16>(b.x, b.y);
            }
            if (it > 0) {
                ok = __all_sync(0xffffffffu, mbar_wait(dk_done, (it - 1) & 1, wc));
                if (!ok)
                    break;
                tc_fence_after();
            }
            tmem_st_x16(t_ds + part * 16 + lanes, pk);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(st_empty + 8 * s);
                mbar_arrive(ds_ready);
            }
        }
        const bool live = key < w.len;
        const int64_t at = w.start + static_cast<int64_t>(key);
        const int from = (part & 1) * (DP / 2), to = (part & 1) ? p.dim : min(p.dim, DP / 2);
        float* sums = p.part + (((part < 2 ? 0 : p.splits) + split) * static_cast<int64_t>(p.tokens) + at) * p.kv_heads * p.dim +
                      kv_head * p.dim;
        if (n == 0) {  // (only where there are more CTAs than blocks of queries)
            if (live)
                for (int c = from; c < to; c += 4)
                    *reinterpret_cast<float4*>(sums + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        } else if (ok && __all_sync(0xffffffffu, mbar_wait(done, 0, wc))) {
            tc_fence_after();
            if (p.splits > 1)
                store_sums((part < 2 ? t_dk : t_dv) + lanes, from, to, sums, live);
            else if (part < 2)
                store_row<FP16>(t_dk + lanes, from, to, p.scale, p.out0 + at * p.row0 + kv_head * p.head0, live);
            else
                store_row<FP16>(t_dv + lanes, from, to, 1.f, p.out1 + at * p.row1 + kv_head * p.head1, live);
        }
    } else {
        set_registers_down<64>();
    }
    settle(abort_flag);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA_WARP)
        tmem_dealloc_cg1(tmem, 512);
    if (threadIdx.x == 0 && *abort_flag && p.error_flag != nullptr)
        *p.error_flag = 1;
}

// Sums of the splits in their order, rounded once: dK (times scale) and dV of the rows that sequences cover.  A thread
// takes eight elements.  Bound by reading the partial sums.
template <bool FP16>
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
    const int pieces = p.dim / 8;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, one = static_cast<int64_t>(p.tokens) * p.kv_heads * pieces;
    if (i >= 2 * one)
        return;
    const int which = i >= one ? 1 : 0;
    const int64_t j = i - which * one, at = j / (p.kv_heads * pieces);
    const int kv_head = static_cast<int>(j / pieces % p.kv_heads), c = static_cast<int>(j % pieces) * 8;
    if (p.cu != nullptr && (at < p.cu[0] || at >= p.cu[p.seqs]))
        return;
    const float* sums = p.part + (which * p.splits * static_cast<int64_t>(p.tokens) + at) * p.kv_heads * p.dim + kv_head * p.dim + c;
    float v[8] = {};
    for (int s = 0; s < p.splits; ++s) {
        const float4 a = __ldcs(reinterpret_cast<const float4*>(sums)), b = __ldcs(reinterpret_cast<const float4*>(sums) + 1);
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
        sums += static_cast<int64_t>(p.tokens) * p.kv_heads * p.dim;
    }
    const float f = which ? 1.f : p.scale;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        w[k] = pack2<FP16>(v[2 * k] * f, v[2 * k + 1] * f);
    uint16_t* to = which ? p.out1 + at * p.row1 + kv_head * p.head1 : p.out0 + at * p.row0 + kv_head * p.head0;
    *reinterpret_cast<uint4*>(to + c) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ================================================================ host side
// [tokens, heads, dim] with boxes of 128 rows x 1 head x 64 elements; columns past the dimension and rows
// past the tensor read as zero
bool make_map(CUtensorMap* map, const Tensor& t, int heads, const Problem& p) {
    auto fn = mgk::gemm::get_encode_fn();
    if (fn == nullptr)
        return false;
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(p.dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(p.tokens)};
    cuuint64_t strides[2] = {static_cast<cuuint64_t>(t.head) * 2, static_cast<cuuint64_t>(t.row) * 2};
    cuuint32_t box[3] = {64, 1, TILE};
    cuuint32_t step[3] = {1, 1, 1};
    return fn(map, p.fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, t.p, dims, strides, box, step,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool bad(const Tensor& t) {
    constexpr int64_t most = int64_t{1} << 38;  // strides of a tensor map are below 2^40 bytes
    return t.p == nullptr || (reinterpret_cast<uintptr_t>(t.p) & 15) || t.row <= 0 || t.head <= 0 || t.row % 8 || t.head % 8 ||
           t.row >= most || t.head >= most;
}
bool bad(const Problem& p) {
    // (tiles reach past the last row, and the search for one past the last sequence: their ends have to be numbers too)
    constexpr int most = 0x7fffffff - 4 * TILE;
    return p.tokens < 0 || p.tokens > most || p.heads < 1 || p.kv_heads < 1 || p.heads % p.kv_heads || p.dim < 8 ||
           p.dim > kMaxDim || p.dim % 8 || p.seqs < 0 || p.seqs > most || (p.cu != nullptr && p.seqs < 1) ||
           (reinterpret_cast<uintptr_t>(p.cu) & 3) || !(p.scale > 0.f) || !(p.scale < INFINITY);
}
// CTAs for the tiles of `rows` rows that find_tile numbers, `heads` for each; 0 when there are too many
unsigned grid_for(const Problem& p, int rows, int heads) {
    const int64_t tiles = p.cu != nullptr ? static_cast<int64_t>(p.tokens) / rows + p.seqs : (p.tokens + rows - 1) / rows;
    const int64_t ctas = tiles * heads;
    return ctas > 0x7fffffff ? 0u : static_cast<unsigned>(ctas);
}
Params params(const Problem& p) {
    Params k{};
    k.cu = p.cu;
    k.seqs = p.seqs;
    k.tokens = p.tokens;
    k.heads = p.heads;
    k.kv_heads = p.kv_heads;
    k.dim = p.dim;
    k.causal = p.causal;
    k.scale = p.scale;
    k.error_flag = p.error_flag;
    return k;
}
template <class F>
cudaError_t pick(const Problem& p, F go) {
    using T = std::true_type;
    using N = std::false_type;
    if (p.dim <= 64)
        return p.fp16 ? go(std::integral_constant<int, 64>{}, T{}) : go(std::integral_constant<int, 64>{}, N{});
    return p.fp16 ? go(std::integral_constant<int, 128>{}, T{}) : go(std::integral_constant<int, 128>{}, N{});
}
// Lets `kernel` have its shared memory on the current device, once for each
template <class... P>
cudaError_t allow_smem(void (*kernel)(P...), std::atomic<uint64_t>& done, int smem) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess)
        return e;
    const uint64_t bit = device < 64 ? uint64_t{1} << device : 0;
    if (done.load(std::memory_order_acquire) & bit)
        return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
        done.fetch_or(bit, std::memory_order_release);
    return e;
}
// `early`: the kernel may start before the one in front of it has ended
template <auto KERNEL, class... A>
cudaError_t run(unsigned grid, int threads, int smem, bool early, cudaStream_t stream, const A&... args) {
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(KERNEL, done, smem);
    if (e != cudaSuccess)
        return e;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = threads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = early ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, KERNEL, args...);
    count_launch();
    return e;
}

}  // namespace

cudaError_t launch_forward(const Problem& p, Tensor q, Tensor k, Tensor v, Tensor out, float* lse, cudaStream_t stream) {
    if (bad(p))
        return cudaErrorInvalidValue;
    if (p.tokens == 0)
        return cudaSuccess;
    if (bad(q) || bad(k) || bad(v) || bad(out) || lse == nullptr || (reinterpret_cast<uintptr_t>(lse) & 3))
        return cudaErrorInvalidValue;
    // Two tiles a CTA while that makes a CTA for every processor, else one: a tile alone takes as long as two, which
    // work in turns.  (1000 tokens, 8 heads of 64: 14.8 us with one, 16.9 with two; 16384 tokens, 8 heads: 753 and 437.)
    const int tiles = grid_for(p, 2 * TILE, p.heads) >= 148 ? 2 : 1;
    const unsigned grid = grid_for(p, tiles * TILE, p.heads);
    CUtensorMap mq, mk, mv;
    if (grid == 0 || !make_map(&mq, q, p.heads, p) || !make_map(&mk, k, p.kv_heads, p) || !make_map(&mv, v, p.kv_heads, p))
        return cudaErrorInvalidValue;
    Params a = params(p);
    a.tiles_per_cta = tiles;
    a.out0 = static_cast<uint16_t*>(out.p);
    a.row0 = out.row;
    a.head0 = out.head;
    a.lse = lse;
    return pick(p, [&](auto dp, auto half) {
        constexpr int DP = decltype(dp)::value;
        return run<forward_kernel<DP, decltype(half)::value>>(grid, FWD_THREADS, fwd_smem<DP>(), false, stream, mq, mk, mv, a);
    });
}

// CTAs that share one tile of keys.  A tile takes the heads of its group one after the other, so that with grouped heads
// few tiles mean long ones: then about two CTAs a processor, but no more than the group has heads (dQ runs beside and
// has as long to go for one head).  The whole backward pass on the device: 4096 tokens, 4 heads of 128 in one group, causal:
// 196 us unshared, 111 by two, 66 by four as chosen; 2048 tokens, 16 heads in 2 groups: 202, 115 and, by eight as
// chosen, 78 (by four 70).  Without groups sharing only costs (1000 tokens, 8 heads of 64: 20 us unshared, 23 by two),
// and so it does where there is a CTA for every processor (5003 tokens, 12 heads of 80 in 4 groups, all keys: 359 to
// 390 unshared, 403 by two).
static int splits_for(const Problem& p) {
    const int64_t seqs = p.cu != nullptr ? p.seqs : 1, group = p.heads / p.kv_heads;
    // (where the sequences end is not known here: half a tile is taken to be empty in each)
    const int64_t full = (p.tokens + TILE - 1) / TILE, ctas = ((full > seqs ? full : seqs) + seqs / 2) * p.kv_heads;
    if (ctas >= 148 || p.tokens == 0)
        return 1;
    const int64_t want = (296 + ctas - 1) / ctas, most = group < 16 ? group : 16;
    return static_cast<int>(want < most ? want : most);
}

size_t backward_workspace(const Problem& p) {
    if (bad(p))
        return 0;
    const size_t rows = static_cast<size_t>(p.tokens) * p.heads, splits = splits_for(p);
    const size_t part = splits > 1 ? 2 * splits * p.tokens * p.kv_heads * p.dim : 0;
    return ((rows + 3) / 4 * 4 + part) * sizeof(float);
}

cudaError_t launch_backward(const Problem& p, Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, const float* lse,
                            Tensor dq, Tensor dk, Tensor dv, void* workspace, cudaStream_t stream) {
    if (bad(p))
        return cudaErrorInvalidValue;
    if (p.tokens == 0)
        return cudaSuccess;
    if (bad(dout) || bad(q) || bad(k) || bad(v) || bad(out) || bad(dq) || bad(dk) || bad(dv) || lse == nullptr || workspace == nullptr ||
        (reinterpret_cast<uintptr_t>(lse) & 3) || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return cudaErrorInvalidValue;
    const int splits = splits_for(p);
    const unsigned grid_q = grid_for(p, TILE, p.heads), grid_k = grid_for(p, TILE, p.kv_heads * splits);
    const int64_t rows = static_cast<int64_t>(p.tokens) * p.heads, joined = 2 * static_cast<int64_t>(p.tokens) * p.kv_heads * (p.dim / 8);
    float* delta = static_cast<float*>(workspace);
    CUtensorMap mq, mk, mv, mo;
    if (grid_q == 0 || grid_k == 0 || (rows + 15) / 16 > 0x7fffffff || joined / 256 >= 0x7fffffff || !make_map(&mq, q, p.heads, p) ||
        !make_map(&mk, k, p.kv_heads, p) || !make_map(&mv, v, p.kv_heads, p) || !make_map(&mo, dout, p.heads, p))
        return cudaErrorInvalidValue;
    auto delta_go = [&](auto kernel) {
        kernel<<<static_cast<unsigned>((rows + 15) / 16), 256, 0, stream>>>(
                static_cast<const uint16_t*>(out.p), out.row, out.head, static_cast<const uint16_t*>(dout.p), dout.row, dout.head,
                p.tokens, p.heads, p.dim, delta);
    };
    p.fp16 ? delta_go(delta_kernel<true>) : delta_go(delta_kernel<false>);
    count_launch();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess)
        return e;
    Params a = params(p);
    a.lse = const_cast<float*>(lse);
    a.delta = delta;
    a.splits = splits;
    a.part = delta + (rows + 3) / 4 * 4;
    return pick(p, [&](auto dp, auto half) {
        constexpr int DP = decltype(dp)::value;
        constexpr bool FP16 = decltype(half)::value;
        a.out0 = static_cast<uint16_t*>(dk.p);
        a.row0 = dk.row;
        a.head0 = dk.head;
        a.out1 = static_cast<uint16_t*>(dv.p);
        a.row1 = dv.row;
        a.head1 = dv.head;
        const cudaError_t first = run<dkv_kernel<DP, FP16>>(grid_k, BWD_THREADS, bwd_smem<DP>(), true, stream, mq, mk, mv, mo, a);
        if (first != cudaSuccess)
            return first;
        Params b = a;
        b.out0 = static_cast<uint16_t*>(dq.p);
        b.row0 = dq.row;
        b.head0 = dq.head;
        const cudaError_t second = run<dq_kernel<DP, FP16>>(grid_q, BWD_THREADS, bwd_smem<DP>(), true, stream, mq, mk, mv, mo, b);
        if (second != cudaSuccess || splits == 1)
            return second;
        join_kernel<FP16><<<static_cast<unsigned>((joined + 255) / 256), 256, 0, stream>>>(a);
        count_launch();
        return cudaGetLastError();
    });
}

}  // namespace attn
}  // namespace mgk
