// Persistent tcgen05 tile loop shared by the int8 scores (sq8_dot.cu) and the
// softmax cross entropy (xent.cu).
//
// A CTA pair (cluster of 2, cta_group::2) computes one 256 x nn tile after the
// other, nn <= 256, D = sum_k A[m, k] B[n, k]:
//   warp 0      TMA producer: per K block of 128 bytes each CTA loads its 128
//               rows of A and its nn / 2 rows of B into a ring of 5 to 7 stages
//               (4 to 6 measure the same where the MMAs bound the tile).
//   warp 1      TMEM (two to eight accumulators, P::kAccCols); the leader's lane 0 issues
//               the MMAs and commits stage releases and finished accumulators.
//   warps 2..17 epilogue, four per TMEM lane quadrant: a thread owns one row of
//               its CTA's 128 and every fourth 32-column chunk of the tile (at
//               most two).  It takes both into registers and releases the
//               accumulator before it works on them, so the MMAs run ahead by up
//               to as many tiles as there are accumulators, 512 / P::kAccCols.  (4,096 x 131,072 x 128 forward: 219 us, 306 with
//               eight warps and one chunk in flight, 137 with no epilogue at
//               all; at d = 768 586, 613 and 556 us.)
// An operand lies either K-major in memory (a row's K elements contiguous: one
// box of 128 bytes x 128 rows per stage) or MN-major (the rows' index
// contiguous: boxes of 64 elements x 64 K rows).  Both use the 128-byte
// swizzle, whose 8-row atoms are 1024 bytes apart along the other axis; an
// MN-major operand's 64-element blocks are 8192 bytes apart.
//
// fp32 operands come as three bf16 planes hi + mid + lo (24 bits, so nothing
// is lost); six products of planes, the ones of at least 2^-18 of the largest,
// are walked as one long K axis.  What they leave out is below 2^-25.
//
// A policy P supplies the tiles and what becomes of them:
//   P::kInt8                       int8 operands, int32 accumulators
//   P::kStages, P::kStgBytes       ring stages, staging bytes per epilogue warp
//   P::kAccCols                    columns of an accumulator: the widest tile.  256: two
//                                  of them; 64 or 128: eight or four, and the epilogue's
//                                  warps take turns.  A tile of few columns and K blocks
//                                  is shorter than the way from its MMAs through the
//                                  epilogue back to a free accumulator (1M x 128 int8
//                                  rows, 32 queries: 82 us with two, 56 with eight).
//   P::Job                         TileJob and what the epilogue needs with it
//   P::Iter(p, pair, npairs)       the pair's tiles: bool next(job), the same
//                                  sequence in every role
//   P::Epi                         per-thread epilogue state
//   p.begin(epi, job, ctx)         while the tile is still being multiplied
//   p.chunk(epi, job, ctx, col, r) 32 accumulators of the warp's rows, from
//                                  column col on (two chunks where the tile is
//                                  that wide)
//   p.end(epi, job, ctx)           after the tile's chunks
//   p.finish(ctx)                  once, after the last tile
// The epilogue's warps never wait for one another: they drift apart by up to as
// many tiles (two of 256 columns, eight of 64), so that one's exponentials overlap
// another's maxima and stores.
//
// Every mbarrier wait is bounded: a role that gives up raises the CTA's abort
// flag and the device status word (also in its host copy), waits (bounded) for
// what it has in flight, and the CTA frees its TMEM and exits.
#pragma once

#include "chain.cuh"
#include "tc_common.cuh"

namespace rdb {
namespace {

constexpr int TT_M = 256;         // rows of a pair's tile
constexpr int TT_N = 256;         // largest columns of a tile
constexpr int TT_MAX_STAGES = 7;
constexpr int TT_MAX_ACCS = 8;    // accumulators of 64 columns in TMEM
constexpr int TT_A_BYTES = 16384;  // 128 rows x 128 bytes
constexpr int TT_STAGE_BYTES = 2 * TT_A_BYTES;
constexpr int TT_BLOCK_BYTES = 8192;  // 64 elements x 64 K rows (MN-major)
constexpr int TT_EPI_WARPS = 16;
constexpr int TT_GROUPS = TT_EPI_WARPS / 4;  // warps per TMEM lane quadrant
constexpr int TT_THREADS = 64 + 32 * TT_EPI_WARPS;
constexpr int TT_BAR_BYTES = 256;
constexpr int TT_STG_BYTES = 4096;  // staging for 32 rows x 32 fp32 columns on their way out
// every policy's shared memory: 7 stages, or 5 and staging for the stores
constexpr int TT_SMEM = TT_MAX_STAGES * TT_STAGE_BYTES + TT_BAR_BYTES + 1024;
static_assert(TT_SMEM <= 232448, "shared memory over 227 KB");

// products of planes (A plane, B plane), the largest last: an accumulator is cut
// (rounded towards zero) at every instruction, which costs a sum least while it
// is small
__device__ constexpr int kSegA[6] = {1, 2, 0, 1, 0, 0};
__device__ constexpr int kSegB[6] = {1, 0, 2, 0, 1, 0};

struct TileJob {
    const CUtensorMap *ma, *mb;  // 3-D maps: (contiguous axis, rows, planes)
    int m0, n0;                  // first row of the pair's tile, first column
    int nn;                      // columns: a multiple of 32 (64 per CTA and block when b_mn)
    int k0, nk;                  // first K block and K blocks per product
    int nseg;                    // products of planes, the last of kSegA / B: 1 or 6
    bool a_mn, b_mn;
    // rows of a CTA's box where the operand is K-major (the maps' box rows, a
    // multiple of 8 up to 128).  A needs only the rows that exist: what an MMA
    // reads behind them ends in accumulator rows that nobody uses.
    int a_rows, b_rows;
    bool a_second;               // the pair's second CTA has rows of A at all
};

__device__ __forceinline__ void tma_load_3d_pair(const CUtensorMap* map, uint32_t bar_cluster, void* dst, int x, int y,
                                                 int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z)
        : "memory");
}

__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// MN-major, SWIZZLE_128B: 64-element blocks TT_BLOCK_BYTES apart (leading
// offset), groups of 8 K rows 1024 bytes apart (stride offset)
__device__ __forceinline__ uint64_t make_sdesc_mn(uint32_t saddr) {
    uint64_t desc = 0;
    desc |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
    desc |= static_cast<uint64_t>(TT_BLOCK_BYTES >> 4) << 16;
    desc |= static_cast<uint64_t>(1024 >> 4) << 32;
    desc |= static_cast<uint64_t>(1) << 46;
    desc |= static_cast<uint64_t>(2) << 61;
    return desc;
}

// kind::i8 with signed operands and int32 accumulators, K-major
__device__ __forceinline__ constexpr uint32_t tc_idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(m >> 4) << 24);
}

// What an epilogue thread knows of its place.
struct TileCtx {
    int row;        // row of the pair's tile
    int quad, grp;  // TMEM lane quadrant, which of its warps
    int col0, col1; // first columns of its two chunks
    int lane;
    uint8_t* stg;   // the warp's P::kStgBytes (1024-byte aligned if they are a multiple)
};

// ---- staged stores: a warp writes 32 rows of 64 or 128 bytes to its staging
// bytes in the tensor map's swizzle (conflict-free: every lane its own row) and
// one lane sends them with a TMA store, which clips at the matrix's edges.

// byte offset of 16-byte unit u of row r: rows of 128 bytes, 128-byte swizzle
__device__ __forceinline__ uint32_t stg_off128(int r, int u) {
    return static_cast<uint32_t>(r * 128 + ((u ^ (r & 7)) << 4));
}
// rows of 64 bytes, 64-byte swizzle
__device__ __forceinline__ uint32_t stg_off64(int r, int u) {
    return static_cast<uint32_t>(r * 64 + ((u ^ ((r >> 1) & 3)) << 4));
}

// the staging bytes may be written again
__device__ __forceinline__ void stg_wait_read(int lane) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}

template <bool ADD>
__device__ __forceinline__ void stg_send(const CUtensorMap* map, const void* src, int lane, int x, int y, int z) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
        if (ADD)
            asm volatile(
                "cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                    reinterpret_cast<uint64_t>(map)),
                "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
                : "memory");
        else
            asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                             reinterpret_cast<uint64_t>(map)),
                         "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
                         : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}

// everything sent has been written
__device__ __forceinline__ void stg_drain(int lane) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
}

__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

struct TileStatus {
    unsigned *word, *mirror;  // device status word, its copy in mapped host memory
};

__device__ __forceinline__ void tt_give_up(volatile int* abort_flag, const TileStatus& st, unsigned code) {
    *abort_flag = 1;
    if (st.word) atomicOr(st.word, code);
    if (st.mirror) atomicOr_system(st.mirror, code);
}

// The body of a kernel launched with __cluster_dims__(2, 1, 1), TT_THREADS
// threads and TT_SMEM bytes.  bf16: operand type of the 16-bit kinds.
template <class P>
__device__ __forceinline__ void tile_loop(uint8_t* smem_raw, const P& p, const bool bf16, const TileStatus st) {
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int TT_STAGES = P::kStages;
    static_assert(TT_STAGES <= TT_MAX_STAGES &&
                      TT_STAGES * TT_STAGE_BYTES + TT_EPI_WARPS * P::kStgBytes <= TT_MAX_STAGES * TT_STAGE_BYTES,
                  "stages and staging over the block's shared memory");
    uint8_t* stg = smem + TT_STAGES * TT_STAGE_BYTES;
    static_assert((2 * TT_STAGES + 2 * TT_MAX_ACCS + 1) * 8 + 8 <= TT_BAR_BYTES, "barriers over their bytes");
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + TT_MAX_STAGES * TT_STAGE_BYTES);
    uint64_t* empty = full + TT_STAGES;
    uint64_t* tfull = empty + TT_STAGES;
    uint64_t* tempty = tfull + TT_MAX_ACCS;
    uint64_t* mma_done = tempty + TT_MAX_ACCS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const int pair = static_cast<int>(blockIdx.x >> 1), npairs = static_cast<int>(gridDim.x >> 1);
    constexpr int kElems = P::kInt8 ? 128 : 64;  // elements of 128 bytes

    if (threadIdx.x == 0) {
        for (int s = 0; s < TT_STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int c = 0; c < TT_MAX_ACCS; ++c) {
            mbar_init(&tfull[c], 1);
            mbar_init(&tempty[c], 2 * TT_EPI_WARPS);
        }
        mbar_init(mma_done, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc_t<true>(tmem_slot, 512);
        tmem_relinquish_t<true>();
    }
    chain_wait();  // what is above touches no global memory
    tc_fence_before();
    cluster_sync_all();  // both CTAs' barriers initialised before any remote use
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    static_assert(TT_N / 32 <= 2 * TT_GROUPS, "at most two chunks per epilogue warp");
    constexpr int kAccs = 512 / P::kAccCols;
    constexpr bool kNarrow = P::kAccCols <= TT_GROUPS * 32;  // one chunk per epilogue warp at most
    static_assert(P::kAccCols <= TT_N && kAccs <= TT_MAX_ACCS && (kAccs & (kAccs - 1)) == 0, "accumulators");

    if (warp == 0) {
        if (lane == 0) {
            // ---------------------------------------------- TMA producer
            const uint32_t full_lead = map_to_rank(&full[0], 0);
            int stage = 0;
            uint32_t phase = 0, issued_mask = 0, issued_phase = 0;
            bool ok = true;
            typename P::Job j;
            typename P::Iter it(p, pair, npairs);
            while (ok && it.next(j)) {
                const int half = j.nn / 2;
                const int am = j.m0 + static_cast<int>(rank) * 128, bn = j.n0 + static_cast<int>(rank) * half;
                const int b_blocks = j.b_mn ? half / 64 : 2;
                const bool load_a = leader || j.a_second;
                const uint32_t bytes =
                    (j.a_second ? 2u : 1u) * (j.a_mn ? TT_A_BYTES : static_cast<uint32_t>(j.a_rows) * 128u) +
                    2u * (j.b_mn ? static_cast<uint32_t>(b_blocks) * TT_BLOCK_BYTES
                                 : static_cast<uint32_t>(j.b_rows) * 128u);
                for (int g = 0; g < j.nseg && ok; ++g) {
                    const int za = kSegA[6 - j.nseg + g], zb = kSegB[6 - j.nseg + g];
                    for (int kb = 0; kb < j.nk; ++kb) {
                        if (!mbar_try_wait(&empty[stage], phase ^ 1) &&
                            !mbar_wait(&empty[stage], phase ^ 1, abort_flag)) {
                            ok = false;
                            break;
                        }
                        uint8_t* sa = smem + stage * TT_STAGE_BYTES;
                        uint8_t* sb = sa + TT_A_BYTES;
                        const uint32_t bar = full_lead + static_cast<uint32_t>(stage * sizeof(uint64_t));
                        if (leader) mbar_arrive_expect_tx(&full[stage], bytes);
                        const int k = (j.k0 + kb) * kElems;
                        if (!load_a) {
                        } else if (j.a_mn) {
                            tma_load_3d_pair(j.ma, bar, sa, am, k, za);
                            tma_load_3d_pair(j.ma, bar, sa + TT_BLOCK_BYTES, am + 64, k, za);
                        } else {
                            tma_load_3d_pair(j.ma, bar, sa, k, am, za);
                        }
                        if (j.b_mn) {
                            tma_load_3d_pair(j.mb, bar, sb, bn, k, zb);
                            if (b_blocks > 1) tma_load_3d_pair(j.mb, bar, sb + TT_BLOCK_BYTES, bn + 64, k, zb);
                        } else {
                            tma_load_3d_pair(j.mb, bar, sb, k, bn, zb);
                        }
                        issued_mask |= 1u << stage;
                        issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                        if (++stage == TT_STAGES) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                }
            }
            if (!ok) {
                tt_give_up(abort_flag, st, DEV_TIMEOUT_PRODUCER);
                // let the loads tracked by this CTA's barriers land before its
                // shared memory is released
                if (leader)
                    for (int s = 0; s < TT_STAGES; ++s)
                        if (issued_mask & (1u << s)) {
                            const uint64_t t0 = globaltimer_ns();
                            while (!mbar_try_wait(&full[s], (issued_phase >> s) & 1) &&
                                   globaltimer_ns() - t0 < kWaitLimitNs) {
                            }
                        }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            // ---------------------------------------------- MMA issuer
            int stage = 0;
            uint32_t phase = 0, tile = 0;
            bool ok = true, any = false;
            typename P::Job j;
            typename P::Iter it(p, pair, npairs);
            for (; ok && it.next(j); ++tile) {
                const int acc = tile % kAccs;
                if (!mbar_wait(&tempty[acc], ((tile / kAccs) & 1) ^ 1, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * P::kAccCols);
                const uint32_t idesc =
                    P::kInt8 ? tc_idesc_i8(TT_M, j.nn)
                             : tc_idesc(bf16, TT_M, j.nn) | (j.a_mn ? 1u << 15 : 0u) | (j.b_mn ? 1u << 16 : 0u);
                // one instruction covers 32 bytes of K: 2 descriptor units
                // along a K-major row, 16 K rows (128 units) when MN-major
                const uint64_t a_step = j.a_mn ? 128 : 2, b_step = j.b_mn ? 128 : 2;
                const int total = j.nseg * j.nk;
                for (int kb = 0; kb < total; ++kb) {
                    if (!mbar_try_wait(&full[stage], phase) && !mbar_wait(&full[stage], phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(smem + stage * TT_STAGE_BYTES);
                    const uint64_t adesc = j.a_mn ? make_sdesc_mn(a_addr) : make_sdesc(a_addr);
                    const uint64_t bdesc =
                        j.b_mn ? make_sdesc_mn(a_addr + TT_A_BYTES) : make_sdesc(a_addr + TT_A_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t more = (kb > 0 || k > 0) ? 1u : 0u;
                        if (P::kInt8)
                            umma_i8_pair(d_tmem, adesc + a_step * k, bdesc + b_step * k, idesc, more);
                        else
                            umma_f16_pair(d_tmem, adesc + a_step * k, bdesc + b_step * k, idesc, more);
                    }
                    any = true;
                    umma_commit_pair_both(&empty[stage]);
                    if (++stage == TT_STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (ok) umma_commit_pair_both(&tfull[acc]);
            }
            if (!ok) tt_give_up(abort_flag, st, DEV_TIMEOUT_MMA);
            if (any) {
                // every MMA issued here has finished before TMEM is freed
                umma_commit_pair_self(mma_done);
                const uint64_t t0 = globaltimer_ns();
                while (!mbar_try_wait(mma_done, 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
                }
            }
        }
    } else {
        // -------------------------------------------------- epilogue
        TileCtx ctx;
        ctx.quad = warp & 3;  // TMEM lanes this warp may read
        ctx.grp = (warp - 2) >> 2;
        ctx.lane = lane;
        ctx.col0 = ctx.grp * 32;
        ctx.col1 = ctx.col0 + TT_GROUPS * 32;
        ctx.row = static_cast<int>(rank) * 128 + ctx.quad * 32 + lane;
        ctx.stg = stg + (warp - 2) * P::kStgBytes;
        const uint32_t tempty_lead = map_to_rank(&tempty[0], 0);
        typename P::Epi epi;
        typename P::Job j;
        typename P::Iter it(p, pair, npairs);
        uint32_t tile = 0;
        for (; it.next(j); ++tile) {
            const int acc = tile % kAccs;
            // the warps of a quadrant take turns at the columns there are
            if (kNarrow) ctx.col0 = (ctx.grp + static_cast<int>(tile)) % TT_GROUPS * 32;
            p.begin(epi, j, ctx);
            if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], (tile / kAccs) & 1, abort_flag))) {
                tt_give_up(abort_flag, st, DEV_TIMEOUT_EPILOGUE);
                break;
            }
            tc_fence_after();
            const uint32_t tbase =
                tmem_base + (static_cast<uint32_t>(ctx.quad * 32) << 16) + static_cast<uint32_t>(acc * P::kAccCols);
            uint32_t ra[32], rb[32];
            // (columns behind a narrow tile hold older values, and columns that its
            // accumulator does not have are read from its first: no policy uses them)
            tmem_ld32_async(tbase + static_cast<uint32_t>(!kNarrow || ctx.col0 < P::kAccCols ? ctx.col0 : 0), ra);
            if (!kNarrow) tmem_ld32_async(tbase + static_cast<uint32_t>(ctx.col1), rb);
            tmem_ld_wait(ra);
            if (!kNarrow) tmem_ld_wait(rb);
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive_cluster_relaxed(tempty_lead + static_cast<uint32_t>(acc * sizeof(uint64_t)));
            if (ctx.col0 < j.nn) p.chunk(epi, j, ctx, ctx.col0, ra);
            __syncwarp();
            if (!kNarrow && ctx.col1 < j.nn) p.chunk(epi, j, ctx, ctx.col1, rb);
            __syncwarp();
            p.end(epi, j, ctx);
        }
        p.finish(ctx);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // neither CTA leaves while its partner may still signal it
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_t<true>(tmem_base, 512);
    }
}

// ------------------------------------------------------------ host side --

// planes x [rows, cols] matrices (row stride ld_bytes, plane stride
// plane_bytes, any for a single plane) in boxes of 128 bytes x box_rows;
// out-of-range elements read 0
int make_map_3d(CUtensorMap* m, CUtensorMapDataType type, int elem, const void* base, int64_t cols, int64_t rows,
                int64_t planes, int64_t ld_bytes, int64_t plane_bytes, int box_rows) {
    auto fn = encode_fn();
    if (!fn) return set_error(RDB_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    // the stride of a single plane is not used, but has to be below 2^40
    if (planes == 1) plane_bytes = ld_bytes < (1LL << 40) / rows ? ld_bytes * rows : ld_bytes;
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
    cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld_bytes), static_cast<cuuint64_t>(plane_bytes)};
    cuuint32_t box[3] = {static_cast<cuuint32_t>(128 / elem), static_cast<cuuint32_t>(box_rows), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(m, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(RDB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return RDB_OK;
}

// planes x [rows, cols] matrices in boxes of 32 columns x 32 rows, for staged stores
int make_store_map(CUtensorMap* m, CUtensorMapDataType type, int elem, const void* base, int64_t cols, int64_t rows,
                   int64_t planes, int64_t ld_bytes, int64_t plane_bytes) {
    auto fn = encode_fn();
    if (!fn) return set_error(RDB_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    if (planes == 1) plane_bytes = ld_bytes < (1LL << 40) / rows ? ld_bytes * rows : ld_bytes;
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
    cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld_bytes), static_cast<cuuint64_t>(plane_bytes)};
    cuuint32_t box[3] = {32, 32, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(m, type, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    elem == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(RDB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return RDB_OK;
}

// shared memory opt-in, once per kernel and device
template <class K>
int tile_smem_attr(K kernel, bool (&done)[64]) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && done[dev]) return RDB_OK;
    RDB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TT_SMEM));
    if (dev >= 0 && dev < 64) done[dev] = true;
    return RDB_OK;
}

inline TileStatus tile_status() { return {device_status_word(), status_mirror_device()}; }

// box rows of a K-major operand of `rows` rows in tiles of `width` per CTA
inline int tile_box_rows(int64_t rows, int width) {
    return static_cast<int>(rows < width ? (rows + 7) / 8 * 8 : width);
}

inline int tile_pairs() { return num_sms() / 2; }

}  // namespace
}  // namespace rdb
