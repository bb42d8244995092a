// tcgen05 tile loop for a few queries against fp32 rows, which it splits itself.
//
// The rows are read from HBM once, as they are: eight converter warps load a K
// block of a tile, split every value into three bf16 planes hi + mid + lo (24
// bits: nothing is lost) and write them to shared memory in the layout the MMAs
// read; the other operand (at most 128 rows: the queries' planes, or those of G)
// comes by TMA.  The alternative, a pass that writes the planes to memory first,
// moves five times the bytes.  Six products of planes make a K block, as in
// tile_tc.cuh.
//
// One CTA per SM, tiles of 128 x 128, K blocks of 64:
//   warp 0        TMA producer of A's planes (3 boxes a stage)
//   warp 1        TMEM; lane 0 issues the MMAs.  Two accumulators of 2 x 128
//                 columns: the product of the largest planes, and the others, so
//                 that the cut at every instruction (towards zero) touches the
//                 large sum 4 times a K block and not 24
//   warps 2..9    converters: two rows' 256 bytes per load, the next K block's
//                 loads in flight while this one is split; P::kBMn says which
//                 way B lies (below)
//   warps 10..17  epilogue, two per TMEM lane quadrant; policies as in
//                 tile_tc.cuh
// A stage is 96 KB (three planes of both operands): two of them.  Per K block the
// MMAs read 192 KB of operands, 96 KB are written, 32 KB pass through L1: 2,500
// cycles of shared memory at 128 bytes a cycle, where the products alone take
// 1,536.  128 x 100,000 x 768 forward: 144 us, of which that explains 92 (the rows'
// HBM time is 47); with two stages a late converter or commit holds up everything.
// With 256 MB written before the call 159, by planes in memory 326.
//
// B is K-major (tile rows = matrix rows, K along the row) or MN-major (tile rows
// = matrix columns, K = matrix rows).
#pragma once

#include "tile_tc.cuh"

namespace rdb {
namespace {

constexpr int TF_N = 128;
constexpr int TF_STAGES = 2;
constexpr int TF_PLANE = 16384;  // 128 rows x 64 bf16, or 2 blocks of 64 columns x 64 K rows
constexpr int TF_STAGE_BYTES = 6 * TF_PLANE;
constexpr int TF_CONV_WARPS = 8, TF_EPI_WARPS = 8;
constexpr int TF_GROUPS = TF_EPI_WARPS / 4;
constexpr int TF_THREADS = 64 + 32 * (TF_CONV_WARPS + TF_EPI_WARPS);
constexpr int TF_SMEM = TF_STAGES * TF_STAGE_BYTES + TF_EPI_WARPS * TT_STG_BYTES + TT_BAR_BYTES + 1024;
static_assert(TF_SMEM <= 232448, "shared memory over 227 KB");

// fp32 matrix [n, d], row stride ld elements, 16-byte aligned rows
struct F32Rows {
    const float* p;
    int64_t ld, n;
    int d;
};

__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// One converter lane's share of a K block: 8 groups of 4 neighbouring floats.
// Group i of warp w (0..7), lane l:
//   K-major   tile row 16 w + 2 i + l / 16, K element 4 (l % 16)
//   MN-major  K row 8 w + i, column 4 l
// so a warp's load is two whole 256-byte pieces of rows, or one of 512 bytes.
struct TfSource {
    const float* p;  // group 0
    int64_t step;    // elements from one group to the next
    int rows;        // groups i with 2 i < rows (K-major), i < rows (MN-major) exist
    int cols;        // columns of the matrix from this lane's first on
};

__device__ __forceinline__ TfSource tf_source(const F32Rows& x, const TileJob& j, int kb, int w, int lane) {
    TfSource s;
    int64_t row, left;
    int col;
    if (j.b_mn) {
        row = static_cast<int64_t>(j.k0 + kb) * 64 + 8 * w;
        col = j.n0 + 4 * lane;
        left = x.n - row;
        s.step = x.ld;
    } else {
        const int r = 16 * w + lane / 16;
        row = static_cast<int64_t>(j.n0) + r;
        col = (j.k0 + kb) * 64 + 4 * (lane & 15);
        left = min(x.n - row, static_cast<int64_t>(j.nn - r));
        s.step = 2 * x.ld;
    }
    s.rows = static_cast<int>(max(static_cast<int64_t>(0), min(left, static_cast<int64_t>(16))));
    s.cols = x.d - col;
    s.p = x.p + row * x.ld + col;
    return s;
}

__device__ __forceinline__ float4 tf_load(const TfSource& s, bool mn, int i) {
    const bool in = (mn ? i : 2 * i) < s.rows;
    const float* p = s.p + i * s.step;
    if (in && s.cols >= 4) return *reinterpret_cast<const float4*>(p);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (in && s.cols > 0) {
        // the row's last columns: nothing behind them is read
        v.x = p[0];
        if (s.cols > 1) v.y = p[1];
        if (s.cols > 2) v.z = p[2];
    }
    return v;
}

// Asks for a K block's lines in L2, some K blocks ahead of its loads.
constexpr int TF_AHEAD = 5;
__device__ __forceinline__ void tf_prefetch(const F32Rows& x, const TileJob& j, int kb, int w, int lane) {
    if (kb >= j.nk) return;
    // one lane per 128-byte line
    if (j.b_mn) {
        // 8 rows of 512 bytes
        const int64_t row = static_cast<int64_t>(j.k0 + kb) * 64 + 8 * w + lane / 4;
        const int col = j.n0 + 32 * (lane & 3);
        if (row < x.n && col < x.d)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(x.p + row * x.ld + col) : "memory");
    } else {
        // 16 rows of 256 bytes
        const int r = 16 * w + lane / 2;
        const int64_t row = static_cast<int64_t>(j.n0) + r;
        const int col = (j.k0 + kb) * 64 + 32 * (lane & 1);
        if (row < x.n && r < j.nn && col < x.d)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(x.p + row * x.ld + col) : "memory");
    }
}

__device__ __forceinline__ uint32_t tf_pack(float a, float b) {
    uint32_t r;  // a in the low half
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

// the three planes of group i, 8 bytes each
__device__ __forceinline__ void tf_store(bool mn, int i, int w, int lane, const float4& v, uint8_t* planes) {
    uint32_t off;
    if (mn) {
        const int k = 8 * w + i, c = 4 * lane;  // 64-column block, K row, 16-byte unit, swizzled by the row
        off = static_cast<uint32_t>((c >> 6) * TT_BLOCK_BYTES + k * 128 + ((((c & 63) >> 3) ^ (k & 7)) << 4) +
                                    ((c & 4) << 1));
    } else {
        const int r = 16 * w + 2 * i + lane / 16, c = 4 * (lane & 15);
        off = static_cast<uint32_t>(r * 128 + (((c >> 3) ^ (r & 7)) << 4) + ((c & 4) << 1));
    }
    float a = v.x, b = v.y, c = v.z, d = v.w;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const uint32_t lo = tf_pack(a, b), hi = tf_pack(c, d);
        *reinterpret_cast<uint2*>(planes + k * TF_PLANE + off) = make_uint2(lo, hi);
        if (k == 2) break;
        // what is left for the next plane: exact in fp32
        a -= __uint_as_float(lo << 16);
        b -= __uint_as_float(lo & 0xffff0000u);
        c -= __uint_as_float(hi << 16);
        d -= __uint_as_float(hi & 0xffff0000u);
    }
}

// Writes the K block in v to `planes`, and every group's successor from `next`
// into its place as soon as it is written: a load has the time of a whole K
// block to arrive.
template <bool MN>
__device__ __forceinline__ void tf_convert(int w, int lane, float4 (&v)[8], uint8_t* planes, const TfSource& next,
                                           bool more) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        tf_store(MN, i, w, lane, v[i], planes);
        if (more) v[i] = tf_load(next, MN, i);
    }
}

template <class P>
__device__ __forceinline__ void tile_loop_f32(uint8_t* smem_raw, const P& p, const F32Rows& x, const TileStatus st) {
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* stg = smem + TF_STAGES * TF_STAGE_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(stg + TF_EPI_WARPS * TT_STG_BYTES);
    uint64_t* empty = full + TF_STAGES;
    uint64_t* tfull = empty + TF_STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* mma_done = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = static_cast<int>(blockIdx.x), nctas = static_cast<int>(gridDim.x);

    if (threadIdx.x == 0) {
        for (int s = 0; s < TF_STAGES; ++s) {
            mbar_init(&full[s], 1 + TF_CONV_WARPS);
            mbar_init(&empty[s], 1);
        }
        for (int c = 0; c < 2; ++c) {
            mbar_init(&tfull[c], 1);
            mbar_init(&tempty[c], TF_EPI_WARPS);
        }
        mbar_init(mma_done, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc_t<false>(tmem_slot, 4 * TF_N);
        tmem_relinquish_t<false>();
    }
    chain_wait();  // what is above touches no global memory
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            // ---------------------------------------------- TMA producer (A)
            int stage = 0;
            uint32_t phase = 0, issued_mask = 0, issued_phase = 0;
            bool ok = true;
            typename P::Job j;
            typename P::Iter it(p, cta, nctas);
            while (ok && it.next(j)) {
                for (int kb = 0; kb < j.nk; ++kb) {
                    if (!mbar_try_wait(&empty[stage], phase ^ 1) && !mbar_wait(&empty[stage], phase ^ 1, abort_flag)) {
                        ok = false;
                        break;
                    }
                    uint8_t* sa = smem + stage * TF_STAGE_BYTES;
                    mbar_arrive_expect_tx(&full[stage], 3u * static_cast<uint32_t>(j.a_rows) * 128u);
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        tma_load_3d(j.ma, &full[stage], sa + k * TF_PLANE, (j.k0 + kb) * 64, j.m0, k);
                    issued_mask |= 1u << stage;
                    issued_phase = (issued_phase & ~(1u << stage)) | (phase << stage);
                    if (++stage == TF_STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!ok) {
                tt_give_up(abort_flag, st, DEV_TIMEOUT_PRODUCER);
                // let the loads land before the shared memory is released (the
                // stage's phase may also wait for converters that gave up)
                for (int s = 0; s < TF_STAGES; ++s)
                    if (issued_mask & (1u << s)) {
                        const uint64_t t0 = globaltimer_ns();
                        while (!mbar_try_wait(&full[s], (issued_phase >> s) & 1) &&
                               globaltimer_ns() - t0 < kWaitLimitNs) {
                        }
                    }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // ---------------------------------------------- MMA issuer
            int stage = 0;
            uint32_t phase = 0, tile = 0;
            bool ok = true, any = false;
            typename P::Job j;
            typename P::Iter it(p, cta, nctas);
            for (; ok && it.next(j); ++tile) {
                const int acc = tile & 1;
                if (!mbar_wait(&tempty[acc], ((tile >> 1) & 1) ^ 1, abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * 2 * TF_N);
                const uint32_t idesc = tc_idesc(true, 128, TF_N) | (j.b_mn ? 1u << 16 : 0u);
                for (int kb = 0; kb < j.nk; ++kb) {
                    if (!mbar_try_wait(&full[stage], phase) && !mbar_wait(&full[stage], phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(smem + stage * TF_STAGE_BYTES);
#pragma unroll 1
                    for (int g = 0; g < 6; ++g) {
                        const uint64_t adesc = make_sdesc(a_addr + kSegA[g] * TF_PLANE);
                        const uint32_t b_addr = a_addr + (3 + kSegB[g]) * TF_PLANE;
                        const uint64_t bdesc = j.b_mn ? make_sdesc_mn(b_addr) : make_sdesc(b_addr);
                        const uint64_t b_step = j.b_mn ? 128 : 2;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f16(d_tmem + (g < 5 ? TF_N : 0), adesc + 2 * k, bdesc + b_step * k, idesc,
                                     (kb > 0 || k > 0 || (g > 0 && g < 5)) ? 1u : 0u);
                    }
                    any = true;
                    umma_commit(&empty[stage]);
                    if (++stage == TF_STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (ok) umma_commit(&tfull[acc]);
            }
            if (!ok) tt_give_up(abort_flag, st, DEV_TIMEOUT_MMA);
            if (any) {
                umma_commit(mma_done);
                const uint64_t t0 = globaltimer_ns();
                while (!mbar_try_wait(mma_done, 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
                }
            }
        }
    } else if (warp < 2 + TF_CONV_WARPS) {
        // -------------------------------------------------- converters (B)
        const int w = warp - 2;
        int stage = 0;
        uint32_t phase = 0;
        typename P::Job j, jn;
        typename P::Iter it(p, cta, nctas);
        bool more = it.next(jn);
        float4 v[8];
        if (more) {
            const TfSource src = tf_source(x, jn, 0, w, lane);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = tf_load(src, P::kBMn, i);
            for (int kb = 1; kb < TF_AHEAD; ++kb) tf_prefetch(x, jn, kb, w, lane);
        }
        bool ok = true;
        while (ok && more) {
            j = jn;
            more = it.next(jn);
            for (int kb = 0; kb < j.nk; ++kb) {
                const bool inner = kb + 1 < j.nk;
                const TfSource next = inner ? tf_source(x, j, kb + 1, w, lane) : tf_source(x, jn, 0, w, lane);
                if (kb + TF_AHEAD < j.nk)
                    tf_prefetch(x, j, kb + TF_AHEAD, w, lane);
                else if (more)
                    tf_prefetch(x, jn, kb + TF_AHEAD - j.nk, w, lane);
                if (!__all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, abort_flag))) {
                    ok = false;
                    break;
                }
                tf_convert<P::kBMn>(w, lane, v, smem + stage * TF_STAGE_BYTES + 3 * TF_PLANE, next, inner || more);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[stage]);
                if (++stage == TF_STAGES) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        if (!ok) tt_give_up(abort_flag, st, DEV_TIMEOUT_PRODUCER);
    } else {
        // -------------------------------------------------- epilogue
        TileCtx ctx;
        ctx.quad = warp & 3;
        ctx.grp = (warp - 2 - TF_CONV_WARPS) >> 2;
        ctx.col0 = ctx.grp * 32;
        ctx.col1 = ctx.col0 + TF_GROUPS * 32;
        ctx.lane = lane;
        ctx.row = ctx.quad * 32 + lane;
        ctx.stg = stg + (warp - 2 - TF_CONV_WARPS) * TT_STG_BYTES;
        typename P::Epi epi;
        typename P::Job j;
        typename P::Iter it(p, cta, nctas);
        uint32_t tile = 0;
        for (; it.next(j); ++tile) {
            const int acc = tile & 1;
            p.begin(epi, j, ctx);
            if (!__all_sync(0xffffffffu, mbar_wait(&tfull[acc], (tile >> 1) & 1, abort_flag))) {
                tt_give_up(abort_flag, st, DEV_TIMEOUT_EPILOGUE);
                break;
            }
            tc_fence_after();
            const uint32_t tbase =
                tmem_base + (static_cast<uint32_t>(ctx.quad * 32) << 16) + static_cast<uint32_t>(acc * 2 * TF_N);
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
                const int col = h ? ctx.col1 : ctx.col0;
                uint32_t ra[32], rb[32];
                tmem_ld32_async(tbase + static_cast<uint32_t>(col), ra);
                tmem_ld32_async(tbase + static_cast<uint32_t>(TF_N + col), rb);
                tmem_ld_wait(ra);
                tmem_ld_wait(rb);
#pragma unroll
                for (int i = 0; i < 32; ++i) ra[i] = __float_as_uint(__uint_as_float(ra[i]) + __uint_as_float(rb[i]));
                if (h) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&tempty[acc]);
                }
                if (col < j.nn) p.chunk(epi, j, ctx, col, ra);
                __syncwarp();
            }
            p.end(epi, j, ctx);
        }
        p.finish(ctx);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_t<false>(tmem_base, 4 * TF_N);
    }
}

template <class K>
int tile_f32_smem_attr(K kernel, bool (&done)[64]) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && done[dev]) return RDB_OK;
    RDB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TF_SMEM));
    if (dev >= 0 && dev < 64) done[dev] = true;
    return RDB_OK;
}

}  // namespace
}  // namespace rdb
