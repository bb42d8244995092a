// Scores of int8 codes: out[b, n] = qs[b] * xs[n] * sum_t qc[b, t] * xc[n, t].
//
// Both operands are SQ8 rows (sq8.cu): int8 codes and one fp32 scale per row,
// so the scales are per query (token) and per database row (channel).  The
// sum is an exact int32 (|code| <= 128 and d <= kMaxDim, so it stays below
// 2^31); one fp32 product of the two scales and one with the sum follow, and
// fp16 / bf16 outputs are rounded once from that fp32 value.
//
// One or two queries: the codes of the rows are what has to be read, so a
// CUDA-core kernel (dp4a) streams them once past query codes held in shared
// memory (1M x 768: 117 us, 6.6 TB/s).
// Otherwise the tcgen05 tile loop (kind::i8) with the rows as the tile's M: few
// queries then make a narrow tile, and as a thread of the epilogue owns one row,
// a warp's store of one query's scores is 32 consecutive elements and needs no
// staging (staged TMA stores spilled registers and measured the same).  32 x
// 100,000 x 768: 20 us from a cold L2, where the codes' bytes take 12 and the scores'
// 2; 32 x 1M x 768 134, 1.1 times its bytes; 4,096 x 16,384 x 1,024 in bf16: 77 us, of which the products take
// 45 and the conversion and scaling of 67M sums the rest.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "tile_tc.cuh"

namespace rdb {
namespace {

// 131071 * 128 * 128 < 2^31
constexpr int kMaxDim = 131071;

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float score(float qs, float xs, int acc) {
    return __fmul_rn(__fmul_rn(qs, xs), static_cast<float>(acc));
}

// ------------------------------------------------------ one or two queries --

constexpr int GV_THREADS = 256;
constexpr int GV_LANES = 8;               // lanes per row: 128 bytes of a row per load
// 16-byte loads a lane has in flight.  Rows of 768 codes take one batch, longer ones
// end with a part of one, which costs nothing: 1M x 1,024 154 us (6.7 TB/s), 700,000
// x 1,152 123 (6.6), 1M x 768 117 (6.6).
constexpr int GV_BATCH = 6;
constexpr int GV_SMEM = 48 * 1024;        // query codes

// The warps take 4 R rows each in turn (shares of their own, rows far apart, cost
// 5 to 9 %); a lane reads B 16-byte chunks of each of R rows at a time, the whole
// of them where R > 1.
template <typename T, int NQ, int B>
__global__ void __launch_bounds__(GV_THREADS, GV_BATCH / B > 1 ? 3 : 4)
    sq8_few_kernel(const int8_t* qc, const float* qs, int nq, int64_t ldq, const int8_t* xc, const float* xs, int64_t n,
                   int64_t ldx, int d, T* out, int64_t ldo) {
    constexpr int R = GV_BATCH / B, kRows = 32 / GV_LANES;
    extern __shared__ __align__(16) int8_t sq[];  // [NQ][dp], zero behind d and behind nq
    chain_wait();
    const int dp = (d + 15) / 16 * 16, chunks = dp / 16;
    for (int i = threadIdx.x; i < NQ * dp; i += GV_THREADS) {
        const int b = i / dp, t = i - b * dp;
        sq[i] = (b < nq && t < d) ? qc[b * ldq + t] : static_cast<int8_t>(0);
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, sub = lane & (GV_LANES - 1);
    const int full = d / 16;  // 16-byte chunks that lie inside the row
    // A row's last chunk may reach behind d, but not behind the row's stride, which
    // is whole chunks: it is read whole, and the query is zero there.  Only the last
    // row may end with its codes.
    auto load = [&](int64_t r, int c) -> int4 {
        const int8_t* x = xc + r * ldx;
        const bool last = r == n - 1;
        if (c < (last ? full : chunks)) return reinterpret_cast<const int4*>(x)[c];
        uint32_t b[4] = {0u, 0u, 0u, 0u};
        if (last && c < chunks) {
#pragma unroll
            for (int t = 0; t < 16; ++t)
                if (c * 16 + t < d)
                    b[t >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(x[c * 16 + t])) << (8 * (t & 3));
        }
        return make_int4(b[0], b[1], b[2], b[3]);
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * (GV_THREADS / 32) * kRows * R;
    int64_t r0 = (static_cast<int64_t>(blockIdx.x) * (GV_THREADS / 32) + threadIdx.x / 32) * kRows * R + lane / GV_LANES;
    int4 v[R][B];
    float sc[R], sq_b[NQ];
#pragma unroll
    for (int b = 0; b < NQ; ++b) sq_b[b] = b < nq ? qs[b] : 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t r = min(r0 + i * kRows, n - 1);
        sc[i] = xs[r];
#pragma unroll
        for (int k = 0; k < B; ++k) v[i][k] = load(r, sub + k * GV_LANES);
    }
    for (; r0 - lane / GV_LANES < n; r0 += step) {
        int acc[R][NQ];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int b = 0; b < NQ; ++b) acc[i][b] = 0;
        for (int c0 = sub; c0 < chunks; c0 += GV_LANES * B) {
            // the next batch, of this row or of a row of the next step, replaces
            // every chunk as soon as it is used: GV_BATCH loads a lane stay in flight
            const bool more = R == 1 && c0 + GV_LANES * B < chunks;
            const int cn = more ? c0 + GV_LANES * B : sub;
#pragma unroll
            for (int k = 0; k < B; ++k) {
                const int c = min(c0 + k * GV_LANES, chunks - 1);
                int4 q[NQ];
#pragma unroll
                for (int b = 0; b < NQ; ++b) q[b] = *reinterpret_cast<const int4*>(sq + b * dp + c * 16);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const int4 x = v[i][k];
#pragma unroll
                    for (int b = 0; b < NQ; ++b) {
                        acc[i][b] = __dp4a(x.x, q[b].x, acc[i][b]);
                        acc[i][b] = __dp4a(x.y, q[b].y, acc[i][b]);
                        acc[i][b] = __dp4a(x.z, q[b].z, acc[i][b]);
                        acc[i][b] = __dp4a(x.w, q[b].w, acc[i][b]);
                    }
                    v[i][k] = load(min(r0 + i * kRows + (more ? 0 : step), n - 1), cn + k * GV_LANES);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t r = r0 + i * kRows;
            const float s = sc[i];
            sc[i] = xs[min(r + step, n - 1)];
#pragma unroll
            for (int b = 0; b < NQ; ++b) {
                int a = acc[i][b];
#pragma unroll
                for (int o = GV_LANES / 2; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
                if (((i * NQ + b) & (GV_LANES - 1)) == sub && r < n && b < nq)
                    out[b * ldo + r] = from_f<T>(score(sq_b[b], s, a));
            }
        }
    }
}

template <typename T, int NQ>
int launch_few(const int8_t* qc, const float* qs, int64_t nq, int64_t ldq, const int8_t* xc, const float* xs,
               int64_t n, int64_t ldx, int d, void* out, int64_t ldo, cudaStream_t s) {
    // the whole row in as few loads as it takes, or GV_BATCH at a time: 4M x 128
    // in 102 us, 2M x 384 in 121 (GV_BATCH for all: 200 and 129)
    const auto kernel = d <= 128   ? sq8_few_kernel<T, NQ, 1>
                        : d <= 256 ? sq8_few_kernel<T, NQ, 2>
                        : d <= 512 ? sq8_few_kernel<T, NQ, 4>
                                   : sq8_few_kernel<T, NQ, GV_BATCH>;
    const int64_t rows = GV_THREADS / GV_LANES * (d <= 128 ? 6 : d <= 256 ? 3 : 1);
    const int64_t blocks = std::min<int64_t>((n + rows - 1) / rows, (d <= 256 ? 3LL : 4LL) * num_sms());
    return launch_chained(kernel, (unsigned)blocks, GV_THREADS, static_cast<size_t>(NQ) * ((d + 15) / 16 * 16), s, qc, qs,
                          (int)nq, ldq, xc, xs, n, ldx, d, static_cast<T*>(out), ldo);
}

// ----------------------------------------------------------- tensor cores --

struct DotArgs {
    const float *qs, *xs;
    int64_t nq, n, ldo;
    int nqt, nxt;  // tiles of 256 queries, of 256 rows
    int nk;
    void* out;
    int x_rows, q_rows;  // box rows
};

// COLS >= nq, or 256
template <typename T, int COLS>
struct DotPolicy {
    static constexpr bool kInt8 = true;
    static constexpr int kAccCols = COLS;
    static constexpr int kStages = 6, kStgBytes = 256;
    // rows are walked in groups of 8 tiles: the tiles in flight form a block of
    // both operands that L2 holds
    static constexpr int kGroup = 8;
    const CUtensorMap *mx, *mq;
    const DotArgs& a;

    using Job = TileJob;
    struct Iter {
        const DotPolicy& p;
        int64_t i;
        int step;
        __device__ Iter(const DotPolicy& pol, int pair, int npairs) : p(pol), i(pair), step(npairs) {}
        __device__ __forceinline__ bool next(Job& j) {
            const DotArgs& a = p.a;
            if (i >= static_cast<int64_t>(a.nqt) * a.nxt) return false;
            const int64_t per = static_cast<int64_t>(kGroup) * a.nqt;
            const int g = static_cast<int>(i / per), in = static_cast<int>(i % per);
            const int gs = min(kGroup, a.nxt - g * kGroup);
            j.ma = p.mx;
            j.mb = p.mq;
            j.m0 = (g * kGroup + in % gs) * TT_M;
            j.n0 = in / gs * TT_N;
            j.nn = static_cast<int>(min(static_cast<int64_t>(TT_N), (a.nq - j.n0 + 31) / 32 * 32));
            j.k0 = 0;
            j.nk = a.nk;
            j.nseg = 1;
            j.a_mn = j.b_mn = false;
            j.a_rows = a.x_rows;
            j.b_rows = a.q_rows;
            j.a_second = j.m0 + 128 < a.n;
            i += step;
            return true;
        }
    };
    struct Epi {
        float xs;
    };

    __device__ __forceinline__ void begin(Epi& e, const Job& j, const TileCtx& c) const {
        if (COLS < TT_N && c.col0 >= j.nn) return;
        const int64_t r = static_cast<int64_t>(j.m0) + c.row;
        e.xs = r < a.n ? a.xs[r] : 0.f;
        // the query scales of the warp's columns
        float* qs = reinterpret_cast<float*>(c.stg);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t b = static_cast<int64_t>(j.n0) + (h ? c.col1 : c.col0) + c.lane;
            qs[h * 32 + c.lane] = b < a.nq ? a.qs[b] : 0.f;
        }
        __syncwarp();
    }

    __device__ __forceinline__ void chunk(Epi& e, const Job& j, const TileCtx& c, int col,
                                          const uint32_t (&r)[32]) const {
        const int64_t x = static_cast<int64_t>(j.m0) + c.row, b0 = static_cast<int64_t>(j.n0) + col;
        if (x >= a.n || b0 >= a.nq) return;
        const float4* qs = reinterpret_cast<const float4*>(c.stg) + (col == c.col0 ? 0 : 8);
        char* o = reinterpret_cast<char*>(static_cast<T*>(a.out) + b0 * a.ldo + x);
        const int64_t step = a.ldo * static_cast<int64_t>(sizeof(T));
        const int valid = static_cast<int>(min(static_cast<int64_t>(32), a.nq - b0));
        const uint64_t xs2 = pack2(e.xs, e.xs);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            const float4 q = qs[i / 4];
            float v[4];
            unpack2(mul_f32x2(mul_f32x2(pack2(q.x, q.y), xs2),
                              pack2(static_cast<float>(static_cast<int>(r[i])), static_cast<float>(static_cast<int>(r[i + 1])))),
                    v[0], v[1]);
            unpack2(mul_f32x2(mul_f32x2(pack2(q.z, q.w), xs2), pack2(static_cast<float>(static_cast<int>(r[i + 2])),
                                                                     static_cast<float>(static_cast<int>(r[i + 3])))),
                    v[2], v[3]);
            if (valid == 32) {
#pragma unroll
                for (int k = 0; k < 4; ++k, o += step) *reinterpret_cast<T*>(o) = from_f<T>(v[k]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k, o += step)
                    if (i + k < valid) *reinterpret_cast<T*>(o) = from_f<T>(v[k]);
            }
        }
    }

    __device__ __forceinline__ void end(Epi&, const Job&, const TileCtx&) const {}
    __device__ __forceinline__ void finish(const TileCtx&) const {}
};

template <typename T, int COLS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TT_THREADS, 1)
    sq8_tile_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mq,
                    const __grid_constant__ DotArgs a, const TileStatus st) {
    extern __shared__ uint8_t smem_raw[];
    const DotPolicy<T, COLS> p{&mx, &mq, a};
    tile_loop(smem_raw, p, false, st);
}

template <typename T, int COLS>
int launch_tile(const int8_t* qc, const float* qs, int64_t nq, int64_t ldq, const int8_t* xc, const float* xs,
                int64_t n, int64_t ldx, int d, void* out, int64_t ldo, cudaStream_t s) {
    static bool attr[64] = {false};
    RDB_TRY(tile_smem_attr(sq8_tile_kernel<T, COLS>, attr));
    DotArgs a{qs, xs, nq, n, ldo, (int)((nq + TT_N - 1) / TT_N), (int)((n + TT_M - 1) / TT_M), (d + 127) / 128, out,
              tile_box_rows(n, 128), tile_box_rows((nq + 31) / 32 * 16, 128)};
    CUtensorMap mx, mq;
    RDB_TRY(make_map_3d(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, xc, d, n, 1, ldx, 0, a.x_rows));
    RDB_TRY(make_map_3d(&mq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, qc, d, nq, 1, ldq, 0, a.q_rows));
    const int64_t tiles = (int64_t)a.nqt * a.nxt;
    return launch_chained(sq8_tile_kernel<T, COLS>, 2 * (unsigned)std::min<int64_t>(tile_pairs(), tiles), TT_THREADS, TT_SMEM, s,
                          mx, mq, a, tile_status());
}

template <typename T>
int launch_dot(const int8_t* qc, const float* qs, int64_t nq, int64_t ldq, const int8_t* xc, const float* xs,
               int64_t n, int64_t ldx, int d, void* out, int64_t ldo, cudaStream_t s) {
    // One or two queries, calls in a row: 1M x 768 in 117 / 118 us against 130 of the
    // tile loop, 1M x 1,024 154 against 163, 4M x 128 102 / 103 against 197, and from
    // L2 100,000 x 768 9.1 / 12.0 against 18.0 and 1,000 x 768 4.4 against 7.2 (100,000
    // x 768 with 256 MB written between the calls: 24.6 for both, against 26.7).  From
    // four on dp4a costs more than the codes' bytes: 150 us for 1M x 768 (4M x 128:
    // 385), the tile loop 134 (198).
    const int64_t dp = (d + 15) / 16 * 16;
    if (nq == 1 && dp <= GV_SMEM) return launch_few<T, 1>(qc, qs, nq, ldq, xc, xs, n, ldx, d, out, ldo, s);
    if (nq == 2 && 2 * dp <= GV_SMEM) return launch_few<T, 2>(qc, qs, nq, ldq, xc, xs, n, ldx, d, out, ldo, s);
    // (128 columns: four accumulators measure the same as two of 256)
    if (nq <= 64) return launch_tile<T, 64>(qc, qs, nq, ldq, xc, xs, n, ldx, d, out, ldo, s);
    return launch_tile<T, TT_N>(qc, qs, nq, ldq, xc, xs, n, ldx, d, out, ldo, s);
}

}  // namespace
}  // namespace rdb

using namespace rdb;

extern "C" {

int rdb_sq8_dot(const int8_t* qc, const float* qs, int64_t nq, int64_t ldq, const int8_t* xc, const float* xs,
                int64_t n, int64_t ldx, int d, int out_dtype, void* out, int64_t ldo, void* stream) {
    RDB_CHECK_ARG(elem_size(out_dtype) != 0, "unknown dtype %d", out_dtype);
    RDB_CHECK_ARG(nq >= 0 && n >= 0 && d >= 1 && ldq >= d && ldx >= d && ldo >= n, "bad shape");
    RDB_CHECK_ARG(d <= kMaxDim, "d must be <= %d (the integer sum has 32 bits)", kMaxDim);
    RDB_CHECK_ARG(nq < (1LL << 31) && n < (1LL << 31), "nq and n must be < 2^31");
    if (nq == 0 || n == 0) return RDB_OK;
    RDB_CHECK_ARG(qc && qs && xc && xs && out, "NULL pointer");
    RDB_CHECK_ARG(ldq % 16 == 0 && ldx % 16 == 0, "row strides must be multiples of 16 bytes");
    RDB_CHECK_ARG((reinterpret_cast<uintptr_t>(qc) & 15) == 0 && (reinterpret_cast<uintptr_t>(xc) & 15) == 0,
                  "codes must be 16-byte aligned");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (out_dtype == RDB_F32) return launch_dot<float>(qc, qs, nq, ldq, xc, xs, n, ldx, d, out, ldo, s);
    if (out_dtype == RDB_F16) return launch_dot<__half>(qc, qs, nq, ldq, xc, xs, n, ldx, d, out, ldo, s);
    return launch_dot<__nv_bfloat16>(qc, qs, nq, ldq, xc, xs, n, ldx, d, out, ldo, s);
}

}  // extern "C"
