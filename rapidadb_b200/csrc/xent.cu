// Softmax cross entropy of queries against every stored row, with gradients.
//
//   s_bn   = scale <q_b, x_n>                  (the [nq, n] matrix is never kept)
//   loss_b = log sum_n exp(s_bn) - s_b,t(b)    (0 where t(b) == ignore_index)
//   G_bn   = w_b scale (p_bn - [n = t(b)]),    p_bn = exp(s_bn) / sum_n exp(s_bn)
//   dq = G x,  dx = G^T q
//
// The products run on the tcgen05 tile loops of tile_tc.cuh and tile_f32.cuh; only
// the logits of one query (fp32: up to four) come from rows streamed past CUDA
// cores, in the forward and in the backward pass: G then divides terms by a sum of
// the very same ones.
//
// Forward: one pass over the rows.  The sum is taken in base 2 around a running
// maximum in the epilogue of each tile, c = scale log2 e,
//   m = max_n c <q, x_n>,   z = sum_n 2^(c <q, x_n> - m),
// held in fp32, one (m, z) per query, row split and epilogue group, joined by
// xent_join_kernel.  The target's own term stays out of the running sum: with
// r = the sum of the other terms relative to the target's, loss = log1p(r), so
// a query that finds its row keeps a loss near 0, and its 1 - p = -expm1(-loss),
// to full precision.
//
// Backward: the rows in pieces.  Per piece one launch recomputes the logits and
// writes a [nq, rows] workspace of G in the operands' type, every row of it over
// its 1 - p_t, one launch multiplies it both ways: dx rows directly (K = nq), dq
// into fp32 partial sums (K = rows, split over several tiles when there are few
// queries), joined at the end.  No atomics on values: every sum has a fixed order.
//
// Bound: the products, 2 nq n d FLOP each, one forward and three backward.  4,096
// queries, 131,072 rows, d = 768, bf16: forward 578 us (1.43 PFLOP/s, the rate
// cuBLAS holds for seconds is 1.40), probabilities 620, gradients 1,240.  Few
// queries: the rows' bytes, 1 x 1M x 768 bf16 225 us (6.8 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "tile_f32.cuh"
#include "tile_tc.cuh"

namespace rdb {
namespace {

constexpr int NT = 256;
constexpr float kLn2 = 0.6931471805599453f;
constexpr double kLog2e = 1.4426950408889634;
// G is held per query as 2^14 (p - [n = t]) / (1 - p_t): the target's entry, by
// far the largest of most rows, is -2^14 exactly, the others add up to 2^14, so
// that rounding G to 16 bits costs dq little (rounding p_t - 1 itself doubled its
// error) and fp16 keeps 11 bits of every entry down to 2^-28 of its row's sum.
// What it leaves, w (1 - p_t), multiplies dq exactly and enters dx with the
// query, rounded once there.
constexpr float kGScale = 16384.f, kGLog2 = 14.f;

inline int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// (M, Z) of two sets of terms: the larger maximum, and the sums relative to it.
// A set without finite terms has M = -inf and Z = 0 (or NaN).
__device__ __forceinline__ void join(float& M, float& Z, float m, float z, float c) {
    const float nm = fmaxf(M, m);
    Z = Z * (M > -INFINITY ? ex2((M - nm) * c) : 1.f) + z * (m > -INFINITY ? ex2((m - nm) * c) : 1.f);
    M = nm;
}

// two floats in the 16-bit type, a in the low half
template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// ---------------------------------------------------------------- forward --

struct FwdArgs {
    int64_t nq, n;       // queries, rows of this piece
    int64_t row0;        // first row of the piece in the base
    int nqb, nsplit, slot0;
    int q_rows, width;   // box rows of the queries, columns of a tile
    int n32;             // 32-row groups of the piece, dealt evenly to the splits
    int nkb, nseg;
    float c;
    const int64_t* targets;
    int groups, parts;   // epilogue groups, parts per query: slots * groups
    float2* part;        // [nq][parts] (max <q, x>, z) of each split and epilogue group
    unsigned* ticket;    // of the join, cleared here
};

struct FwdPolicy {
    static constexpr bool kInt8 = false;
    static constexpr int kAccCols = TT_N;
    static constexpr int kStages = 7, kStgBytes = 0;
    [[maybe_unused]] static constexpr bool kBMn = false;  // (tile_f32.cuh)
    const CUtensorMap *mq, *mx;
    const FwdArgs& a;

    struct Job : TileJob {
        int split;
        bool first, last;
    };
    // units of (query block, row split), query blocks first, so that the pairs
    // in flight read the same rows
    struct Iter {
        const FwdPolicy& p;
        int unit, step, lo, at, hi;  // 32-row groups
        __device__ Iter(const FwdPolicy& pol, int pair, int npairs) : p(pol), unit(pair - npairs), step(npairs), lo(0), at(0), hi(0) {}
        __device__ __forceinline__ bool next(Job& j) {
            if (at >= hi) {
                unit += step;
                if (unit >= p.a.nqb * p.a.nsplit) return false;
                const int64_t sp = unit / p.a.nqb;
                lo = at = static_cast<int>(sp * p.a.n32 / p.a.nsplit);
                hi = static_cast<int>((sp + 1) * p.a.n32 / p.a.nsplit);
            }
            j.ma = p.mq;
            j.mb = p.mx;
            j.m0 = unit % p.a.nqb * TT_M;
            j.n0 = at * 32;
            j.nn = min(p.a.width, (hi - at) * 32);
            j.k0 = 0;
            j.nk = p.a.nkb;
            j.nseg = p.a.nseg;
            j.a_mn = j.b_mn = false;
            j.a_rows = p.a.q_rows;
            j.b_rows = p.a.width / 2;
            j.a_second = j.m0 + 128 < p.a.nq;
            j.split = unit / p.a.nqb;
            j.first = at == lo;
            at += p.a.width / 32;
            j.last = at >= hi;
            return true;
        }
    };
    struct Epi {
        float m, mb, z;  // running maximum of <q, x>, c times it, sum
        int64_t tgt;     // target as a row of the piece (any value: not there)
    };

    __device__ __forceinline__ void begin(Epi& e, const Job& j, const TileCtx& c) const {
        if (!j.first) return;
        e.m = -INFINITY;
        e.mb = e.z = 0.f;
        const int64_t b = j.m0 + c.row;
        e.tgt = b < a.nq ? a.targets[b] - a.row0 : -1;
    }

    // 32 columns from column col on: columns behind the last row count as -inf,
    // and so does the target's, whose term is kept apart
    __device__ __forceinline__ void mask(const Epi& e, const Job& j, int col, float (&v)[32]) const {
        const int64_t c0 = static_cast<int64_t>(j.n0) + col;
        if (c0 + 32 > a.n) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (c0 + i >= a.n) v[i] = -INFINITY;
        }
        const int64_t rel = e.tgt - c0;
        if (rel >= 0 && rel < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                v[i] = i == static_cast<int>(rel) ? -INFINITY : v[i];
        }
    }
    static __device__ __forceinline__ float largest(const float (&v)[32]) {
        float m0 = max3(v[0], v[1], v[2]), m1 = max3(v[3], v[4], v[5]);
#pragma unroll
        for (int i = 6; i < 30; i += 4) {
            m0 = max3(m0, v[i], v[i + 1]);
            m1 = max3(m1, v[i + 2], v[i + 3]);
        }
        return fmaxf(max3(m0, v[30], v[31]), m1);
    }
    // sums of 2^(c v - c m), two columns per instruction
    static __device__ __forceinline__ void add_terms(const float (&v)[32], uint64_t c2, uint64_t b2, uint64_t& s0,
                                                     uint64_t& s1) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            float x0, x1, x2, x3;
            unpack2(fma_f32x2(pack2(v[i], v[i + 1]), c2, b2), x0, x1);
            unpack2(fma_f32x2(pack2(v[i + 2], v[i + 3]), c2, b2), x2, x3);
            s0 = add_f32x2(s0, pack2(ex2(x0), ex2(x1)));
            s1 = add_f32x2(s1, pack2(ex2(x2), ex2(x3)));
        }
    }

    __device__ __forceinline__ void chunk(Epi& e, const Job& j, const TileCtx& c, int col,
                                          const uint32_t (&r)[32]) const {
        if (j.m0 + c.row - c.lane >= a.nq) return;  // no query in this warp's 32 rows
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        mask(e, j, col, v);
        const float mx = largest(v);
        if (mx > e.m) {
            e.z *= ex2((e.m - mx) * a.c);  // 0 before the first finite value
            e.m = mx;
            e.mb = mx * a.c;
        }
        const uint64_t c2 = pack2(a.c, a.c), b2 = pack2(-e.mb, -e.mb);
        uint64_t s0 = 0, s1 = 0;
        add_terms(v, c2, b2, s0, s1);
        float p0, p1;
        unpack2(add_f32x2(s0, s1), p0, p1);
        e.z += p0 + p1;
    }

    __device__ __forceinline__ void end(Epi& e, const Job& j, const TileCtx& c) const {
        const int64_t b = j.m0 + c.row;
        if (j.last && b < a.nq)
            a.part[b * a.parts + (a.slot0 + j.split) * a.groups + c.grp] = make_float2(e.m, e.z);
    }
    __device__ __forceinline__ void finish(const TileCtx&) const {}
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TT_THREADS, 1)
    xent_scan_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mx,
                     const __grid_constant__ FwdArgs a, const bool bf16, const TileStatus st) {
    extern __shared__ uint8_t smem_raw[];
    const FwdPolicy p{&mq, &mx, a};
    tile_loop(smem_raw, p, bf16, st);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0u;
}

// the same for at most 128 queries and fp32 rows as they are
__global__ void __launch_bounds__(TF_THREADS, 1)
    xent_scan_f32_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ F32Rows x,
                         const __grid_constant__ FwdArgs a, const TileStatus st) {
    extern __shared__ uint8_t smem_raw[];
    const FwdPolicy p{&mq, nullptr, a};
    tile_loop_f32(smem_raw, p, x, st);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0u;
}

// What turns a query's logits into its row of G, 2^14 (p - [n = t]) / (1 - p_t): the
// terms 2^(c <q, x> - m - lz), -2^14 at the target, or nothing.  Two roundings, of
// the exponent relative to the largest logit and of the one relative to their sum:
// both small for the terms that count.
struct GTerm {
    float m, lz;
    int64_t tgt;  // target as a row of the piece (any value: not there)
    bool zero;    // an ignored query, one whose target is certain, or none
    __device__ __forceinline__ GTerm() : m(0.f), lz(0.f), tgt(-1), zero(true) {}
    __device__ __forceinline__ GTerm(const float* stats, const int64_t* targets, int64_t b, int64_t nq, int64_t ignore,
                                     int64_t row0) {
        const int64_t t = targets[b];
        const float rest = -expm1f(-stats[2 * nq + b]);  // 1 - p_t
        zero = t == ignore || rest == 0.f;
        tgt = zero ? -1 : t - row0;
        m = stats[b];
        lz = stats[nq + b] + log2f(rest) - kGLog2;
    }
};

// ---- the same for a few queries, without tensor cores

constexpr int ST_MAX_DIM = 1024;  // 32 elements of every query a lane

// one 16-byte unit of a row as pairs of floats
template <typename T>
__device__ __forceinline__ void pairs16(const uint4& u, uint64_t (&v)[8 / sizeof(T)]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 4) {
        v[0] = pack2(__uint_as_float(w[0]), __uint_as_float(w[1]));
        v[1] = pack2(__uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T* e = reinterpret_cast<const T*>(&w[i]);
            v[i] = pack2(to_f(e[0]), to_f(e[1]));
        }
    }
}

// rows a warp has in flight: about 12 loads a lane
constexpr int stream_rows(int units) { return units == 1 ? 8 : units <= 3 ? 4 : 2; }

// A lane holds every 32nd 16-byte unit of the queries in registers, U of them, as
// fp32; the warps take R rows each in turn (shares of their own, rows far apart,
// are up to 20 % slower).  The products are fp32 fma chains; the lanes' sums of
// R x NQ products are joined so that each lane ends up with one of them, whose
// (m, z) it keeps.  One part per query and block.  (Queries in shared memory cost
// a load per use: 50 us instead of 32 for 100,000 x 768 bf16.)
// PROB: the backward pass, which writes G of a piece of the rows instead.  (From
// the tile loop's logits, whose sums are cut where these are rounded, fp32
// gradients were off by up to 4e-5; and 1M x 768 in fp32 takes 0.5 ms here, 1.2
// there.)
struct StreamOut {
    float2* part;      // forward
    unsigned* ticket;
    void* g;           // PROB: G of the piece in T, fp32 as three bf16 planes
    int64_t ldg, plane, row0;
    const float* stats;
    int64_t ignore;
};

template <typename T, int NQ, int U, bool PROB>
__global__ void __launch_bounds__(NT, NQ == 1 ? 2 : 1)
    xent_stream_kernel(const T* q, int nq, int64_t ldq, const T* x, int64_t n, int64_t ldx, int d, const int64_t* targets,
                       float c, const __grid_constant__ StreamOut out) {
    constexpr int E = 16 / sizeof(T), P = E / 2;  // elements and pairs of a unit
    constexpr int R = stream_rows(U), V = R * NQ, kDup = 32 / V;
    __shared__ float2 sj[NT / 32][NQ];
    chain_wait();
    if (!PROB && blockIdx.x == 0 && threadIdx.x == 0) *out.ticket = 0u;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int full = d / E, units = (d + E - 1) / E;
    // A row's last unit may reach behind d, but not behind the row's stride, which
    // is whole units: it is read whole and cut when it is used.  Only the last row
    // may end with its elements.
    auto load = [&](const T* row, bool last, int u) -> uint4 {
        if (u < (last ? full : units)) return reinterpret_cast<const uint4*>(row)[u];
        union {
            uint4 v;
            T e[E];
        } o;
        o.v = make_uint4(0u, 0u, 0u, 0u);
        if (last) {
#pragma unroll
            for (int t = 0; t < E; ++t)
                if (u * E + t < d) o.e[t] = row[u * E + t];
        }
        return o.v;
    };
    auto cut = [&](uint4& v, int u) {
        if (d % E == 0 || u != full) return;
        uint32_t* o = reinterpret_cast<uint32_t*>(&v);
        const int bytes = (d - full * E) * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int left = bytes - 4 * i;
            o[i] = left >= 4 ? o[i] : left > 0 ? o[i] & 0xffffu : 0u;
        }
    };
    uint64_t qv[NQ][U * P];
#pragma unroll
    for (int b = 0; b < NQ; ++b)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            uint64_t v[P];
            pairs16<T>(b < nq ? load(q + b * ldq, true, u * 32 + lane) : make_uint4(0u, 0u, 0u, 0u), v);
#pragma unroll
            for (int i = 0; i < P; ++i) qv[b][u * P + i] = v[i];
        }
    const int row = lane / kDup / NQ, bq = lane / kDup % NQ;  // of the sum this lane ends up with
    const GTerm term = PROB && bq < nq ? GTerm(out.stats, targets, bq, nq, out.ignore, out.row0) : GTerm();
    const int64_t tgt = PROB || bq >= nq ? -1 : targets[bq];
    const int64_t w = static_cast<int64_t>(blockIdx.x) * (NT / 32) + warp;
    const int64_t nw = static_cast<int64_t>(gridDim.x) * (NT / 32);
    int64_t r0 = w * R;
    float m = -INFINITY, mb = 0.f, z = 0.f;
    uint4 v[R][U];
    if (r0 < n) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t i = min(r0 + r, n - 1);
                v[r][u] = load(x + i * ldx, i == n - 1, u * 32 + lane);
            }
    }
    for (; r0 < n; r0 += R * nw) {
        float s[V];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            uint64_t acc[NQ][2];
#pragma unroll
            for (int b = 0; b < NQ; ++b) acc[b][0] = acc[b][1] = 0;
            // its successor replaces a unit as soon as it is used
            const int64_t next = min(r0 + R * nw + r, n - 1);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint64_t xv[P];
                cut(v[r][u], u * 32 + lane);
                pairs16<T>(v[r][u], xv);
                v[r][u] = load(x + next * ldx, next == n - 1, u * 32 + lane);
#pragma unroll
                for (int b = 0; b < NQ; ++b)
#pragma unroll
                    for (int i = 0; i < P; ++i) acc[b][i & 1] = fma_f32x2(xv[i], qv[b][u * P + i], acc[b][i & 1]);
            }
#pragma unroll
            for (int b = 0; b < NQ; ++b) {
                float a0, a1;
                unpack2(add_f32x2(acc[b][0], acc[b][1]), a0, a1);
                s[r * NQ + b] = a0 + a1;
            }
        }
        // each half of the lanes goes on with half of the sums
#pragma unroll
        for (int o = 16, k = V; o > 0; o >>= 1) {
            if (k > 1) {
                k /= 2;
#pragma unroll
                for (int i = 0; i < V / 2; ++i)
                    if (i < k) {
                        const float keep = lane & o ? s[i + k] : s[i], give = lane & o ? s[i] : s[i + k];
                        s[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                    }
            } else {
                s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
            }
        }
        const int64_t r = r0 + row;
        if constexpr (PROB) {
            if (r < n && bq < nq && lane % kDup == 0) {
                float v = term.zero ? 0.f : r == term.tgt ? -kGScale : ex2(fmaf(s[0], c, -term.m) - term.lz);
                const int64_t at = bq * out.ldg + r;
                if constexpr (sizeof(T) == 2) {
                    static_cast<T*>(out.g)[at] = from_f<T>(v);
                } else {
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        const __nv_bfloat16 h = __float2bfloat16_rn(v);
                        static_cast<__nv_bfloat16*>(out.g)[k * out.plane + at] = h;
                        v -= __bfloat162float(h);  // exact
                    }
                }
            }
        } else if (r < n && r != tgt) {
            if (s[0] > m) {
                z *= ex2((m - s[0]) * c);
                m = s[0];
                mb = m * c;
            }
            z += ex2(fmaf(s[0], c, -mb));
        }
    }
    if constexpr (!PROB) {
        // the warp's R sets of a query, in the first lanes' order, then the block's
#pragma unroll
        for (int o = 16; o >= kDup * NQ; o >>= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, m, o), oz = __shfl_xor_sync(0xffffffffu, z, o);
            join(m, z, om, oz, c);
        }
        if (row == 0 && lane % kDup == 0) sj[warp][bq] = make_float2(m, z);
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < nq) {
            float2 a = sj[0][threadIdx.x];
            for (int k = 1; k < NT / 32; ++k) join(a.x, a.y, sj[k][threadIdx.x].x, sj[k][threadIdx.x].y, c);
            out.part[threadIdx.x * gridDim.x + blockIdx.x] = a;
        }
    }
}

// mean or sum of the losses of the queries that count, and their number, by one
// block in index order; in 64 bits, since a thread's part of many queries is one
// long chain (in fp32 the sum of 2^20 losses was off by 4e-5)
__device__ void reduce_losses(float* stats, const int64_t* targets, int64_t ignore, int64_t nq, int reduction,
                              float* total, double* ss, int* sc) {
    double s = 0.;
    int cnt = 0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < nq; i += NT) {
        const float l = __ldcg(stats + 2 * nq + i);
        const bool counts = targets[i] != ignore;
        s += counts ? static_cast<double>(l) : 0.;
        cnt += counts;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    if ((threadIdx.x & 31) == 0) ss[threadIdx.x >> 5] = s, sc[threadIdx.x >> 5] = cnt;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < NT / 32; ++w) ss[0] += ss[w], sc[0] += sc[w];
        *total = static_cast<float>(reduction == RDB_REDUCE_MEAN ? ss[0] / sc[0] : ss[0]);
        stats[3 * nq] = static_cast<float>(sc[0]);
    }
}

// 8 elements of a row from column t on as floats; what lies behind d is neither
// read nor kept
template <typename T>
__device__ __forceinline__ void load8(const T* row, int t, int d, float (&v)[8]) {
    if (t + 8 <= d) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(row + t), b = *reinterpret_cast<const float4*>(row + t + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(row + t);
            const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f(e[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = t + i < d ? to_f(row[t + i]) : 0.f;
    }
}

// <q, x> of two rows by one warp: 8 fp32 fma chains a lane, joined
template <typename T>
__device__ __forceinline__ float warp_dot(const T* q, const T* x, int d, int lane) {
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int t = lane * 8; t < d; t += 256) {
        float a[8], b[8];
        load8(q, t, d, a);
        load8(x, t, d, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = fmaf(a[i], b[i], s[i]);
    }
    float v = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Joins the parts of each query, by one warp, or by a whole block where there are
// no more queries than SMs (wide); stats and loss of each.
// The target's logit is computed here, in rounded fp32: the tensor cores cut
// their sums towards zero, which shifts the largest logits of a query alike, and
// only the target's shift would remain in the loss (7e-6 of it at d = 768).
// An ignored query has loss 0; one whose target is no row is NaN throughout.
// For a reduced loss the last block to finish sums the losses (in index order,
// whoever it is) and leaves the number of queries that count behind the stats;
// `ticket` was cleared by the scan.
template <typename T>
__global__ void __launch_bounds__(NT)
    xent_join_kernel(const float2* part, int parts, const T* q, int64_t ldq, const T* x, int64_t ldx, int d,
                     const int64_t* targets, int64_t ignore, int64_t n, float c, int64_t nq, bool wide, float* stats,
                     float* loss, int reduction, float* total, unsigned* ticket) {
    chain_wait();
    __shared__ float2 sj[NT / 32];
    __shared__ double ss[NT / 32];
    __shared__ int sc[NT / 32];
    __shared__ bool last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = wide ? 1 : NT / 32;  // queries per block and step
    for (int64_t b0 = static_cast<int64_t>(blockIdx.x) * per; b0 < nq; b0 += static_cast<int64_t>(gridDim.x) * per) {
        const int64_t b = wide ? b0 : b0 + warp;
        const bool mine = b < nq && (!wide || warp == 0);  // the warp that finishes the query
        const int64_t t = b < nq ? targets[b] : -1;
        const bool ignored = t == ignore, has = t >= 0 && t < n;
        const float td = mine && has ? warp_dot(q + b * ldq, x + t * ldx, d, lane) : -INFINITY;
        float M = -INFINITY, Z = 0.f;
        if (b < nq)
#pragma unroll 4
            for (int s = wide ? threadIdx.x : lane; s < parts; s += wide ? NT : 32) {
                const float2 v = part[b * parts + s];
                join(M, Z, v.x, v.y, c);
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float m = __shfl_xor_sync(0xffffffffu, M, o), z = __shfl_xor_sync(0xffffffffu, Z, o);
            // the same operands in the same order on both sides
            float lo_m = lane & o ? m : M, lo_z = lane & o ? z : Z;
            join(lo_m, lo_z, lane & o ? M : m, lane & o ? Z : z, c);
            M = lo_m, Z = lo_z;
        }
        if (wide) {
            if (lane == 0) sj[warp] = make_float2(M, Z);
            __syncthreads();
            for (int k = 1; k < NT / 32; ++k)
                if (warp == 0) join(M, Z, sj[k].x, sj[k].y, c);
            __syncthreads();
        }
        if (lane == 0 && mine) {
            const float nan = __int_as_float(0x7fc00000);
            // Z sums 2^(c v - c M); u: the target's exponent relative to that
            const float Mc = M > -INFINITY ? M * c : 0.f;
            const float u = fmaf(td, c, -Mc);
            float m = Mc, lz, l;
            if (u >= 0.f || (has && !(M > -INFINITY))) {
                // the target is the largest (or the only) term
                m = td * c;
                const float rest = M > -INFINITY ? Z * ex2(-u) : 0.f * Z;
                l = isfinite(td) ? log1pf(rest) : nan;
                lz = log2f(rest + ex2(fmaf(td, c, -m)));
            } else {
                lz = log2f(Z + (has ? ex2(u) : 0.f));
                l = kLn2 * (lz - u);
            }
            if (ignored) l = 0.f;
            else if (!has) l = lz = nan;
            stats[b] = m;
            stats[nq + b] = lz;
            stats[2 * nq + b] = l;
            if (reduction == RDB_REDUCE_NONE) loss[b] = l;
        }
    }
    if (reduction == RDB_REDUCE_NONE) {
        if (blockIdx.x == 0 && threadIdx.x == 0) stats[3 * nq] = 0.f;
        return;
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(ticket, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    reduce_losses(stats, targets, ignore, nq, reduction, total, ss, sc);
}

// the reduced loss of no queries
__global__ void __launch_bounds__(NT)
    xent_reduce_kernel(const int64_t* targets, int64_t ignore, int64_t nq, int reduction, float* stats, float* total) {
    chain_wait();
    __shared__ double ss[NT / 32];
    __shared__ int sc[NT / 32];
    reduce_losses(stats, targets, ignore, nq, reduction, total, ss, sc);
}

// --------------------------------------------------------------- backward --

// u_b = w_b (1 - p_t) of a query, w_b the weight of its loss: g[b], or for a
// reduced loss g[0], over the number of queries for the mean (0 when none count).
struct Weights {
    const float* g;
    const float* count;   // nullptr: not a mean
    const float* loss;    // [nq]
    const int64_t* targets;
    int64_t ignore;
    bool equal;
    __device__ __forceinline__ float u(int64_t b) const {
        if (targets[b] == ignore) return 0.f;
        float w = g[equal ? 0 : b];
        if (count) w = *count > 0.f ? w / *count : 0.f;
        return w * -expm1f(-loss[b]);
    }
};

// Largest |u_b| (x) over the queries of one block out of `blocks`, and for fp16 the
// largest |u_b| max_t |q_bt| (y).  Every thread gets them; a NaN makes its own
// products NaN.
template <typename T>
__device__ float2 largest_weight(const Weights& w, const T* q, int64_t nq, int64_t ldq, int d, int block, int blocks,
                                 float2* sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float mx = 0.f, my = 0.f;
    if constexpr (std::is_same<T, __half>::value) {
        for (int64_t b = block * (NT / 32) + warp; b < nq; b += blocks * (NT / 32)) {
            const float u = fabsf(w.u(b));
            if (!(u > 0.f)) continue;  // an ignored query may hold anything
            float a = 0.f;
#pragma unroll 4
            for (int t = lane * 8; t < d; t += 256) {
                float v[8];
                load8(q + b * ldq, t, d, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) a = fmaxf(a, fabsf(v[k]));
            }
            mx = fmaxf(mx, u);
            my = fmaxf(my, u * a);
        }
        my = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(my)));
    } else {
#pragma unroll 4
        for (int64_t i = static_cast<int64_t>(block) * NT + threadIdx.x; i < nq; i += static_cast<int64_t>(blocks) * NT)
            mx = fmaxf(mx, fabsf(w.u(i)));
    }
    mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
    if (lane == 0) sm[warp] = make_float2(mx, my);
    __syncthreads();
    float2 m = sm[0];
#pragma unroll
    for (int k = 1; k < NT / 32; ++k) m = make_float2(fmaxf(m.x, sm[k].x), fmaxf(m.y, sm[k].y));
    return m;
}

constexpr int kWeightBlocks = 128;

template <typename T>
__global__ void __launch_bounds__(NT)
    xent_wmax_kernel(const T* q, int64_t nq, int64_t ldq, int d, const Weights w, float2* parts) {
    chain_wait();
    __shared__ float2 sm[NT / 32];
    const float2 m = largest_weight(w, q, nq, ldq, d, blockIdx.x, gridDim.x, sm);
    if (threadIdx.x == 0) parts[blockIdx.x] = m;
}

// What the weighted queries are multiplied by besides 1 / max |u|.  bf16 (and the
// planes of fp32) has fp32's exponents: 1.  fp16: the power of two that brings the
// largest element between 2^14 and 2^15, so that elements keep their 11 bits down
// to 2^-28 of it, as far as dx itself does.  (At 1 the largest of a unit query of
// 768 elements is about 0.1, and a query of 1 / 500 of the largest weight is
// subnormal: rows of dx that only such queries move lost up to all their digits.)
template <typename T>
__device__ __forceinline__ float weight_top(const float2& m) {
    if constexpr (!std::is_same<T, __half>::value) return 1.f;
    const float r = 32768.f * (m.x / m.y);
    if (!(m.y > 0.f) || isnan(r)) return 1.f;  // nothing to weigh, or an infinite weight
    // an element is at most 65,504: below 1/2 the product m.y has overflown
    return __uint_as_float(__float_as_uint(fminf(fmaxf(r, 0.5f), 0x1p100f)) & 0x7f800000u);
}

// the three bf16 planes of 8 floats, plane stride in elements
__device__ __forceinline__ void store_planes(const float (&v)[8], __nv_bfloat16* o, int64_t plane) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        uint32_t w[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            w[h] = pack16<__nv_bfloat16>(r[2 * h], r[2 * h + 1]);
            // what is left for the next plane: exact in fp32
            r[2 * h] -= __uint_as_float(w[h] << 16);
            r[2 * h + 1] -= __uint_as_float(w[h] & 0xffff0000u);
        }
        *reinterpret_cast<uint4*>(o + k * plane) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Queries as an operand of dx = G^T (u q): out[b] = q[b] u_b / wmax, wmax = max |u|
// over the above, so that the type's range is used whatever the size of the
// gradients; zero rows for ignored queries, whatever they hold.  fp32: three bf16
// planes.  nparts: sets of largest weights; 0: every block finds them itself (few
// queries).  The first block leaves wmax behind.
template <typename T>
__global__ void __launch_bounds__(NT)
    xent_weighted_kernel(const T* q, int64_t nq, int64_t ldq, int d, const Weights w, const float2* parts, int nparts,
                         float* wmax, void* out, int64_t ldo) {
    chain_wait();
    __shared__ float2 sm[NT / 32];
    float2 m = make_float2(0.f, 0.f);
    if (!std::is_same<T, __half>::value && nparts == 0) {
        m = largest_weight(w, q, nq, ldq, d, 0, 1, sm);
    } else {
#pragma unroll
        for (int k = 0; k < kWeightBlocks / 32; ++k) {
            const int i = k * 32 + (threadIdx.x & 31);
            const float2 v = i < nparts ? parts[i] : make_float2(0.f, 0.f);
            m = make_float2(fmaxf(m.x, v.x), fmaxf(m.y, v.y));
        }
        m.x = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m.x)));
        m.y = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m.y)));
    }
    const float mx = m.x, top = weight_top<T>(m);
    if (blockIdx.x == 0 && threadIdx.x == 0) *wmax = mx / top;
    const int64_t units = ldo / 8, total = nq * units;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * NT + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * NT) {
        const int64_t b = i / units;
        const int t = static_cast<int>(i - b * units) * 8;
        float v[8];
        if (w.targets[b] == w.ignore) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = 0.f;
        } else {
            load8(q + b * ldq, t, d, v);
            const float u = w.u(b), f = u == 0.f ? 0.f : u / mx * top;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] *= f;
        }
        if constexpr (sizeof(T) == 4)
            store_planes(v, static_cast<__nv_bfloat16*>(out) + b * ldo + t, nq * ldo);
        else
            *reinterpret_cast<uint4*>(static_cast<T*>(out) + b * ldo + t) =
                make_uint4(pack16<T>(v[0], v[1]), pack16<T>(v[2], v[3]), pack16<T>(v[4], v[5]), pack16<T>(v[6], v[7]));
    }
}

// fp32 rows -> three bf16 planes [3][n][ldo], ldo a multiple of 8
__global__ void __launch_bounds__(NT)
    xent_split_kernel(const float* x, int64_t n, int64_t ldx, int d, __nv_bfloat16* out, int64_t ldo) {
    chain_wait();
    const int64_t units = ldo / 8, total = n * units;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * NT + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * NT) {
        const int64_t r = i / units;
        const int t = static_cast<int>(i - r * units) * 8;
        float v[8];
        load8(x + r * ldx, t, d, v);
        store_planes(v, out + r * ldo + t, n * ldo);
    }
}

struct ProbArgs {
    int64_t nq, n, row0;  // queries, rows of the piece, its first row
    int nqb, njobs, nkb, nseg;
    int q_rows, width;    // box rows of the queries, columns of a tile
    float c;
    const int64_t* targets;
    int64_t ignore;
    const float* stats;
};

// G tiles of one piece: 2^14 (p - [n = t]) / (1 - p_t)
template <typename T>
struct ProbPolicy {
    static constexpr bool kInt8 = false;
    static constexpr int kAccCols = TT_N;
    static constexpr int kStages = 5, kStgBytes = TT_STG_BYTES;
    [[maybe_unused]] static constexpr bool kBMn = false;
    const CUtensorMap *mq, *mx, *mg;
    const ProbArgs& a;

    using Job = TileJob;
    struct Iter {
        const ProbPolicy& p;
        int i, step;
        __device__ Iter(const ProbPolicy& pol, int pair, int npairs) : p(pol), i(pair), step(npairs) {}
        __device__ __forceinline__ bool next(Job& j) {
            if (i >= p.a.njobs) return false;
            j.ma = p.mq;
            j.mb = p.mx;
            j.m0 = i % p.a.nqb * TT_M;
            j.n0 = i / p.a.nqb * p.a.width;
            j.nn = p.a.width;
            j.k0 = 0;
            j.nk = p.a.nkb;
            j.nseg = p.a.nseg;
            j.a_mn = j.b_mn = false;
            j.a_rows = p.a.q_rows;
            j.b_rows = p.a.width / 2;
            j.a_second = j.m0 + 128 < p.a.nq;
            i += step;
            return true;
        }
    };
    using Epi = GTerm;

    __device__ __forceinline__ void begin(Epi& e, const Job& j, const TileCtx& c) const {
        const int64_t b = j.m0 + c.row;
        e = b < a.nq ? GTerm(a.stats, a.targets, b, a.nq, a.ignore, a.row0) : GTerm();
    }

    __device__ __forceinline__ void chunk(Epi& e, const Job& j, const TileCtx& c, int col,
                                          const uint32_t (&r)[32]) const {
        const int y = j.m0 + c.row - c.lane, x = j.n0 + col;
        if (y >= a.nq || x >= a.n) return;
        float v[32];
        const uint64_t c2 = pack2(a.c, a.c), m2 = pack2(-e.m, -e.m), z2 = pack2(-e.lz, -e.lz);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            unpack2(add_f32x2(fma_f32x2(pack2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), c2, m2), z2), x0, x1);
            v[i] = ex2(x0);
            v[i + 1] = ex2(x1);
        }
        if (e.zero) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;
        }
        const int64_t rel = e.tgt - x;
        if (rel >= 0 && rel < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                v[i] = i == static_cast<int>(rel) ? -kGScale : v[i];
        }
        __syncwarp();
        // (columns behind the piece's last row lie outside the map)
#pragma unroll
        for (int k = 0; k < (sizeof(T) == 2 ? 1 : 3); ++k) {
            stg_wait_read(c.lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w[4];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    float &a0 = v[8 * i + 2 * h], &a1 = v[8 * i + 2 * h + 1];
                    if constexpr (sizeof(T) == 2) {
                        w[h] = pack16<T>(a0, a1);
                    } else {
                        w[h] = pack16<__nv_bfloat16>(a0, a1);
                        // what is left for the next plane
                        a0 -= __uint_as_float(w[h] << 16);
                        a1 -= __uint_as_float(w[h] & 0xffff0000u);
                    }
                }
                *reinterpret_cast<uint4*>(c.stg + stg_off64(c.lane, i)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            stg_send<false>(mg, c.stg, c.lane, x, y, k);
        }
    }

    __device__ __forceinline__ void end(Epi&, const Job&, const TileCtx&) const {}
    __device__ __forceinline__ void finish(const TileCtx& c) const { stg_drain(c.lane); }
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TT_THREADS, 1)
    xent_prob_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mx,
                     const __grid_constant__ CUtensorMap mg, const __grid_constant__ ProbArgs a, const bool bf16, const TileStatus st) {
    extern __shared__ uint8_t smem_raw[];
    const ProbPolicy<T> p{&mq, &mx, &mg, a};
    tile_loop(smem_raw, p, bf16, st);
}

__global__ void __launch_bounds__(TF_THREADS, 1)
    xent_prob_f32_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mg,
                         const __grid_constant__ F32Rows x, const __grid_constant__ ProbArgs a, const TileStatus st) {
    extern __shared__ uint8_t smem_raw[];
    const ProbPolicy<float> p{&mq, nullptr, &mg, a};
    tile_loop_f32(smem_raw, p, x, st);
}

struct GradArgs {
    int64_t nq, n;         // queries, rows of the piece
    int d, nseg;
    int nt, width;         // column tiles of d, their columns
    int q_rows;            // box rows of G as dq's operand
    int q_blocks, q_split, q_per;  // dq: 256-query blocks, K splits, K blocks per split (0 blocks: not wanted)
    int kc, kq;            // K blocks of the piece and of the queries
    int x_blocks;          // dx: 256-row blocks (0: not wanted)
    bool q_first;          // the longer tiles come first
    bool add;              // a piece before this one wrote the partial sums
    void* dx;              // rows of the piece, where dx_tma is false
    int64_t lddx;
    bool dx_tma;           // the rows of dx have 16-byte strides
    bool dx_sums;          // dx in 16 bits goes to fp32 sums first, by mdx
    float scale;
    const float* wmax;     // what dx has to be multiplied with besides
};

// A tile's K axis is walked in runs of this many blocks of 64, added up in rounded
// fp32 where the result lies, by the one CTA that owns the tile: the tensor cores
// cut an accumulator towards zero at every instruction (four a block), by 1e-7 of
// the final sum each where all terms have one sign (dq over 2^25 rows in one run a
// split: 3.3e-3 too small).  fp32: 32 cuts of the large accumulator.  16 bits: 512,
// 5e-5, where the result is rounded by up to 5e-4 (fp16); backward of 4,096 x
// 131,072 x 768 bf16 1,876 us, 1,853 in one run, 1,919 in runs of 64 blocks.  dx in
// 16 bits is stored after one run, and only more than 8,192 queries need fp32 sums
// beside it.
constexpr int kRun32 = 8, kRun16 = 128;

template <typename T>
struct GradPolicy {
    static constexpr bool kInt8 = false;
    static constexpr int kAccCols = TT_N;
    static constexpr int kStages = 5, kStgBytes = TT_STG_BYTES;
    [[maybe_unused]] static constexpr bool kBMn = true;
    const CUtensorMap *gk, *gmn, *xmn, *qmn, *mpart, *mdx;
    const GradArgs& a;

    struct Job : TileJob {
        bool is_dx, more;  // more: adds to what this CTA stored before
        int split;
    };
    static constexpr int kRun = sizeof(T) == 4 ? kRun32 : kRun16;
    struct Iter {
        const GradPolicy& p;
        int i, step, left;  // K blocks of the last tile still to do
        __device__ Iter(const GradPolicy& pol, int pair, int npairs) : p(pol), i(pair), step(npairs), left(0) {}
        __device__ __forceinline__ bool next(Job& j) {
            const GradArgs& a = p.a;
            if (left > 0) {
                j.more = true;
                j.k0 += kRun;
                j.nk = min(left, kRun);
                left -= j.nk;
                return true;
            }
            j.more = false;
            const int nqj = a.q_blocks * a.nt * a.q_split, nxj = a.x_blocks * a.nt;
            if (i >= nqj + nxj) return false;
            const int head = a.q_first ? nqj : nxj;
            j.is_dx = (i < head) != a.q_first;
            int k = i < head ? i : i - head;
            i += step;
            j.nseg = a.nseg;
            j.b_mn = true;
            j.b_rows = 128;
            j.n0 = k % a.nt * a.width;
            k /= a.nt;
            j.nn = min(a.width, (a.d - j.n0 + 127) / 128 * 128);
            if (j.is_dx) {
                j.ma = p.gmn;
                j.mb = p.qmn;
                j.a_mn = true;
                j.a_rows = 128;
                j.m0 = k * TT_M;
                j.a_second = j.m0 + 128 < a.n;
                j.k0 = 0;
                j.nk = a.kq;
                j.split = 0;
            } else {
                j.ma = p.gk;
                j.mb = p.xmn;
                j.a_mn = false;
                j.split = k / a.q_blocks;
                j.m0 = k % a.q_blocks * TT_M;
                j.a_rows = a.q_rows;
                j.a_second = j.m0 + 128 < a.nq;
                j.k0 = j.split * a.q_per;
                j.nk = min(a.q_per, a.kc - j.k0);
            }
            left = max(0, j.nk - kRun);
            j.nk -= left;
            return true;
        }
    };
    struct Epi {
        float f;
    };

    __device__ __forceinline__ void begin(Epi& e, const Job& j, const TileCtx&) const {
        e.f = j.is_dx ? a.scale * (1.f / kGScale) * *a.wmax : 1.f;
    }

    __device__ __forceinline__ void chunk(Epi& e, const Job& j, const TileCtx& c, int col,
                                          const uint32_t (&r)[32]) const {
        const int y = j.m0 + c.row - c.lane, x = j.n0 + col;
        if (x >= a.d || y >= (j.is_dx ? a.n : a.nq)) return;
        if (j.is_dx && !a.dx_tma) {
            stg_wait_read(c.lane);
            // rows that no tensor map can describe: transposed in the staging
            // bytes, so that a store writes 32 columns of one row
            float* t = reinterpret_cast<float*>(c.stg);
#pragma unroll
            for (int i = 0; i < 32; ++i) t[c.lane * 32 + ((i + c.lane) & 31)] = __uint_as_float(r[i]) * e.f;
            __syncwarp();
            T* o = static_cast<T*>(a.dx) + static_cast<int64_t>(y) * a.lddx + x + c.lane;
            const int rows = static_cast<int>(min(static_cast<int64_t>(32), a.n - y));
            if (x + c.lane < a.d)
                for (int i = 0; i < rows; ++i, o += a.lddx) {
                    float v = t[i * 32 + ((c.lane + i) & 31)];
                    if (sizeof(T) == 4 && j.more) v += to_f(*o);
                    *o = from_f<T>(v);
                }
            __syncwarp();
            return;
        }
        if (j.more)
            stg_drain(c.lane);  // what is added to has been written
        else
            stg_wait_read(c.lane);
        bool wide = true;
        if constexpr (sizeof(T) == 2) {
            if (j.is_dx && !a.dx_sums) {
                wide = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t w[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        w[h] = pack16<T>(__uint_as_float(r[8 * i + 2 * h]) * e.f,
                                         __uint_as_float(r[8 * i + 2 * h + 1]) * e.f);
                    *reinterpret_cast<uint4*>(c.stg + stg_off64(c.lane, i)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        if (wide) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                *reinterpret_cast<float4*>(c.stg + stg_off128(c.lane, i)) =
                    make_float4(__uint_as_float(r[4 * i]) * e.f, __uint_as_float(r[4 * i + 1]) * e.f,
                                __uint_as_float(r[4 * i + 2]) * e.f, __uint_as_float(r[4 * i + 3]) * e.f);
        }
        if (j.is_dx && j.more)
            stg_send<true>(mdx, c.stg, c.lane, x, y, 0);
        else if (j.is_dx)
            stg_send<false>(mdx, c.stg, c.lane, x, y, 0);
        else if (a.add || j.more)
            stg_send<true>(mpart, c.stg, c.lane, x, y, j.split);
        else
            stg_send<false>(mpart, c.stg, c.lane, x, y, j.split);
    }

    __device__ __forceinline__ void end(Epi&, const Job&, const TileCtx&) const {}
    __device__ __forceinline__ void finish(const TileCtx& c) const { stg_drain(c.lane); }
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TT_THREADS, 1)
    xent_grad_kernel(const __grid_constant__ CUtensorMap gk, const __grid_constant__ CUtensorMap gmn,
                     const __grid_constant__ CUtensorMap xmn, const __grid_constant__ CUtensorMap qmn,
                     const __grid_constant__ CUtensorMap mpart, const __grid_constant__ CUtensorMap mdx,
                     const __grid_constant__ GradArgs a, const bool bf16, const TileStatus st) {
    extern __shared__ uint8_t smem_raw[];
    const GradPolicy<T> p{&gk, &gmn, &xmn, &qmn, &mpart, &mdx, a};
    tile_loop(smem_raw, p, bf16, st);
}

// dq of at most 128 queries from fp32 rows as they are
__global__ void __launch_bounds__(TF_THREADS, 1)
    xent_grad_f32_kernel(const __grid_constant__ CUtensorMap gk, const __grid_constant__ CUtensorMap mpart,
                         const __grid_constant__ F32Rows x, const __grid_constant__ GradArgs a, const TileStatus st) {
    extern __shared__ uint8_t smem_raw[];
    const GradPolicy<float> p{&gk, nullptr, nullptr, nullptr, &mpart, nullptr, a};
    tile_loop_f32(smem_raw, p, x, st);
}

// dq_b = u_b scale 2^-14 (sum of the parts, in split order)
template <typename T>
__global__ void __launch_bounds__(NT)
    xent_dq_kernel(const float* part, int splits, int64_t nq, int d, int dp, const Weights w, float scale, T* dq,
                   int64_t lddq) {
    chain_wait();
    const int64_t units = dp / 4, total = nq * units;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * NT + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * NT) {
        const int64_t b = i / units;
        const int t = static_cast<int>(i - b * units) * 4;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int k = 0; k < splits; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(part + (k * nq + b) * dp + t);
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        const bool skip = w.targets[b] == w.ignore;
        const float f = w.u(b) * scale * (1.f / kGScale);
        const float o[4] = {s.x * f, s.y * f, s.z * f, s.w * f};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (t + k < d) dq[b * lddq + t + k] = from_f<T>(skip ? 0.f : o[k]);
    }
}

// dx in 16 bits from its sums in fp32
template <typename T>
__global__ void __launch_bounds__(NT)
    xent_dx_kernel(const float* sums, int64_t n, int d, int dp, T* dx, int64_t lddx) {
    chain_wait();
    const int64_t units = dp / 4, total = n * units;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * NT + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * NT) {
        const int64_t r = i / units;
        const int t = static_cast<int>(i - r * units) * 4;
        const float4 v = *reinterpret_cast<const float4*>(sums + r * dp + t);
        const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (t + k < d) dx[r * lddx + t + k] = from_f<T>(o[k]);
    }
}

// -------------------------------------------------------------- host side --

constexpr int64_t kMaxRows = (1LL << 31) - 1;
constexpr int kMaxDim = INT_MAX - 256;  // K blocks are counted in int

// sizes for which there is a plan
bool plannable(int dtype, int64_t nq, int64_t n, int d) {
    return elem_size(dtype) != 0 && nq >= 0 && nq <= kMaxRows && n >= 1 && n <= kMaxRows && d >= 1 && d <= kMaxDim;
}

int check_common(int dtype, const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n, int64_t ldx, int d,
                 const int64_t* targets, float scale, int reduction) {
    const int64_t e = (int64_t)elem_size(dtype);
    RDB_CHECK_ARG(e != 0, "unknown dtype %d", dtype);
    RDB_CHECK_ARG(nq >= 0 && n >= 1 && d >= 1 && ldq >= d && ldx >= d, "bad shape");
    RDB_CHECK_ARG(nq <= kMaxRows && n <= kMaxRows, "nq and n must be < 2^31");
    RDB_CHECK_ARG(d <= kMaxDim, "d must be < 2^31 - 256");
    RDB_CHECK_ARG(scale > 0.f && scale <= 2.0e38f, "scale must be positive and finite");
    RDB_CHECK_ARG(reduction >= RDB_REDUCE_NONE && reduction <= RDB_REDUCE_SUM, "unknown reduction %d", reduction);
    RDB_CHECK_ARG(x && (nq == 0 || (q && targets)), "NULL pointer");
    RDB_CHECK_ARG((ldq * e) % 16 == 0 && (ldx * e) % 16 == 0, "row strides must be multiples of 16 bytes");
    RDB_CHECK_ARG((reinterpret_cast<uintptr_t>(q) & 15) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0,
                  "base pointers must be 16-byte aligned");
    return RDB_OK;
}

CUtensorMapDataType map_type(int dtype) {
    return dtype == RDB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// operand rows as 16-bit planes: the caller's rows, or the bf16 planes of fp32
struct Planes {
    const void* p;
    int64_t ld, plane;  // elements
    int count;
};

// box_rows: of a K-major operand; 0: MN-major
int operand_map(CUtensorMap* m, int dtype, const Planes& o, int64_t cols, int64_t rows, int box_rows) {
    return make_map_3d(m, map_type(dtype), 2, o.p, cols, rows, o.count, o.ld * 2,
                       o.count > 1 ? o.plane * 2 : 0, box_rows ? box_rows : 64);
}

struct Arena {
    char* base;
    size_t used = 0;
    template <typename T>
    T* take(size_t count) {
        T* p = reinterpret_cast<T*>(base + used);
        used += (count * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

// rows of a piece: n split evenly into pieces of at most `most` (a multiple of 256)
int64_t piece_rows(int64_t n, int64_t most) {
    most = std::max<int64_t>(256, most / 256 * 256);
    const int64_t pieces = (n + most - 1) / most;
    return up((n + pieces - 1) / pieces, 256);
}

struct FwdPlan {
    int64_t rows;  // rows per piece
    bool stream, direct;
    int pieces, nqb, nkb, nseg, groups, workers, slots, width, nsplit[2];  // nsplit of a full and of the last piece
};

// Row splits of one piece: as many as give every pair the same number of rows
// (in groups of 32), for the number of rounds that costs least; a split costs
// about a third of a tile (its fill and parts).  A tile counts as 256 columns; of
// the direct plan's 128 two count as one.
int fwd_splits(int nqb, int64_t rows, int pairs) {
    const int64_t n32 = (rows + 31) / 32;
    int64_t best = 1;
    double best_cost = 1e30;
    for (int64_t round = 1; round <= 16; ++round) {
        const int64_t s = std::max<int64_t>(1, std::min<int64_t>(n32, round * pairs / nqb));
        const double tiles = (double)((n32 + s - 1) / s) / (TT_N / 32);
        const double cost = (double)((nqb * s + pairs - 1) / pairs) * (tiles + 0.3);
        if (cost < best_cost) best_cost = cost, best = s;
    }
    return (int)best;
}

// fp32 rows are split on the way (tile_f32.cuh) where one block of 128 queries
// reads them; more queries share planes written once per piece.  100,000 x 768, us,
// forward / forward and dq, on the way / by planes (cold L2): 5 queries 153 / 309
// and 429 / 773, 128 queries 159 / 326 and 457 / 872; by planes alone 129 queries 313
// / 847, 256 336 / 906, 1,024 832 / 2,530.  A block holds no more than 128 queries:
// beyond, the rows would be split once per block, and two forward passes of 159 take
// as long as the planes of 129 to 256.
bool f32_direct(int dtype, int64_t nq) { return dtype == RDB_F32 && nq <= 128; }

// A pass of CUDA cores where their products hide behind the rows' bytes: one
// query, or up to four of fp32, whose six products of planes are the tile loop's
// limit.  Whole forward call, us, streaming / tile loop:
//   1 query,  bf16, 100,000 x 768   32.2 / 42.8     1M x 768   254 / 268
//                   200,000 x 384   49 / 49 (shorter rows: equal)
//   2 queries                       52 / 50                    317 / 268
//   1 query,  fp32, 100,000 x 768   74 / 150        1M x 768   473 / 1,155
//   4 queries                       78 / 150                   551 / 1,155
bool streamed(int dtype, int64_t nq, int d) {
    return nq >= 1 && nq <= (dtype == RDB_F32 ? 4 : 1) && d <= ST_MAX_DIM;
}

int stream_blocks(int64_t nq, int64_t rows) {
    return (int)std::min<int64_t>((rows + 31) / 32, (nq == 1 ? 2LL : 1LL) * num_sms());
}

FwdPlan fwd_plan(int dtype, int64_t nq, int64_t n, int d) {
    FwdPlan p{};
    const int64_t dp = up(d, 8);
    p.stream = streamed(dtype, nq, d);
    if (p.stream) {
        p.pieces = p.groups = 1;
        p.slots = stream_blocks(nq, n);
        return p;
    }
    p.direct = f32_direct(dtype, nq);
    // fp32: 256 MB of planes at a time
    p.rows = dtype == RDB_F32 && !p.direct ? piece_rows(n, (256LL << 20) / (6 * dp)) : up(n, 256);
    p.pieces = (int)((n + p.rows - 1) / p.rows);
    p.nqb = (int)std::max<int64_t>(1, (nq + TT_M - 1) / TT_M);
    p.nkb = (d + 63) / 64;
    p.nseg = dtype == RDB_F32 ? 6 : 1;
    p.groups = p.direct ? TF_GROUPS : TT_GROUPS;
    p.workers = p.direct ? num_sms() : tile_pairs();
    p.nsplit[0] = fwd_splits(p.nqb, std::min(p.rows, n), p.workers);
    p.nsplit[1] = fwd_splits(p.nqb, n - (p.pieces - 1) * p.rows, p.workers);
    // (few rows in all: a narrow tile is all a split has)
    p.width = p.direct ? TF_N
                       : (int)std::min<int64_t>(TT_N, up((up(p.rows, 32) / 32 + p.nsplit[0] - 1) / p.nsplit[0] * 32, 64));
    p.slots = (p.pieces - 1) * p.nsplit[0] + p.nsplit[1];
    return p;
}

struct FwdWs {
    unsigned* ticket;
    float2* part;
    __nv_bfloat16 *qp, *xp;
    size_t bytes;
};

FwdWs fwd_ws(void* base, const FwdPlan& p, int dtype, int64_t nq, int d) {
    FwdWs w{};
    Arena a{static_cast<char*>(base)};
    const int64_t dp = up(d, 8);
    w.ticket = a.take<unsigned>(1);
    w.part = a.take<float2>((size_t)p.groups * p.slots * nq);
    if (dtype == RDB_F32 && !p.stream) {
        w.qp = a.take<__nv_bfloat16>(3 * nq * dp);
        if (!p.direct) w.xp = a.take<__nv_bfloat16>(3 * p.rows * dp);
    }
    w.bytes = a.used + 256;
    return w;
}

struct BwdPlan {
    int64_t rows;  // rows per piece
    bool stream;   // rows past CUDA cores (probabilities)
    bool direct;   // fp32 rows split on the way (dq, probabilities)
    bool dx_sums;  // dx of a piece in fp32 first
    int pieces, planes, nqb, nt, nkb, nseg, kq, dp;
    int q_nt, q_width, q_split, q_per;  // dq: column tiles, K splits, K blocks per split
    bool q_first;
};

// Rounds of `jobs` tiles dealt out in turn to `workers`.
int64_t rounds(int64_t jobs, int64_t workers) { return (jobs + workers - 1) / workers; }

BwdPlan bwd_plan(int dtype, int64_t nq, int64_t n, int d, bool need_dq, bool need_dx) {
    BwdPlan p;
    p.stream = streamed(dtype, nq, d);
    p.direct = f32_direct(dtype, nq);
    p.planes = dtype == RDB_F32 ? 3 : 1;
    p.nseg = dtype == RDB_F32 ? 6 : 1;
    p.kq = (int)((nq + 63) / 64);
    p.dp = (int)up(d, 32);
    p.dx_sums = need_dx && dtype != RDB_F32 && p.kq > kRun16;
    const int64_t col = std::max<int64_t>(1, nq * 2 * p.planes);  // bytes of G per row
    // G of a piece: 512 MB.  Pieces that stay in L2 (64 MB) have fewer tiles to
    // deal out and more launches, and the products are bound by the tensor
    // cores, not by reading G: 4,096 x 131,072 x 768 both gradients 2,013 us at
    // 64 MB, 1,971 at 128, 1,924 at 256, 1,865 at 512.  At least 4,096 rows
    // within 2 GB: the partial sums of dq are read and written once a piece.  Never
    // less than a tile's 256 rows.
    int64_t most = (512LL << 20) / col;
    if (most < 4096) most = std::max(most, std::min<int64_t>(4096, (2LL << 30) / col));
    if (dtype == RDB_F32 && !p.direct) most = std::min<int64_t>(most, (256LL << 20) / (6 * up(d, 8)));
    if (p.dx_sums) most = std::min<int64_t>(most, (512LL << 20) / (4LL * p.dp));  // (counts from d = 4,096 on)
    p.rows = piece_rows(n, most);
    p.pieces = (int)((n + p.rows - 1) / p.rows);
    p.nqb = (int)std::max<int64_t>(1, (nq + TT_M - 1) / TT_M);
    p.nt = (d + TT_N - 1) / TT_N;
    p.nkb = (d + 63) / 64;
    p.q_width = p.direct ? TF_N : TT_N;
    p.q_nt = (d + p.q_width - 1) / p.q_width;
    // K splits of dq: the split that ends first, tiles dealt out in turn; a
    // tile costs about six K blocks on top of its own (fill, drain, store).
    // Direct dq tiles have a launch of their own.  Limits: 64 splits (4 x 200,000 x
    // 768 bf16 backward 137 us with up to 16, 126 with 32 to 256; 32 queries 159, 141
    // with 32 to 128, 135 with 256), of the direct plan about one per SM (8 and 128 x
    // 100,000 x 768 fp32: the same within 3 % from 40 to 320), and 64 MB of parts
    // (4,096 x 131,072 x 768 1,371 us at 16 MB, 1,255 at 64 and at 256).
    const int64_t workers = p.direct ? num_sms() : tile_pairs(), kc = std::min(p.rows, up(n, 64)) / 64;
    const int64_t nx = need_dx && !p.direct ? (p.rows + TT_M - 1) / TT_M * p.nt : 0, lx = (int64_t)p.kq * p.nseg + 6;
    p.q_split = 1;
    p.q_per = (int)kc;
    if (need_dq) {
        int64_t best = INT64_MAX;
        const int64_t most_splits = std::min<int64_t>(kc, p.direct ? 160 : 64);
        for (int64_t s = 1; s <= most_splits; ++s) {
            if (s > 1 && s * nq * p.dp * 4 > (64LL << 20)) break;
            const int64_t per = (kc + s - 1) / s, used = (kc + per - 1) / per;
            if (used < s) continue;
            const int64_t nj = (int64_t)p.nqb * p.q_nt * used, lq = per * p.nseg + 6;
            int64_t cost = rounds(nj, workers) * lq + rounds(nx, workers) * lx;
            if (nx) {
                // tiles of the second kind fill the first's last round
                const int64_t rest = std::max<int64_t>(0, nx - (rounds(nj, workers) * workers - nj));
                cost = std::min(cost, rounds(nj, workers) * std::max(lq, lx) + rounds(rest, workers) * lx);
            }
            cost += s / 4;  // parts to join
            if (cost < best) best = cost, p.q_split = (int)used, p.q_per = (int)per;
        }
    }
    p.q_first = (int64_t)p.q_per >= p.kq;
    return p;
}

struct BwdWs {
    float *wmax, *part, *dx;
    float2* wparts;
    void *g, *qw;
    __nv_bfloat16 *qp, *xp;
    size_t bytes;
};

BwdWs bwd_ws(void* base, const BwdPlan& p, int dtype, int64_t nq, int d, bool need_dq, bool need_dx) {
    BwdWs w{};
    Arena a{static_cast<char*>(base)};
    const int64_t d8 = up(d, 8);
    w.wmax = a.take<float>(1);
    if (need_dx) w.wparts = a.take<float2>(kWeightBlocks);
    w.g = a.take<uint16_t>((size_t)p.planes * nq * p.rows);
    if (need_dq) w.part = a.take<float>((size_t)p.q_split * nq * p.dp);
    if (need_dx) w.qw = a.take<uint16_t>((size_t)p.planes * nq * d8);
    if (p.dx_sums) w.dx = a.take<float>((size_t)p.rows * p.dp);
    if (dtype == RDB_F32) {
        w.qp = a.take<__nv_bfloat16>(3 * nq * d8);
        if (!p.direct) w.xp = a.take<__nv_bfloat16>(3 * p.rows * d8);
    }
    w.bytes = a.used + 256;
    return w;
}

unsigned elementwise_blocks(int64_t items) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + NT - 1) / NT, 8LL * num_sms()));
}

// tile width of the probability pass: 256, or narrower where that deals the
// rows of few query blocks out more evenly (a tile costs about 48 columns more
// than its width)
int prob_width(int64_t rows, int nqb, int pairs) {
    int best = TT_N;
    double best_cost = 1e30;
    for (int w = TT_N; w >= 64; w /= 2) {
        const double jobs = (double)((rows + w - 1) / w) * nqb;
        const double cost = std::ceil(jobs / pairs) * (w + 48);
        if (cost < 0.97 * best_cost) best_cost = cost, best = w;
    }
    return best;
}

int split_rows(const void* x, int64_t n, int64_t ldx, int d, __nv_bfloat16* out, cudaStream_t s) {
    RDB_TRY(launch_chained(xent_split_kernel, elementwise_blocks(n * up(d, 8) / 8), NT, 0, s,
                           static_cast<const float*>(x), n, ldx, d, out, up(d, 8)));
    return RDB_OK;
}

// Whether every block of the weighted queries' launch finds the largest weight
// itself, or a launch before it does.  Captured backward pass, us, itself / before:
// 256 x 256 x 768 bf16 20.8 / 22.5, 1,024 x 1,024 x 256 24.6 / 24.8, 2,048 x 4,096 x
// 128 34.7 / 32.8.  fp16, which reads the queries for it: always before (77 x 5,003
// x 100 30.7 / 24.6).
bool scan_weights(int dtype, int64_t nq) { return dtype != RDB_F16 && nq <= 1024; }

// rows [r0, r0 + rows) as operand planes (fp32: split into xp first)
int piece_operand(int dtype, const void* x, int64_t r0, int64_t rows, int64_t ldx, int d, __nv_bfloat16* xp, Planes* o,
                  cudaStream_t s) {
    const char* base = static_cast<const char*>(x) + r0 * ldx * (int64_t)elem_size(dtype);
    if (dtype != RDB_F32) {
        *o = {base, ldx, 0, 1};
        return RDB_OK;
    }
    *o = {xp, up(d, 8), rows * up(d, 8), 3};
    return split_rows(base, rows, ldx, d, xp, s);
}

template <typename T, int NQ, bool PROB>
int launch_stream_t(const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n, int64_t ldx, int d,
                    const int64_t* targets, float c, const StreamOut& out, int blocks, cudaStream_t s) {
    constexpr int k = sizeof(T) == 4 ? 2 : 1;  // units of 8 elements
    const auto kernel = d * (int)sizeof(T) <= 512 ? xent_stream_kernel<T, NQ, 1, PROB>
                        : d <= 256                ? xent_stream_kernel<T, NQ, k, PROB>
                        : d <= 512                ? xent_stream_kernel<T, NQ, 2 * k, PROB>
                        : d <= 768                ? xent_stream_kernel<T, NQ, 3 * k, PROB>
                                                  : xent_stream_kernel<T, NQ, 4 * k, PROB>;
    return launch_chained(kernel, (unsigned)blocks, NT, 0, s, static_cast<const T*>(q), (int)nq, ldq,
                          static_cast<const T*>(x), n, ldx, d, targets, c, out);
}

template <bool PROB>
int launch_stream(int dtype, const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n, int64_t ldx, int d,
                  const int64_t* targets, float c, const StreamOut& out, int blocks, cudaStream_t s) {
    const auto launch = dtype == RDB_BF16  ? launch_stream_t<__nv_bfloat16, 1, PROB>
                        : dtype == RDB_F16 ? launch_stream_t<__half, 1, PROB>
                        : nq == 1          ? launch_stream_t<float, 1, PROB>
                                           : launch_stream_t<float, 4, PROB>;
    return launch(q, nq, ldq, x, n, ldx, d, targets, c, out, blocks, s);
}

template <typename T>
int backward_t(int dtype, const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n, int64_t ldx, int d,
               const int64_t* targets, float scale, int64_t ignore, int reduction, const float* grad,
               const float* stats, void* dq, int64_t lddq, void* dx, int64_t lddx, void* ws, cudaStream_t s) {
    static bool attr_p[64] = {false}, attr_g[64] = {false}, attr_dp[64] = {false}, attr_dg[64] = {false};
    const BwdPlan p = bwd_plan(dtype, nq, n, d, dq != nullptr, dx != nullptr);
    const BwdWs w = bwd_ws(ws, p, dtype, nq, d, dq != nullptr, dx != nullptr);
    const int64_t d8 = up(d, 8);
    const TileStatus st = tile_status();
    const bool bf16 = dtype != RDB_F16;
    const int pairs = tile_pairs();
    if (p.direct) {
        RDB_TRY(tile_f32_smem_attr(xent_prob_f32_kernel, attr_dp));
        RDB_TRY(tile_f32_smem_attr(xent_grad_f32_kernel, attr_dg));
    } else {
        RDB_TRY(tile_smem_attr(xent_prob_kernel<T>, attr_p));
    }
    RDB_TRY(tile_smem_attr(xent_grad_kernel<T>, attr_g));

    const Weights wt{grad,
                     reduction == RDB_REDUCE_MEAN ? stats + 3 * nq : nullptr,
                     stats + 2 * nq,
                     targets,
                     ignore,
                     reduction != RDB_REDUCE_NONE};
    if (dx) {
        const bool scan = scan_weights(dtype, nq);
        const int per = dtype == RDB_F16 ? NT / 32 : NT;  // queries a block reads at a time
        const int nparts = scan ? 0 : (int)std::min<int64_t>(kWeightBlocks, (nq + per - 1) / per);
        if (!scan) {
            RDB_TRY(launch_chained(xent_wmax_kernel<T>, nparts, NT, 0, s, static_cast<const T*>(q), nq, ldq, d, wt,
                                   w.wparts));
        }
        const int64_t items = nq * d8 / 8;
        RDB_TRY(launch_chained(xent_weighted_kernel<T>,
                               scan ? (unsigned)std::min<int64_t>((items + NT - 1) / NT, num_sms()) : elementwise_blocks(items),
                               NT, 0, s, static_cast<const T*>(q), nq, ldq, d, wt, w.wparts, nparts, w.wmax, w.qw, d8));
    }
    Planes qo{w.qp, d8, nq * d8, 3};
    if (!p.stream || dtype != RDB_F32) RDB_TRY(piece_operand(dtype, q, 0, nq, ldq, d, w.qp, &qo, s));
    CUtensorMap mq, mqw;  // (mq of streamed queries is read by nobody)
    RDB_TRY(operand_map(&mq, dtype, qo, d, nq, tile_box_rows(nq, 128)));
    mqw = mq;
    if (dx) RDB_TRY(operand_map(&mqw, dtype, Planes{w.qw, d8, nq * d8, p.planes}, d, nq, 0));

    ProbArgs pa{};
    pa.nq = nq;
    pa.nqb = p.nqb;
    pa.nkb = p.nkb;
    pa.q_rows = tile_box_rows(nq, 128);
    pa.nseg = p.nseg;
    pa.c = (float)(scale * kLog2e);
    pa.targets = targets;
    pa.ignore = ignore;
    pa.stats = stats;
    GradArgs ga{};
    ga.nq = nq;
    ga.d = d;
    ga.nseg = p.nseg;
    ga.nt = p.nt;
    ga.width = TT_N;
    ga.q_rows = tile_box_rows(nq, 128);
    ga.q_per = p.q_per;
    ga.kq = p.kq;
    ga.q_first = p.q_first;
    ga.lddx = lddx;
    ga.dx_sums = p.dx_sums;
    ga.dx_tma = p.dx_sums || (dx && (reinterpret_cast<uintptr_t>(dx) & 15) == 0 && (lddx * (int64_t)sizeof(T)) % 16 == 0);
    ga.scale = scale;
    ga.wmax = w.wmax;
    const Planes go{w.g, p.rows, nq * p.rows, p.planes};
    CUtensorMap mpart = mq, mdx = mq;  // (any valid map where there is nothing to store)
    if (dq)
        RDB_TRY(make_store_map(&mpart, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, w.part, p.dp, nq, p.q_split, 4LL * p.dp,
                               4LL * p.dp * nq));

    for (int i = 0; i < p.pieces; ++i) {
        const int64_t r0 = i * p.rows, rows = std::min(p.rows, n - r0);
        const F32Rows xr{static_cast<const float*>(x) + r0 * ldx, ldx, rows, d};  // (direct only)
        CUtensorMap mx, mxmn = mq, mgk, mgmn, mg;
        RDB_TRY(operand_map(&mgk, dtype, go, rows, nq, ga.q_rows));
        RDB_TRY(operand_map(&mgmn, dtype, go, rows, nq, 0));
        RDB_TRY(make_store_map(&mg, map_type(dtype), 2, w.g, rows, nq, p.planes, 2 * p.rows, 2 * p.rows * nq));
        pa.n = rows;
        pa.row0 = r0;
        pa.width = p.direct ? TF_N : prob_width(rows, p.nqb, pairs);
        const int64_t tiles = (rows + pa.width - 1) / pa.width * p.nqb;
        RDB_CHECK_ARG(tiles < (1LL << 31), "too many tiles for one launch");
        pa.njobs = (int)tiles;
        if (p.stream)
            RDB_TRY(launch_stream<true>(dtype, q, nq, ldq, static_cast<const T*>(x) + r0 * ldx, rows, ldx, d, targets,
                                        pa.c, StreamOut{nullptr, nullptr, w.g, p.rows, nq * p.rows, r0, stats, ignore},
                                        stream_blocks(nq, rows), s));
        else if (p.direct)
            RDB_TRY(launch_chained(xent_prob_f32_kernel, (unsigned)std::min<int64_t>(num_sms(), tiles), TF_THREADS,
                                   TF_SMEM, s, mq, mg, xr, pa, st));
        if (!p.direct) {
            Planes xo;
            RDB_TRY(piece_operand(dtype, x, r0, rows, ldx, d, w.xp, &xo, s));
            RDB_TRY(operand_map(&mx, dtype, xo, d, rows, pa.width / 2));
            RDB_TRY(operand_map(&mxmn, dtype, xo, d, rows, 0));
            if (!p.stream)
                RDB_TRY(launch_chained(xent_prob_kernel<T>, 2 * (unsigned)std::min<int64_t>(pairs, tiles), TT_THREADS,
                                   TT_SMEM, s, mq, mx, mg, pa, bf16, st));
        }

        ga.n = rows;
        ga.kc = (int)((rows + 63) / 64);
        // a shorter last piece may leave splits without rows: their parts stay
        ga.q_split = (ga.kc + p.q_per - 1) / p.q_per;
        ga.add = i > 0;
        ga.dx = dx ? static_cast<T*>(dx) + r0 * lddx : nullptr;
        if (p.dx_sums)
            RDB_TRY(make_store_map(&mdx, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, w.dx, p.dp, rows, 1, 4LL * p.dp, 0));
        else if (ga.dx_tma)
            RDB_TRY(make_store_map(&mdx, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : map_type(dtype),
                                   (int)sizeof(T), ga.dx, d, rows, 1, lddx * (int64_t)sizeof(T), 0));
        if (p.direct && dq) {
            GradArgs gq = ga;
            gq.nt = p.q_nt;
            gq.width = p.q_width;
            gq.q_blocks = 1;
            gq.x_blocks = 0;
            gq.q_first = true;
            const int64_t jobs = (int64_t)gq.nt * gq.q_split;
            RDB_TRY(launch_chained(xent_grad_f32_kernel, (unsigned)std::min<int64_t>(num_sms(), jobs), TF_THREADS,
                                   TF_SMEM, s, mgk, mpart, xr, gq, st));
        }
        ga.q_blocks = dq && !p.direct ? p.nqb : 0;
        ga.x_blocks = dx ? (int)((rows + TT_M - 1) / TT_M) : 0;
        const int64_t jobs = (int64_t)ga.nt * ((int64_t)ga.q_blocks * ga.q_split + ga.x_blocks);
        if (jobs == 0) continue;
        RDB_CHECK_ARG(jobs < (1LL << 31), "too many tiles for one launch");
        RDB_TRY(launch_chained(xent_grad_kernel<T>, 2 * (unsigned)std::min<int64_t>(pairs, jobs), TT_THREADS, TT_SMEM,
                               s, mgk, mgmn, mxmn, mqw, mpart, mdx, ga, bf16, st));
        if constexpr (sizeof(T) == 2) {
            if (p.dx_sums)
                RDB_TRY(launch_chained(xent_dx_kernel<T>, elementwise_blocks(rows * p.dp / 4), NT, 0, s, w.dx, rows, d,
                                       p.dp, static_cast<T*>(ga.dx), lddx));
        }
    }
    if (dq) {
        RDB_TRY(launch_chained(xent_dq_kernel<T>, elementwise_blocks(nq * p.dp / 4), NT, 0, s, w.part, p.q_split, nq,
                               d, p.dp, wt, scale, static_cast<T*>(dq), lddq));
    }
    return RDB_OK;
}

// (max, sum) of every query's parts
int tile_pass(int dtype, const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n, int64_t ldx, int d,
              const int64_t* targets, float c, const FwdPlan& p, const FwdWs& w, cudaStream_t s) {
    static bool attr[64] = {false}, attr_d[64] = {false};
    if (p.direct)
        RDB_TRY(tile_f32_smem_attr(xent_scan_f32_kernel, attr_d));
    else
        RDB_TRY(tile_smem_attr(xent_scan_kernel, attr));
    const TileStatus st = tile_status();
    Planes qo;
    RDB_TRY(piece_operand(dtype, q, 0, nq, ldq, d, w.qp, &qo, s));
    CUtensorMap mq, mx;
    RDB_TRY(operand_map(&mq, dtype, qo, d, nq, tile_box_rows(nq, 128)));
    FwdArgs a{};
    a.q_rows = tile_box_rows(nq, 128);
    a.width = p.width;
    a.nq = nq;
    a.nqb = p.nqb;
    a.nkb = p.nkb;
    a.nseg = p.nseg;
    a.c = c;
    a.targets = targets;
    a.groups = p.groups;
    a.parts = p.slots * p.groups;
    a.part = w.part;
    a.ticket = w.ticket;
    for (int i = 0; i < p.pieces; ++i) {
        const int64_t r0 = i * p.rows, rows = std::min(p.rows, n - r0);
        a.n = rows;
        a.row0 = r0;
        a.n32 = (int)((rows + 31) / 32);
        a.nsplit = p.nsplit[i == p.pieces - 1];
        a.slot0 = i * p.nsplit[0];
        const int64_t units = (int64_t)a.nsplit * p.nqb;
        RDB_CHECK_ARG(units < (1LL << 31), "too many tiles for one launch");
        const unsigned workers = (unsigned)std::min<int64_t>(p.workers, units);
        if (p.direct) {
            const F32Rows xr{static_cast<const float*>(x), ldx, n, d};
            RDB_TRY(launch_chained(xent_scan_f32_kernel, workers, TF_THREADS, TF_SMEM, s, mq, xr, a, st));
        } else {
            Planes xo;
            RDB_TRY(piece_operand(dtype, x, r0, rows, ldx, d, w.xp, &xo, s));
            RDB_TRY(operand_map(&mx, dtype, xo, d, rows, p.width / 2));
            RDB_TRY(launch_chained(xent_scan_kernel, 2 * workers, TT_THREADS, TT_SMEM, s, mq, mx, a,
                                   dtype != RDB_F16, st));
        }
    }
    return RDB_OK;
}

}  // namespace
}  // namespace rdb

using namespace rdb;

extern "C" {

size_t rdb_softmax_xent_workspace(int dtype, int64_t nq, int64_t n, int d, int reduction) {
    (void)reduction;
    if (!plannable(dtype, nq, n, d)) return 0;
    const FwdPlan p = fwd_plan(dtype, nq, n, d);
    return fwd_ws(nullptr, p, dtype, nq, d).bytes;
}

int rdb_softmax_xent(int dtype, const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n, int64_t ldx, int d,
                     const int64_t* targets, float scale, int64_t ignore_index, int reduction, float* loss,
                     float* stats, void* ws, size_t ws_bytes, void* stream) {
    RDB_TRY(check_common(dtype, q, nq, ldq, x, n, ldx, d, targets, scale, reduction));
    RDB_CHECK_ARG(stats && (loss || (nq == 0 && reduction == RDB_REDUCE_NONE)), "NULL pointer");
    RDB_CHECK_ARG((reinterpret_cast<uintptr_t>(ws) & 15) == 0, "ws must be 16-byte aligned");
    const FwdPlan p = fwd_plan(dtype, nq, n, d);
    const FwdWs w = fwd_ws(ws, p, dtype, nq, d);
    if (!ws || ws_bytes < w.bytes) return set_error(RDB_ERR_WORKSPACE, "workspace too small");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const float c = (float)(scale * kLog2e);
    if (nq > 0) {
        if (p.stream)
            RDB_TRY(launch_stream<false>(dtype, q, nq, ldq, x, n, ldx, d, targets, c,
                                         StreamOut{w.part, w.ticket, nullptr, 0, 0, 0, nullptr, 0}, p.slots, s));
        else
            RDB_TRY(tile_pass(dtype, q, nq, ldq, x, n, ldx, d, targets, c, p, w, s));
        const bool wide = nq <= num_sms();
        const unsigned blocks = (unsigned)std::min<int64_t>(wide ? nq : (nq + NT / 32 - 1) / (NT / 32), 16LL * num_sms());
        const int parts = p.slots * p.groups;
        if (dtype == RDB_F32)
            RDB_TRY(launch_chained(xent_join_kernel<float>, blocks, NT, 0, s, w.part, parts,
                                   static_cast<const float*>(q), ldq, static_cast<const float*>(x), ldx, d, targets,
                                   ignore_index, n, c, nq, wide, stats, loss, reduction, loss, w.ticket));
        else if (dtype == RDB_F16)
            RDB_TRY(launch_chained(xent_join_kernel<__half>, blocks, NT, 0, s, w.part, parts,
                                   static_cast<const __half*>(q), ldq, static_cast<const __half*>(x), ldx, d, targets,
                                   ignore_index, n, c, nq, wide, stats, loss, reduction, loss, w.ticket));
        else
            RDB_TRY(launch_chained(xent_join_kernel<__nv_bfloat16>, blocks, NT, 0, s, w.part, parts,
                                   static_cast<const __nv_bfloat16*>(q), ldq, static_cast<const __nv_bfloat16*>(x),
                                   ldx, d, targets, ignore_index, n, c, nq, wide, stats, loss, reduction, loss,
                                   w.ticket));
    } else if (reduction != RDB_REDUCE_NONE) {
        RDB_TRY(launch_chained(xent_reduce_kernel, 1, NT, 0, s, targets, ignore_index, nq, reduction, stats, loss));
    }
    return RDB_OK;
}

size_t rdb_softmax_xent_backward_workspace(int dtype, int64_t nq, int64_t n, int d, int need_dq, int need_dx) {
    if (!plannable(dtype, nq, n, d)) return 0;
    const BwdPlan p = bwd_plan(dtype, nq, n, d, need_dq != 0, need_dx != 0);
    return bwd_ws(nullptr, p, dtype, nq, d, need_dq != 0, need_dx != 0).bytes;
}

int rdb_softmax_xent_backward(int dtype, const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n,
                              int64_t ldx, int d, const int64_t* targets, float scale, int64_t ignore_index,
                              int reduction, const float* grad, const float* stats, void* dq, int64_t lddq, void* dx,
                              int64_t lddx, void* ws, size_t ws_bytes, void* stream) {
    RDB_TRY(check_common(dtype, q, nq, ldq, x, n, ldx, d, targets, scale, reduction));
    RDB_CHECK_ARG((!dq || lddq >= d) && (!dx || lddx >= d), "bad shape");
    RDB_CHECK_ARG(nq == 0 || (grad && stats), "NULL pointer");
    RDB_CHECK_ARG((reinterpret_cast<uintptr_t>(ws) & 15) == 0, "ws must be 16-byte aligned");
    if (!ws || ws_bytes < rdb_softmax_xent_backward_workspace(dtype, nq, n, d, dq != nullptr, dx != nullptr))
        return set_error(RDB_ERR_WORKSPACE, "workspace too small");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (nq == 0) {
        if (dx)
            RDB_CUDA_TRY(cudaMemset2DAsync(dx, (size_t)lddx * elem_size(dtype), 0, (size_t)d * elem_size(dtype),
                                           (size_t)n, s));
        return RDB_OK;
    }
    if (!dq && !dx) return RDB_OK;
    if (dtype == RDB_F32)
        return backward_t<float>(dtype, q, nq, ldq, x, n, ldx, d, targets, scale, ignore_index, reduction, grad, stats,
                                 dq, lddq, dx, lddx, ws, s);
    if (dtype == RDB_F16)
        return backward_t<__half>(dtype, q, nq, ldq, x, n, ldx, d, targets, scale, ignore_index, reduction, grad,
                                  stats, dq, lddq, dx, lddx, ws, s);
    return backward_t<__nv_bfloat16>(dtype, q, nq, ldq, x, n, ldx, d, targets, scale, ignore_index, reduction, grad,
                                     stats, dq, lddq, dx, lddx, ws, s);
}

}  // extern "C"
