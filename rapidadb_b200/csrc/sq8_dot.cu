// Scores of int8 codes: out[b, n] = qs[b] * xs[n] * sum_t qc[b, t] * xc[n, t].
//
// Both operands are SQ8 rows (sq8.cu): int8 codes and one fp32 scale per row,
// so the scales are per query (token) and per database row (channel).  The
// sum is an exact int32 (|code| <= 128 and d <= kMaxDim, so it stays below
// 2^31); one fp32 product of the two scales and one with the sum follow, and
// fp16 / bf16 outputs are rounded once from that fp32 value.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

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

// one warp per (query, row)
template <typename T>
__global__ void sq8_dot_kernel(const int8_t* __restrict__ qc, const float* __restrict__ qs, int64_t nq, int64_t ldq,
                               const int8_t* __restrict__ xc, const float* __restrict__ xs, int64_t n, int64_t ldx,
                               int d, T* __restrict__ out, int64_t ldo) {
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t b = w / n, r = w % n;
    if (b >= nq) return;
    const int8_t *q = qc + b * ldq, *x = xc + r * ldx;
    int acc = 0;
    const int d4 = d & ~3;
    for (int t = 4 * lane; t < d4; t += 128)
        acc = __dp4a(*reinterpret_cast<const int*>(q + t), *reinterpret_cast<const int*>(x + t), acc);
    if (lane < (d & 3)) acc += static_cast<int>(q[d4 + lane]) * static_cast<int>(x[d4 + lane]);
    acc = __reduce_add_sync(0xffffffffu, acc);
    if (lane == 0) out[b * ldo + r] = from_f<T>(__fmul_rn(__fmul_rn(qs[b], xs[r]), static_cast<float>(acc)));
}

template <typename T>
int launch_dot(const int8_t* qc, const float* qs, int64_t nq, int64_t ldq, const int8_t* xc, const float* xs,
               int64_t n, int64_t ldx, int d, void* out, int64_t ldo, cudaStream_t s) {
    const int64_t blocks = (nq * n + 7) / 8;
    RDB_CHECK_ARG(blocks < (1LL << 31), "too many scores for one launch");
    sq8_dot_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(qc, qs, nq, ldq, xc, xs, n, ldx, d, static_cast<T*>(out), ldo);
    RDB_LAUNCH_CHECK();
    return RDB_OK;
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
