// INT8 storage: per-row symmetric scalar quantisation (SQ8).
//
// The reference lists INT8 among its storage precisions
// (csrc/include/rapidadb/core/types.h:9-14, python/rapidadb/config.py:21-26,
// README.md:13) without defining it.  Here a row x is stored as
//   scale = max_i |x_i| / 127                (fp32 division; 0 for a zero row)
//   code_i = rint(x_i / scale), clamped to [-127, 127]   (ties to even; 0 if scale == 0)
// and stands for the dequantised row  x^_i = fl(scale * code_i).  Searches over
// SQ8 rows are exact searches over x^ with fp32 queries (the reference
// formulas), one byte per element in HBM instead of four.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "chain.cuh"
#include "common.cuh"

namespace rdb {
namespace {

__device__ __forceinline__ float ld_any(int dtype, const void* p, int64_t i) {
    if (dtype == RDB_F32) return static_cast<const float*>(p)[i];
    if (dtype == RDB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}

// one warp per row, any layout
__global__ void sq8_encode_kernel(int dtype, const void* x, int64_t n, int64_t ldx, int d, int8_t* codes, int64_t ldc,
                                  float* scales) {
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= n) return;
    float amax = 0.f;
    for (int t = lane; t < d; t += 32) amax = fmaxf(amax, fabsf(ld_any(dtype, x, row * ldx + t)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float scale = __fdiv_rn(amax, 127.f);
    for (int t = lane; t < (int)ldc; t += 32) {
        int c = 0;
        if (t < d && scale > 0.f) {
            const float v = rintf(__fdiv_rn(ld_any(dtype, x, row * ldx + t), scale));
            c = (int)fminf(fmaxf(v, -127.f), 127.f);
        }
        codes[row * ldc + t] = static_cast<int8_t>(c);
    }
    if (lane == 0) scales[row] = scale;
}

// Codes without divisions or conversions.  kRound = 1.5 * 2^23: adding it rounds
// to the nearest integer (ties to even) and leaves that integer, modulo 256, in
// the sum's low byte.  t = x * (1 / scale) + kRound (one rounding) gives
// rint(x / scale) unless x / scale lies next to a half: 1 / scale is off by
// 2^-24 of itself and the quotient by its own rounding, at most 127 * 2^-23 <
// 2^-16 together, so wherever the distance to the integer is below 1/2 - 2^-14
// the two agree.  The others (one in 10^4), NaN, and whole rows with a subnormal
// or infinite scale go through the division and the clamp.
constexpr float kRound = 12582912.f, kNearHalf = 0.5f - 6.103515625e-05f;

__device__ __forceinline__ uint32_t slow_code(float x, float scale) {
    const float c = scale > 0.f ? rintf(__fdiv_rn(x, scale)) : 0.f;
    return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(c, -127.f), 127.f)));
}

// four codes in one word
__device__ __forceinline__ uint32_t codes4(const float* x, float scale, float inv, bool fast) {
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float s = fmaf(x[i], inv, kRound);
        fast &= fabsf(fmaf(x[i], inv, kRound - s)) < kNearHalf;
        t[i] = __float_as_uint(s);
    }
    if (!fast) {
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = slow_code(x[i], scale);
    }
    return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}

template <typename T>
__device__ __forceinline__ void load16(const void* p, float (&v)[16 / sizeof(T)]) {
    const uint4 u = *static_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        } else {
            v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}

// The same codes from rows of 16-byte units (d * size a multiple of 16 bytes,
// bases and strides aligned): one warp per row, which it reads once, U units a
// lane held in registers.  The bytes of the row and of its codes bound it: 1M x
// 768 bf16 in 400 us, 5.8 TB/s (508 us with a division and two conversions each).
template <typename T, int U>
__global__ void __launch_bounds__(256)
    sq8_encode_rows_kernel(const T* x, int64_t n, int64_t ldx, int units, int8_t* codes, int64_t ldc, float* scales) {
    constexpr int E = 16 / sizeof(T);  // elements of a unit
    chain_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= n) return;
    float v[U][E];
    float amax = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u * 32 + lane < units) load16<T>(x + row * ldx + (u * 32 + lane) * E, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u * 32 + lane < units)
#pragma unroll
            for (int i = 0; i < E; ++i) amax = fmaxf(amax, fabsf(v[u][i]));
    // amax >= 0: its bits order like integers
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    const float scale = __fdiv_rn(amax, 127.f), inv = __fdiv_rn(1.f, scale);
    const bool fast = scale >= 1.17549435e-38f && scale < INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (u * 32 + lane >= units) continue;
        int8_t* o = codes + row * ldc + (u * 32 + lane) * E;
        if constexpr (E == 8)
            *reinterpret_cast<uint2*>(o) =
                make_uint2(codes4(v[u], scale, inv, fast), codes4(v[u] + 4, scale, inv, fast));
        else
            *reinterpret_cast<uint32_t*>(o) = codes4(v[u], scale, inv, fast);
    }
    // columns behind d are zero
    for (int64_t t = (int64_t)units * E + lane; t < ldc; t += 32) codes[row * ldc + t] = 0;
    if (lane == 0) scales[row] = scale;
}

// rows that the kernel above takes
bool whole_units(int elem, const void* x, int64_t ldx, int d, const int8_t* codes, int64_t ldc) {
    const int e = 16 / elem;
    return d % e == 0 && ldx % e == 0 && ldc % e == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 &&
           (reinterpret_cast<uintptr_t>(codes) & (e - 1)) == 0 && d / e <= 256;
}

template <typename T>
int encode_rows(const void* x, int64_t n, int64_t ldx, int d, int8_t* codes, int64_t ldc, float* scales,
                cudaStream_t s) {
    const int units = d / (16 / (int)sizeof(T));
    const auto kernel = units <= 32    ? sq8_encode_rows_kernel<T, 1>
                        : units <= 64  ? sq8_encode_rows_kernel<T, 2>
                        : units <= 96  ? sq8_encode_rows_kernel<T, 3>
                        : units <= 128 ? sq8_encode_rows_kernel<T, 4>
                        : units <= 192 ? sq8_encode_rows_kernel<T, 6>
                                       : sq8_encode_rows_kernel<T, 8>;
    return launch_chained(kernel, (unsigned)((n + 7) / 8), 256, 0, s, static_cast<const T*>(x), n, ldx, units, codes, ldc,
                          scales);
}

// per-row metric value of the dequantised row: |x^|^2 (L2), |x^| or
// sqrt(|x^|^2 + 1e-8) (cosine), 0 (dot)
__global__ void sq8_values_kernel(int metric, int cos_small, const int8_t* codes, const float* scales, int64_t n,
                                  int64_t ldc, int d, float* out) {
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= n) return;
    const float s = scales[row];
    float acc = 0.f;
    for (int t = lane; t < d; t += 32) {
        const float v = __fmul_rn(s, static_cast<float>(codes[row * ldc + t]));
        acc = fmaf(v, v, acc);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) out[row] = vec_value(metric, cos_small, acc);
}

}  // namespace
}  // namespace rdb

using namespace rdb;

extern "C" {

int rdb_sq8_encode(int dtype, const void* x, int64_t n, int64_t ldx, int d, int8_t* codes, int64_t ldc, float* scales,
                   void* stream) {
    RDB_CHECK_ARG(elem_size(dtype) != 0, "unknown dtype %d", dtype);
    RDB_CHECK_ARG(n >= 0 && d >= 1 && ldx >= d && ldc >= d, "bad shape");
    if (n == 0) return RDB_OK;
    RDB_CHECK_ARG(x && codes && scales, "NULL pointer");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (whole_units((int)elem_size(dtype), x, ldx, d, codes, ldc)) {
        if (dtype == RDB_F32) return encode_rows<float>(x, n, ldx, d, codes, ldc, scales, s);
        if (dtype == RDB_F16) return encode_rows<__half>(x, n, ldx, d, codes, ldc, scales, s);
        return encode_rows<__nv_bfloat16>(x, n, ldx, d, codes, ldc, scales, s);
    }
    sq8_encode_kernel<<<(unsigned)((n + 7) / 8), 256, 0, s>>>(dtype, x, n, ldx, d, codes, ldc, scales);
    RDB_LAUNCH_CHECK();
    return RDB_OK;
}

int rdb_sq8_row_values(int metric, const int8_t* codes, const float* scales, int64_t n, int64_t ldc, int d,
                       float* out, void* stream) {
    RDB_CHECK_ARG(metric >= 0 && metric <= 2, "unknown metric %d", metric);
    RDB_CHECK_ARG(n >= 0 && d >= 1 && ldc >= d, "bad shape");
    if (n == 0) return RDB_OK;
    RDB_CHECK_ARG(codes && scales && out, "NULL pointer");
    const unsigned blocks = (unsigned)((n + 7) / 8);
    sq8_values_kernel<<<blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(metric, d <= 128 ? 1 : 0, codes, scales,
                                                                             n, ldc, d, out);
    RDB_LAUNCH_CHECK();
    return RDB_OK;
}

}  // extern "C"
