// Softmax cross entropy of queries against every stored row, with gradients.
//
//   s_bn   = scale <q_b, x_n>                  (never written to memory)
//   loss_b = log sum_n exp(s_bn) - s_b,t(b)    (0 where t(b) == ignore_index)
//   G_bn   = g_b scale (exp(s_bn) / sum_n exp(s_bn) - [n = t(b)])
//   dq = G x,  dx = G^T q
//
// The sum is taken in base 2 around a running maximum: with c = scale log2 e,
//   m = max_n c <q, x_n>,   z = sum_n 2^(c <q, x_n> - m),
// held in fp32; log sum exp = ln 2 (m + log2 z).  The target's own term stays out
// of the running sum: with r = the sum of the other terms relative to the
// target's, loss = log1p(r), so a query that finds its row keeps a loss near 0,
// and its p - 1 = expm1(-loss), to full precision.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace rdb {
namespace {

constexpr int NT = 256, NW = NT / 32;
constexpr float kLn2 = 0.6931471805599453f;
constexpr double kLog2e = 1.4426950408889634;

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

template <typename T>
__device__ __forceinline__ float warp_dot(const T* a, const T* b, int d, int lane) {
    float s = 0.f;
    for (int t = lane; t < d; t += 32) s = fmaf(to_f(a[t]), to_f(b[t]), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

// 2^(a - m) with an empty or all -inf running maximum standing for "no terms"
__device__ __forceinline__ float exp2_from(float a, float m) { return exp2f(a - (m == -INFINITY ? 0.f : m)); }

// (M, Z): running maximum and sum over the rows but the target, tv the target's
// value -> st = (largest value m, log2 sum 2^(s - m), loss) of the query.  An
// ignored query has loss 0; one whose target is not a row is NaN throughout.
__device__ __forceinline__ void finish_row(float M, float Z, float tv, bool has, bool ignored, float (&st)[3]) {
    const float m = fmaxf(M, tv), mr = m == -INFINITY ? 0.f : m;
    const float rest = Z * exp2_from(M, m);
    st[0] = m;
    st[1] = log2f(rest + exp2f(tv - mr));
    if (ignored) {
        st[2] = 0.f;
    } else if (!has) {
        st[1] = st[2] = __int_as_float(0x7fc00000);
    } else {
        st[2] = tv >= M ? log1pf(rest) : kLn2 * (st[1] + (m - tv));
    }
}

template <typename T>
__global__ void __launch_bounds__(NT) xent_forward_kernel(const T* q, int64_t ldq, const T* x, int64_t n, int64_t ldx,
                                                          int d, const int64_t* targets, float c, int64_t ignore,
                                                          float* loss, float* stats, int64_t nq) {
    __shared__ float sm[NW], sz[NW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t b = blockIdx.x;
    const int64_t t = targets[b];
    float m = -INFINITY, z = 0.f;
    for (int64_t r = warp; r < n; r += NW) {
        if (r == t) continue;
        const float a = c * warp_dot(q + b * ldq, x + r * ldx, d, lane);
        const float mn = fmaxf(m, a);
        z = z * exp2_from(m, mn) + exp2_from(a, mn);
        m = mn;
    }
    if (lane == 0) sm[warp] = m, sz[warp] = z;
    __syncthreads();
    if (warp == 0) {
        float M = -INFINITY, Z = 0.f;
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w]);
        for (int w = 0; w < NW; ++w) Z += sz[w] * exp2_from(sm[w], M);
        const bool has = t >= 0 && t < n;
        const float tv = has ? c * warp_dot(q + b * ldq, x + t * ldx, d, lane) : -INFINITY;
        float st[3];
        finish_row(M, Z, tv, has, t == ignore, st);
        if (lane == 0) loss[b] = st[2], stats[b] = st[0], stats[nq + b] = st[1], stats[2 * nq + b] = st[2];
    }
}

// sum and count of the valid rows -> the reduced loss
__global__ void xent_reduce_kernel(const float* loss_q, const int64_t* targets, int64_t ignore, int64_t nq, int mean,
                                   float* loss) {
    __shared__ float ss[NW];
    __shared__ long long sc[NW];
    float s = 0.f;
    long long cnt = 0;
    for (int64_t i = threadIdx.x; i < nq; i += NT) {
        const bool ok = targets[i] != ignore;
        s += ok ? loss_q[i] : 0.f;
        cnt += ok;
    }
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
    if ((threadIdx.x & 31) == 0) ss[threadIdx.x >> 5] = s, sc[threadIdx.x >> 5] = cnt;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < NW; ++w) ss[0] += ss[w], sc[0] += sc[w];
        *loss = mean ? ss[0] / static_cast<float>(sc[0]) : ss[0];
    }
}

// g_b of every query: the incoming gradient (divided by the valid queries for
// the mean), 0 for an ignored one
__global__ void __launch_bounds__(NT) xent_weights_kernel(const float* grad, const int64_t* targets, int64_t ignore,
                                                          int64_t nq, int reduction, float* w) {
    __shared__ long long sc[NW];
    long long cnt = 0;
    if (reduction == RDB_REDUCE_MEAN) {
        for (int64_t i = threadIdx.x; i < nq; i += NT) cnt += targets[i] != ignore;
        for (int o = 16; o > 0; o >>= 1) cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
        if ((threadIdx.x & 31) == 0) sc[threadIdx.x >> 5] = cnt;
        __syncthreads();
        cnt = 0;
        for (int k = 0; k < NW; ++k) cnt += sc[k];
    }
    for (int64_t i = threadIdx.x; i < nq; i += NT) {
        float g = grad[reduction == RDB_REDUCE_NONE ? i : 0];
        if (reduction == RDB_REDUCE_MEAN) g /= static_cast<float>(cnt);
        w[i] = targets[i] == ignore ? 0.f : g;
    }
}

template <typename T>
__device__ __forceinline__ float grad_logit(const T* q, const T* x, int d, float c, float m, float lz, float loss,
                                            bool hit, int lane) {
    const float a = c * warp_dot(q, x, d, lane);
    return hit ? expm1f(-loss) : exp2f(a - m - lz);
}

// one block per query (DX = false: dq) or per row (DX = true: dx); acc is the
// block's [d] fp32 row of the workspace
template <typename T, bool DX>
__global__ void __launch_bounds__(NT)
    xent_backward_kernel(const T* q, int64_t nq, int64_t ldq, const T* x, int64_t n, int64_t ldx, int d,
                         const int64_t* targets, float scale, float c, int64_t ignore, const float* weight,
                         const float* stats, T* out, int64_t ldo, float* acc_ws) {
    __shared__ float w[NW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t count = DX ? nq : n;
    float* acc = acc_ws + (int64_t)blockIdx.x * d;
    for (int64_t self = blockIdx.x; self < (DX ? n : nq); self += gridDim.x) {
        for (int t = threadIdx.x; t < d; t += NT) acc[t] = 0.f;
        for (int64_t o0 = 0; o0 < count; o0 += NW) {
            const int64_t o = o0 + warp;
            const int64_t b = DX ? o : self, r = DX ? self : o;
            float v = 0.f;
            if (o < count && targets[b] != ignore)
                v = scale * weight[b] *
                    grad_logit(q + b * ldq, x + r * ldx, d, c, stats[b], stats[nq + b], stats[2 * nq + b],
                                targets[b] == r, lane);
            if (lane == 0) w[warp] = v;
            __syncthreads();
            for (int k = 0; k < NW && o0 + k < count; ++k) {
                if (targets[DX ? o0 + k : self] == ignore) continue;  // whatever an ignored query holds
                const T* row = DX ? q + (o0 + k) * ldq : x + (o0 + k) * ldx;
                for (int t = threadIdx.x; t < d; t += NT) acc[t] = fmaf(w[k], to_f(row[t]), acc[t]);
            }
            __syncthreads();
        }
        for (int t = threadIdx.x; t < d; t += NT) out[self * ldo + t] = from_f<T>(acc[t]);
    }
}

int check_common(int dtype, const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n, int64_t ldx, int d,
                 const int64_t* targets, float scale, int reduction) {
    const int64_t e = (int64_t)elem_size(dtype);
    RDB_CHECK_ARG(e != 0, "unknown dtype %d", dtype);
    RDB_CHECK_ARG(nq >= 0 && n >= 1 && d >= 1 && ldq >= d && ldx >= d, "bad shape");
    RDB_CHECK_ARG(nq < (1LL << 31) && n < (1LL << 31), "nq and n must be < 2^31");
    RDB_CHECK_ARG(scale > 0.f && scale <= 3.0e38f, "scale must be positive and finite");
    RDB_CHECK_ARG(reduction >= RDB_REDUCE_NONE && reduction <= RDB_REDUCE_SUM, "unknown reduction %d", reduction);
    RDB_CHECK_ARG(x && (nq == 0 || (q && targets)), "NULL pointer");
    RDB_CHECK_ARG((ldq * e) % 16 == 0 && (ldx * e) % 16 == 0, "row strides must be multiples of 16 bytes");
    RDB_CHECK_ARG((reinterpret_cast<uintptr_t>(q) & 15) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0,
                  "base pointers must be 16-byte aligned");
    return RDB_OK;
}

template <typename T>
int forward_t(const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n, int64_t ldx, int d,
              const int64_t* targets, float scale, int64_t ignore, float* loss_q, float* stats, cudaStream_t s) {
    xent_forward_kernel<T><<<(unsigned)nq, NT, 0, s>>>(static_cast<const T*>(q), ldq, static_cast<const T*>(x), n, ldx,
                                                       d, targets, (float)(scale * kLog2e), ignore, loss_q, stats, nq);
    RDB_LAUNCH_CHECK();
    return RDB_OK;
}

constexpr int64_t kBlocks = 1024;

template <typename T>
int backward_t(const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n, int64_t ldx, int d,
               const int64_t* targets, float scale, int64_t ignore, int reduction, const float* grad,
               const float* stats, void* dq, int64_t lddq, void* dx, int64_t lddx, float* ws, cudaStream_t s) {
    const T *tq = static_cast<const T*>(q), *tx = static_cast<const T*>(x);
    const float c = (float)(scale * kLog2e);
    float *weight = ws, *acc = ws + (nq + 63) / 64 * 64;
    xent_weights_kernel<<<1, NT, 0, s>>>(grad, targets, ignore, nq, reduction, weight);
    RDB_LAUNCH_CHECK();
    if (dq) {
        xent_backward_kernel<T, false><<<(unsigned)(nq < kBlocks ? nq : kBlocks), NT, 0, s>>>(
            tq, nq, ldq, tx, n, ldx, d, targets, scale, c, ignore, weight, stats, static_cast<T*>(dq), lddq, acc);
        RDB_LAUNCH_CHECK();
    }
    if (dx) {
        xent_backward_kernel<T, true><<<(unsigned)(n < kBlocks ? n : kBlocks), NT, 0, s>>>(
            tq, nq, ldq, tx, n, ldx, d, targets, scale, c, ignore, weight, stats, static_cast<T*>(dx), lddx, acc);
        RDB_LAUNCH_CHECK();
    }
    return RDB_OK;
}

}  // namespace
}  // namespace rdb

using namespace rdb;

extern "C" {

size_t rdb_softmax_xent_workspace(int dtype, int64_t nq, int64_t n, int d, int reduction) {
    (void)dtype, (void)n, (void)d, (void)reduction;
    return 4 * (size_t)(nq > 0 ? nq : 0) + 256;
}

int rdb_softmax_xent(int dtype, const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n, int64_t ldx, int d,
                     const int64_t* targets, float scale, int64_t ignore_index, int reduction, float* loss,
                     float* stats, void* ws, size_t ws_bytes, void* stream) {
    RDB_TRY(check_common(dtype, q, nq, ldq, x, n, ldx, d, targets, scale, reduction));
    RDB_CHECK_ARG((loss || (nq == 0 && reduction == RDB_REDUCE_NONE)) && (nq == 0 || stats), "NULL pointer");
    if (!ws || ws_bytes < rdb_softmax_xent_workspace(dtype, nq, n, d, reduction))
        return set_error(RDB_ERR_WORKSPACE, "workspace too small");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    float* loss_q = reduction == RDB_REDUCE_NONE ? loss : static_cast<float*>(ws);
    if (nq > 0) {
        if (dtype == RDB_F32)
            RDB_TRY(forward_t<float>(q, nq, ldq, x, n, ldx, d, targets, scale, ignore_index, loss_q, stats, s));
        else if (dtype == RDB_F16)
            RDB_TRY(forward_t<__half>(q, nq, ldq, x, n, ldx, d, targets, scale, ignore_index, loss_q, stats, s));
        else
            RDB_TRY(forward_t<__nv_bfloat16>(q, nq, ldq, x, n, ldx, d, targets, scale, ignore_index, loss_q, stats, s));
    }
    if (reduction != RDB_REDUCE_NONE) {
        xent_reduce_kernel<<<1, NT, 0, s>>>(loss_q, targets, ignore_index, nq, reduction == RDB_REDUCE_MEAN, loss);
        RDB_LAUNCH_CHECK();
    }
    return RDB_OK;
}

size_t rdb_softmax_xent_backward_workspace(int dtype, int64_t nq, int64_t n, int d, int need_dq, int need_dx) {
    (void)dtype, (void)n, (void)need_dq, (void)need_dx;
    return 4 * ((size_t)(nq > 0 ? nq : 0) + (size_t)kBlocks * (size_t)(d > 0 ? d : 0)) + 512;
}

int rdb_softmax_xent_backward(int dtype, const void* q, int64_t nq, int64_t ldq, const void* x, int64_t n,
                              int64_t ldx, int d, const int64_t* targets, float scale, int64_t ignore_index,
                              int reduction, const float* grad, const float* stats, void* dq, int64_t lddq, void* dx,
                              int64_t lddx, void* ws, size_t ws_bytes, void* stream) {
    RDB_TRY(check_common(dtype, q, nq, ldq, x, n, ldx, d, targets, scale, reduction));
    RDB_CHECK_ARG((!dq || lddq >= d) && (!dx || lddx >= d), "bad shape");
    RDB_CHECK_ARG(nq == 0 || (grad && stats), "NULL pointer");
    if (!ws || ws_bytes < rdb_softmax_xent_backward_workspace(dtype, nq, n, d, dq != nullptr, dx != nullptr))
        return set_error(RDB_ERR_WORKSPACE, "workspace too small");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (nq == 0) {
        if (dx)
            RDB_CUDA_TRY(cudaMemset2DAsync(dx, (size_t)lddx * elem_size(dtype), 0, (size_t)d * elem_size(dtype),
                                           (size_t)n, s));
        return RDB_OK;
    }
    float* w = static_cast<float*>(ws);
    if (dtype == RDB_F32)
        return backward_t<float>(q, nq, ldq, x, n, ldx, d, targets, scale, ignore_index, reduction, grad, stats, dq,
                                 lddq, dx, lddx, w, s);
    if (dtype == RDB_F16)
        return backward_t<__half>(q, nq, ldq, x, n, ldx, d, targets, scale, ignore_index, reduction, grad, stats, dq,
                                  lddq, dx, lddx, w, s);
    return backward_t<__nv_bfloat16>(q, nq, ldq, x, n, ldx, d, targets, scale, ignore_index, reduction, grad, stats,
                                     dq, lddq, dx, lddx, w, s);
}

}  // extern "C"
