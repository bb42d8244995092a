// Copy of matrix rows to a 16-byte row stride, zero behind the last column: the
// layout TMA and 16-byte loads need, for operands that do not have it.
#include <algorithm>

#include "chain.cuh"
#include "common.cuh"

namespace rdb {
namespace {

// one thread per 16-byte unit of the copy, reading W bytes at a time
template <typename W>
__global__ void __launch_bounds__(256)
    pad_rows_kernel(const uint8_t* src, int64_t rows, int64_t row_bytes, int64_t src_stride,
                    uint4* dst, int64_t units) {
    chain_wait();
    const int64_t total = rows * units;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = i / units, t = (i - r * units) * 16;
        union {
            uint4 v;
            W w[16 / sizeof(W)];
        } u;
        u.v = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int k = 0; k < (int)(16 / sizeof(W)); ++k)
            if (t + (int)sizeof(W) * (k + 1) <= row_bytes)
                u.w[k] = *reinterpret_cast<const W*>(src + r * src_stride + t + sizeof(W) * k);
        dst[i] = u.v;
    }
}

}  // namespace
}  // namespace rdb

using namespace rdb;

extern "C" int rdb_pad_rows(const void* src, int64_t rows, int64_t row_bytes, int64_t src_stride, void* dst,
                            int64_t dst_stride, void* stream) {
    RDB_CHECK_ARG(rows >= 0 && row_bytes >= 1 && src_stride >= 0, "bad shape");
    RDB_CHECK_ARG(dst_stride >= row_bytes && dst_stride % 16 == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0,
                  "the copy's base and stride must be multiples of 16 bytes");
    if (rows == 0) return RDB_OK;
    RDB_CHECK_ARG(src && dst, "NULL pointer");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t units = dst_stride / 16;
    const unsigned blocks = (unsigned)std::min<int64_t>((rows * units + 255) / 256, 16LL * num_sms());
    const uint8_t* p = static_cast<const uint8_t*>(src);
    uint4* o = static_cast<uint4*>(dst);
    // the widest access that base, stride and row length allow
    const uint64_t align = reinterpret_cast<uintptr_t>(src) | (uint64_t)src_stride | (uint64_t)row_bytes;
    const auto kernel = align % 8 == 0   ? pad_rows_kernel<uint2>
                        : align % 4 == 0 ? pad_rows_kernel<uint32_t>
                        : align % 2 == 0 ? pad_rows_kernel<uint16_t>
                                         : pad_rows_kernel<uint8_t>;
    return launch_chained(kernel, blocks, 256, 0, s, p, rows, row_bytes, src_stride, o, units);
}
