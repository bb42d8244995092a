// Launches whose start overlaps the end of what runs before them in the stream
// (programmatic dependent launch): such a kernel is placed and set up (barriers,
// tensor memory) while its predecessor drains, and waits before it touches global
// memory.  Captured, in a row: a training step of 256 x 256 x 768 bf16 32.3 us
// instead of 35.0, 77 x 5,003 x 100 fp16 37.6 instead of 40.1, 64 x 4,096 x 256 fp32
// 56.2 instead of 57.5, the loss of one query over 100,000 x 768 bf16 29.7 instead
// of 30.9 (from a cold L2 43.8 instead of 47); the int8 scores of one query and
// 100,000 rows are as fast without (8.7 and 8.4; cold 24.6 both).
//
// Every thread of a kernel launched this way calls chain_wait() before any access
// to global memory: a kernel then finishes only after all before it, and what
// follows it in the stream, launched in whichever way, sees all of them finished.
// Its inputs are loaded by ordinary loads: the kernel is resident while they are
// still being written, so the read-only path (__ldg, const __restrict__
// parameters), which takes them as constant for its whole life and is not held
// back by the wait, is closed to it.
#pragma once

#include <utility>

#include "common.cuh"

namespace rdb {
namespace {

// What is before has finished and is visible; the next kernel may be placed.  (In
// the other order a chain of short kernels is placed at once, each holding its
// threads while it waits for all before it: the steps above take 33.5, 38.9 and
// 62.5 us.)
__device__ __forceinline__ void chain_wait() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <class... K, class... A>
int launch_chained(void (*kernel)(K...), unsigned blocks, unsigned threads, size_t smem, cudaStream_t s, A&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    RDB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...));
    note_launch();
    return RDB_OK;
}

}  // namespace
}  // namespace rdb
