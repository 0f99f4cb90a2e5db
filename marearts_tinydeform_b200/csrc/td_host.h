// td_host.h -- host-side services that the library's translation units share: error reports, device facts, the launch
// counter, the kernel policy and tensor maps. They live in tinydeform.cu (hidden symbols of the one shared object).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>

#include "../../include/tinydeform.h"

namespace td {

constexpr int kSms = 148;  // B200's, for plans that workspace sizes follow from

namespace host {

// Writes the printf-style message into err[0 .. err_len) and returns code.
int fail(char* err, size_t err_len, int code, const char* fmt, ...);
// Whether the kernel policy is TD_POLICY_BEST.
bool best_policy();
void count_launch();
// cuTensorMapEncodeTiled of 16-bit elements (no interleave, 256-byte L2 promotion, zero fill outside).
CUresult encode_tiled_u16(CUtensorMap* map, uint32_t rank, const void* base, const uint64_t* dims,
                          const uint64_t* strides, const uint32_t* box, CUtensorMapSwizzle swizzle);
// The same of a 2-D tensor of bytes.
CUresult encode_tiled_u8(CUtensorMap* map, const void* base, uint64_t cols, uint64_t rows, uint64_t pitch,
                         uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle);
// Of a dense [layers, rows, cols] tensor of 1, 2 or 4-byte elements, boxes within a layer.
CUresult encode_tiled_rows(CUtensorMap* map, int element, const void* base, uint64_t cols, uint64_t rows,
                           uint64_t layers, uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle);

// Launches `kernel` with an optional programmatic dependent launch (see launch_kernel in tinydeform.cu), counts it
// and reports a launch error.
template <typename K, typename... Args>
int launch(char* err, size_t err_len, const char* what, K kernel, dim3 grid, dim3 block, size_t smem,
           cudaStream_t stream, bool pdl, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(err, err_len, TD_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    }
    count_launch();
    return TD_OK;
}

// Raises a kernel's dynamic shared memory limit where it needs more than the 48 KB every kernel has: the attribute is
// the device's, so once per kernel and device (a host-side write, legal during capture; two threads may both do it).
template <auto Kernel>
int allow_smem(size_t bytes, char* err, size_t err_len) {
    static std::atomic<uint64_t> done{0};
    if (bytes <= 48 * 1024) return TD_OK;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1) != 0) return TD_OK;
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(err, err_len, TD_ERR_CUDA, "shared memory limit of %zu bytes: %s", bytes, cudaGetErrorString(e));
    }
    if (dev < 64) done.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    return TD_OK;
}

}  // namespace host

// The device error word of td_attention_tc.cu (a translation unit has its own copy of the word td_ptx.cuh declares;
// td_fp8.cu has another; the kernels of the rest wait for nothing).
cudaError_t attention_tc_device_error(int clear, unsigned int* code);
// That of td_fp8.cu.
cudaError_t fp8_device_error(int clear, unsigned int* code);

}  // namespace td
