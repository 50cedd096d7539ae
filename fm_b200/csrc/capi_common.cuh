// What the C ABI's translation units for the state-space operators share: status of runtime calls, checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>

#include "fm_scan_b200.h"

#define FMS_EXPORT extern "C" __attribute__((visibility("default")))

namespace fms {
int record_cuda_error(cudaError_t e);  // fm_scan_capi.cu: this thread's fms_last_cuda_error
}

namespace {  // internal to each translation unit

constexpr int64_t kMaxGrid = 0x7fffffff;
constexpr size_t kMaxSmem = 227 * 1024;  // of a CTA on sm_100

inline int check_launch() { return fms::record_cuda_error(cudaGetLastError()); }
inline bool dtype_ok(int d) { return d == FMS_F32 || d == FMS_F16 || d == FMS_BF16; }
inline int64_t elem_size(int d) { return d == FMS_F32 ? 4 : 2; }
inline bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// a * b * c * ... with every product below 2^59, so that byte offsets fit int64
bool product_ok(std::initializer_list<int64_t> v) {
    int64_t p = 1;
    for (int64_t k : v) {
        if (k < 0) return false;
        if (k && p > (int64_t{1} << 59) / k) return false;
        p *= k ? k : 1;
    }
    return true;
}

// every row of a tensor with these element strides starts on a 16-byte boundary
bool rows16(const void *p, const int64_t *stride, int n, int64_t es) {
    if (!aligned_to(p, 16)) return false;
    for (int i = 0; i < n; ++i)
        if (stride[i] * es % 16) return false;
    return true;
}

__global__ void fill_kernel(const float *__restrict__ src, float *__restrict__ dst, int64_t n) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i < n) dst[i] = src ? src[i] : 0.f;
}
int copy_or_zero(const float *src, float *dst, int64_t n, cudaStream_t st) {
    if (!dst || n == 0) return FMS_OK;
    if ((n + 255) / 256 > kMaxGrid) return FMS_ERR_TOO_LARGE;
    fill_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, st>>>(src, dst, n);
    return check_launch();
}

}  // namespace

#define FMS_BY_TYPE(dtype, CALL)                                         \
    switch (dtype) {                                                     \
        case FMS_F32: { using S = float; return CALL; }                  \
        case FMS_F16: { using S = __half; return CALL; }                 \
        default: { using S = __nv_bfloat16; return CALL; }               \
    }
