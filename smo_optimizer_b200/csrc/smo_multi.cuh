// smo_multi.cuh -- many tensors in one launch, for the elementwise kernels.
//
// The descriptors travel as a kernel parameter (no copy to the device, nothing
// to keep alive, and a captured graph holds its own).  Work is cut into chunks
// of a fixed number of elements, numbered through all tensors of the launch.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "smo_b200.h"
#include "smo_common.cuh"
#include "smo_internal.cuh"

namespace smo {

// 32,764 bytes is the most that one launch's parameters may hold
constexpr size_t kMaxParamBytes = 32764;

// Launch of a kernel whose one parameter is the batch, as a programmatic
// dependent launch: its CTAs may start while the kernel in front of it in the
// stream ends (2 us less between two kernels).  So every kernel launched this way
// calls wait_for_previous() before it touches memory that anything in front of it
// may touch.
template <class B>
cudaError_t launch_batch(void (*kernel)(B), unsigned ctas, unsigned threads, const B &b, cudaStream_t s) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, b);
}

// every kernel before this one in the stream has ended and its writes are visible
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// The next kernel may start as soon as every CTA has come here (or ended).  Only
// where that is a kernel of this library that knows what it may read before it
// waits, and only once everything in front has ended: after wait_for_previous(),
// or in a kernel that could itself start early for that reason.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// index of the tensor that holds chunk `c`: the last i with start[i] <= c
__device__ __forceinline__ int tensor_of(const int32_t *start, int n, int32_t c) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= c) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Eight consecutive elements as fp32, and back.  `p` must be 16-byte aligned.
template <class T>
__device__ __forceinline__ void ld8(const T *p, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        const T *e = reinterpret_cast<const T *>(&a);
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = ld<T>(e + k);
    }
}

template <class T>
__device__ __forceinline__ void st8(T *p, const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint4 a;
        T *e = reinterpret_cast<T *>(&a);
#pragma unroll
        for (int k = 0; k < 8; k++) st<T>(e + k, x[k]);
        *reinterpret_cast<uint4 *>(p) = a;
    }
}

// the status of a CUDA call; an error is taken from the runtime, so that it is not
// blamed on a later call
inline int cuda_status(cudaError_t e) {
    if (e == cudaSuccess) return SMO_OK;
    g_last_cuda_error = (int)e;
    (void)cudaGetLastError();
    return SMO_ERR_CUDA;
}

// chunks of n >= 0 elements
inline int64_t chunks_of(int64_t n, int64_t chunk) { return n / chunk + (n % chunk != 0); }
inline bool is_aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }
inline size_t dtype_bytes(int32_t dtype) { return dtype == SMO_DTYPE_F32 ? 4 : 2; }
inline bool known_dtype(int32_t dtype) {
    return dtype == SMO_DTYPE_F32 || dtype == SMO_DTYPE_BF16 || dtype == SMO_DTYPE_F16;
}

// smo_gradnorm.cu: the norm of n gradients (grad_of(items, i) is the i-th) into
// norm_out (may be null), and the factor min(1, max_norm / (norm + 1e-6)), times
// *scale where given, into *coef_out (a device float in the workspace; written
// only with max_norm > 0).
using GradOf = smo_grad (*)(const void *items, int32_t i);
size_t grad_norm_workspace(int32_t n);
int grad_norm_enqueue(GradOf grad_of, const void *items, int32_t n, const float *scale, float max_norm,
                      float *norm_out, void *workspace, float **coef_out, cudaStream_t stream);

}  // namespace smo
