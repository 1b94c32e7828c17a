// smo_gradnorm.cu -- the 2-norm over many gradient tensors, and clipping by it.
//
// Each gradient is read once; squares and sums are held in double, so that the
// norm is right to the last fp32 bit whatever the order of the additions (a
// clipped step's 8-bit codes depend on every bit of the factor), and squares of
// large elements do not overflow.  A CTA adds up every gridDim-th chunk and
// writes one partial sum; a last CTA adds the partial sums in their order.  The
// order goes by the sizes alone: no atomics, the same bits every time.
#include <climits>
#include <cstring>

#include "smo_multi.cuh"

namespace smo {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = kThreads * 8 * 4;  // elements of a chunk
constexpr int kCap = 1024;                // tensors of one launch
constexpr int kParts = 148 * 8;           // CTAs of one launch at most: one partial sum each

struct GradDesc {
    void *g;
    int64_t n;
};

struct GradBatch {
    int32_t n;
    double *part;
    const float *coef;
    int32_t start[kCap + 1];
    GradDesc d[kCap];
};
static_assert(sizeof(GradBatch) <= kMaxParamBytes, "launch parameters");

// sum over the CTA, in thread 0
__device__ __forceinline__ double cta_sum(double x) {
    __shared__ double warp[kThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_down_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) == 0) warp[threadIdx.x >> 5] = x;
    __syncthreads();
    x = threadIdx.x < kThreads / 32 ? warp[threadIdx.x] : 0.0;
    if (threadIdx.x < 32)
#pragma unroll
        for (int o = kThreads / 64; o > 0; o >>= 1) x += __shfl_down_sync(0xffffffffu, x, o);
    return x;
}

template <class T>
__global__ void __launch_bounds__(kThreads) sumsq_kernel(const __grid_constant__ GradBatch b) {
    const int32_t total = b.start[b.n];
    double acc = 0.0;
    int t = tensor_of(b.start, b.n, blockIdx.x);
    for (int32_t c = blockIdx.x; c < total; c += gridDim.x) {
        while (b.start[t + 1] <= c) t++;
        const GradDesc &d = b.d[t];
        const T *g = (const T *)d.g;
        const int64_t base = (int64_t)(c - b.start[t]) * kChunk;
        const int64_t end = base + kChunk < d.n ? base + kChunk : d.n;
        if (((uintptr_t)g & 15) == 0 && base + kChunk <= d.n) {
#pragma unroll
            for (int u = 0; u < 4; u++) {
                float x[8];
                ld8<T>(g + base + (u * kThreads + threadIdx.x) * 8, x);
#pragma unroll
                for (int k = 0; k < 8; k++) acc = fma((double)x[k], (double)x[k], acc);
            }
        } else {
            for (int64_t i = base + threadIdx.x; i < end; i += kThreads) {
                const double x = ld<T>(g + i);
                acc = fma(x, x, acc);
            }
        }
    }
    acc = cta_sum(acc);
    if (threadIdx.x == 0) b.part[blockIdx.x] = acc;
}

// norm = sqrt(sum of the parts) * |scale|; coef = min(1, max_norm / (norm + 1e-6)) * scale
__global__ void __launch_bounds__(kThreads) norm_kernel(const double *part, int32_t n, const float *scale,
                                                        float max_norm, float *norm_out, float *coef) {
    double acc = 0.0;
    for (int32_t i = threadIdx.x; i < n; i += kThreads) acc += part[i];
    acc = cta_sum(acc);
    if (threadIdx.x != 0) return;
    const float s = scale ? *scale : 1.0f;
    const float norm = (float)(sqrt(acc) * (double)fabsf(s));
    if (norm_out) *norm_out = norm;
    if (max_norm > 0.0f) {
        const float c = __fdiv_rn(max_norm, __fadd_rn(norm, 1e-6f));
        *coef = __fmul_rn(c > 1.0f ? 1.0f : c, s);  // a NaN norm gives a NaN factor
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ GradBatch b) {
    const int t = tensor_of(b.start, b.n, blockIdx.x);
    const GradDesc &d = b.d[t];
    const float c = *b.coef;
    T *g = (T *)d.g;
    const int64_t base = (int64_t)(blockIdx.x - b.start[t]) * kChunk;
    const int64_t end = base + kChunk < d.n ? base + kChunk : d.n;
    if (((uintptr_t)g & 15) == 0 && base + kChunk <= d.n) {
        float x[4][8];
#pragma unroll
        for (int u = 0; u < 4; u++) ld8<T>(g + base + (u * kThreads + threadIdx.x) * 8, x[u]);
#pragma unroll
        for (int u = 0; u < 4; u++) {
#pragma unroll
            for (int k = 0; k < 8; k++) x[u][k] = __fmul_rn(x[u][k], c);
            st8<T>(g + base + (u * kThreads + threadIdx.x) * 8, x[u]);
        }
    } else {
        for (int64_t i = base + threadIdx.x; i < end; i += kThreads) st<T>(g + i, __fmul_rn(ld<T>(g + i), c));
    }
}

// ---------------------------------------------------------------- host side

int cuda_status(cudaError_t e) {
    if (e == cudaSuccess) return SMO_OK;
    g_last_cuda_error = (int)e;
    return SMO_ERR_CUDA;
}

// launches over n tensors: full batches, and up to one more for each dtype
int32_t most_launches(int32_t n) { return n / kCap + 3; }

template <class T>
int launch(const GradBatch &b, bool scale, int32_t &parts, cudaStream_t s) {
    if (b.n == 0) return SMO_OK;
    const int32_t chunks = b.start[b.n];
    if (scale) {
        scale_kernel<T><<<(unsigned)chunks, kThreads, 0, s>>>(b);
    } else {
        const int32_t ctas = chunks < kParts ? chunks : kParts;
        sumsq_kernel<T><<<(unsigned)ctas, kThreads, 0, s>>>(b);
        parts += ctas;
    }
    g_launches++;
    return cuda_status(cudaGetLastError());
}

int launch(const GradBatch &b, int32_t dtype, bool scale, int32_t &parts, cudaStream_t s) {
    if (dtype == SMO_DTYPE_F32) return launch<float>(b, scale, parts, s);
    if (dtype == SMO_DTYPE_BF16) return launch<__nv_bfloat16>(b, scale, parts, s);
    return launch<__half>(b, scale, parts, s);
}

// every gradient, batched by dtype: partial sums (coef null) or scaling by *coef
int run(GradOf grad_of, const void *items, int32_t n, double *part, const float *coef, int32_t &parts,
        cudaStream_t s) {
    static thread_local GradBatch b;
    for (int32_t dt = SMO_DTYPE_F32; dt <= SMO_DTYPE_F16; dt++) {
        b.n = 0;
        b.start[0] = 0;
        b.coef = coef;
        for (int32_t i = 0; i <= n; i++) {
            const bool end = i == n;
            const smo_grad g = end ? smo_grad{} : grad_of(items, i);
            if (!end && (g.dtype != dt || g.n == 0)) continue;
            const int64_t chunks = (g.n + kChunk - 1) / kChunk;
            if (end || b.n == kCap) {
                b.part = part + parts;
                const int st = launch(b, dt, coef != nullptr, parts, s);
                if (st != SMO_OK) return st;
                b.n = 0;
                if (end) break;
            }
            b.d[b.n] = GradDesc{g.grad, g.n};
            b.start[b.n + 1] = b.start[b.n] + (int32_t)chunks;
            b.n++;
        }
    }
    return SMO_OK;
}

}  // namespace

// workspace: the factor (one float, 256 bytes), then the partial sums
size_t grad_norm_workspace(int32_t n) {
    return n <= 0 ? 0 : kScratchAlign + (size_t)most_launches(n) * kParts * sizeof(double);
}

static int validate_grads(const smo_grad *g, int32_t n) {
    if (n < 0 || (n > 0 && !g)) return SMO_ERR_INVALID;
    int64_t chunks = 0;
    for (int32_t i = 0; i < n; i++) {
        if (g[i].n < 0 || !known_dtype(g[i].dtype) || g[i].reserved != 0) return SMO_ERR_INVALID;
        if (g[i].n == 0) continue;
        if (!g[i].grad) return SMO_ERR_INVALID;
        if (!is_aligned(g[i].grad, dtype_bytes(g[i].dtype))) return SMO_ERR_ALIGNMENT;
        chunks += (g[i].n + kChunk - 1) / kChunk;
        if (chunks > INT32_MAX) return SMO_ERR_INVALID;  // they are counted in 32 bits (1.7e13 elements)
    }
    return SMO_OK;
}

int grad_norm_enqueue(GradOf grad_of, const void *items, int32_t n, const float *scale, float max_norm, float *norm_out,
                      void *workspace, float **coef_out, cudaStream_t s) {
    float *coef = (float *)workspace;
    double *part = (double *)((char *)workspace + kScratchAlign);
    int32_t parts = 0;
    const int st = run(grad_of, items, n, part, nullptr, parts, s);
    if (st != SMO_OK) return st;
    norm_kernel<<<1, kThreads, 0, s>>>(part, parts, scale, max_norm, norm_out, coef);
    g_launches++;
    if (coef_out) *coef_out = coef;
    return cuda_status(cudaGetLastError());
}

}  // namespace smo

using namespace smo;

extern "C" {

static smo_grad grad_at(const void *items, int32_t i) { return ((const smo_grad *)items)[i]; }

size_t smo_grad_norm_workspace_size(int32_t n) { return grad_norm_workspace(n); }

int smo_grad_norm(const smo_grad *g, int32_t n, float max_norm, float *norm_out, void *workspace,
                  size_t workspace_bytes, void *stream_ptr) {
    int st = validate_grads(g, n);
    if (st != SMO_OK) return st;
    if (!norm_out || !(max_norm >= 0.0f)) return SMO_ERR_INVALID;
    if (!is_aligned(norm_out, 4)) return SMO_ERR_ALIGNMENT;
    cudaStream_t s = (cudaStream_t)stream_ptr;
    if (n == 0) return cuda_status(cudaMemsetAsync(norm_out, 0, sizeof(float), s));
    if (!workspace || workspace_bytes < grad_norm_workspace(n) || !is_aligned(workspace, kScratchAlign))
        return SMO_ERR_WORKSPACE;
    float *coef = nullptr;
    st = grad_norm_enqueue(grad_at, g, n, nullptr, max_norm, norm_out, workspace, &coef, s);
    if (st != SMO_OK || !(max_norm > 0.0f)) return st;
    int32_t parts = 0;
    return run(grad_at, g, n, nullptr, coef, parts, s);
}

}  // extern "C"
