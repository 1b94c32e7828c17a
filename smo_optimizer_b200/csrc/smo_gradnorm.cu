// smo_gradnorm.cu -- the 2-norm over many gradient tensors, and clipping by it.
//
// Each gradient is read once; squares and sums are held in double, so that the
// norm is right to the last fp32 bit (but where it lies within a 64-bit rounding of
// the middle between two) whatever the order of the additions (a clipped step's
// 8-bit codes depend on every bit of the factor), and squares of large elements do
// not overflow.  A CTA adds up every gridDim-th chunk and writes one partial sum; a
// last CTA, in a launch of its own, adds the partial sums in their order.  The order
// goes only by the sizes and by which tensors are aligned: no atomics, the same bits
// every time.  A tensor whose first element is not aligned is read element by
// element throughout (38M bf16 elements in 148 tensors: 19.8 us aligned nowhere,
// 16.4 us aligned; scaling included 48 and 30 us; fp32: 29.0 and 26.7, 72 and 70 us).
#include <climits>
#include <cstring>

#include "smo_multi.cuh"

namespace smo {
namespace {

constexpr int kThreads = 256;
constexpr int kVecs = 4;                  // eight-element accesses of a thread and chunk
constexpr int kChunk = kThreads * 8 * kVecs;
constexpr int kCap = 1024;                // tensors of one launch
constexpr int kFewCap = 128;              // where there are fewer, a smaller parameter: 2 us less to launch
// CTAs of one launch at most, one partial sum each: four times what is resident,
// so that sets of up to 39M elements have one chunk a CTA and the last CTAs level
// out.  38M bf16 elements in 148 tensors, read from L2: 22.6 us with as many CTAs
// as are resident, 16.4 us so; 757M: 227 and 220 us.  Chunks of half the size:
// 26.6 and 232 us.
constexpr int kParts = 148 * 8 * 4;
constexpr int kSumThreads = 1024;         // of the CTA that adds the partial sums

struct GradDesc {
    void *g;
    int64_t n;
};

template <int CAP>
struct GradBatch {
    int32_t n;
    double *part;
    const float *coef;
    int32_t start[CAP + 1];
    GradDesc d[CAP];
};
static_assert(sizeof(GradBatch<kCap>) <= kMaxParamBytes, "launch parameters");

// sum over the CTA, in thread 0
template <int THREADS>
__device__ __forceinline__ double cta_sum(double x) {
    __shared__ double warp[THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_down_sync(0xffffffffu, x, o);
    if ((threadIdx.x & 31) == 0) warp[threadIdx.x >> 5] = x;
    __syncthreads();
    x = threadIdx.x < THREADS / 32 ? warp[threadIdx.x] : 0.0;
    if (threadIdx.x < 32)
#pragma unroll
        for (int o = THREADS / 64; o > 0; o >>= 1) x += __shfl_down_sync(0xffffffffu, x, o);
    return x;
}

template <class T, int CAP>
__global__ void __launch_bounds__(kThreads) sumsq_kernel(const __grid_constant__ GradBatch<CAP> b) {
    wait_for_previous();
    let_next_start();
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
            for (int u = 0; u < kVecs; u++) {
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
    acc = cta_sum<kThreads>(acc);
    if (threadIdx.x == 0) b.part[blockIdx.x] = acc;
}

struct NormArgs {
    const double *part;
    int32_t n;
    const float *scale;
    float max_norm;
    float *norm_out, *coef;
};

// norm = sqrt(sum of the parts) * |scale|; coef = min(1, max_norm / (norm + 1e-6)) * scale
__global__ void __launch_bounds__(kSumThreads) norm_kernel(NormArgs a) {
    // the step or scaling that uses the factor may start: everything in front of the
    // partial sums had ended when those let this kernel start
    if (a.max_norm > 0.0f && a.n > 0) let_next_start();
    wait_for_previous();
    double acc = 0.0;
    for (int32_t i = threadIdx.x; i < a.n; i += kSumThreads) acc += a.part[i];
    acc = cta_sum<kSumThreads>(acc);
    if (threadIdx.x != 0) return;
    const float s = a.scale ? *a.scale : 1.0f;
    const float norm = (float)(sqrt(acc) * (double)fabsf(s));
    if (a.norm_out) *a.norm_out = norm;
    if (a.max_norm > 0.0f) {
        const float c = __fdiv_rn(a.max_norm, __fadd_rn(norm, 1e-6f));
        *a.coef = __fmul_rn(c > 1.0f ? 1.0f : c, s);  // a NaN norm gives a NaN factor
    }
}

template <class T, int CAP>
__global__ void __launch_bounds__(kThreads) scale_kernel(const __grid_constant__ GradBatch<CAP> b) {
    // from the last chunk to the first: what the norm read last is still in L2
    const int32_t chunk = (int32_t)(gridDim.x - 1 - blockIdx.x), t = tensor_of(b.start, b.n, chunk);
    const GradDesc &d = b.d[t];
    T *g = (T *)d.g;
    const int64_t base = (int64_t)(chunk - b.start[t]) * kChunk;
    const int64_t end = base + kChunk < d.n ? base + kChunk : d.n;
    if (((uintptr_t)g & 15) == 0 && base + kChunk <= d.n) {
        float x[kVecs][8];
#pragma unroll
        for (int u = 0; u < kVecs; u++) ld8<T>(g + base + (u * kThreads + threadIdx.x) * 8, x[u]);
        wait_for_previous();
        const float c = *b.coef;
#pragma unroll
        for (int u = 0; u < kVecs; u++) {
#pragma unroll
            for (int k = 0; k < 8; k++) x[u][k] = __fmul_rn(x[u][k], c);
            st8<T>(g + base + (u * kThreads + threadIdx.x) * 8, x[u]);
        }
    } else {
        wait_for_previous();
        const float c = *b.coef;
        for (int64_t i = base + threadIdx.x; i < end; i += kThreads) st<T>(g + i, __fmul_rn(ld<T>(g + i), c));
    }
}

// ---------------------------------------------------------------- host side

// launches over n tensors: full batches, and up to one more for each dtype
int32_t most_launches(int32_t n) { return n / kCap + 3; }

template <class T, int CAP>
int launch(const GradBatch<CAP> &b, int32_t &parts, cudaStream_t s) {
    const int32_t chunks = b.start[b.n];
    cudaError_t e;
    if (b.coef) {
        e = launch_batch(scale_kernel<T, CAP>, (unsigned)chunks, kThreads, b, s);
    } else {
        const int32_t ctas = chunks < kParts ? chunks : kParts;
        e = launch_batch(sumsq_kernel<T, CAP>, (unsigned)ctas, kThreads, b, s);
        parts += ctas;
    }
    g_launches++;
    return cuda_status(e);
}

// the gradients of one dtype: partial sums (coef null) or scaling by *coef
template <class T, int CAP>
int run_type(GradOf grad_of, const void *items, int32_t n, int32_t dtype, double *part, const float *coef,
             int32_t &parts, cudaStream_t s) {
    static thread_local GradBatch<CAP> b;
    b.n = 0;
    b.start[0] = 0;
    b.coef = coef;
    for (int32_t i = 0; i <= n; i++) {
        const bool end = i == n;
        const smo_grad g = end ? smo_grad{} : grad_of(items, i);
        if (!end && (g.dtype != dtype || g.n == 0)) continue;
        if (b.n > 0 && (end || b.n == CAP)) {
            b.part = part + parts;
            const int st = launch<T, CAP>(b, parts, s);
            if (st != SMO_OK) return st;
            b.n = 0;
        }
        if (end) break;
        b.d[b.n] = GradDesc{g.grad, g.n};
        b.start[b.n + 1] = b.start[b.n] + (int32_t)chunks_of(g.n, kChunk);
        b.n++;
    }
    return SMO_OK;
}

// every gradient, batched by dtype
int run(GradOf grad_of, const void *items, int32_t n, double *part, const float *coef, int32_t &parts,
        cudaStream_t s) {
    int st = SMO_OK;
    const bool few = n <= kFewCap;
    for (int32_t dt = SMO_DTYPE_F32; dt <= SMO_DTYPE_F16 && st == SMO_OK; dt++) {
        const auto f = dt == SMO_DTYPE_F32    ? (few ? run_type<float, kFewCap> : run_type<float, kCap>)
                       : dt == SMO_DTYPE_BF16 ? (few ? run_type<__nv_bfloat16, kFewCap> : run_type<__nv_bfloat16, kCap>)
                                              : (few ? run_type<__half, kFewCap> : run_type<__half, kCap>);
        st = f(grad_of, items, n, dt, part, coef, parts, s);
    }
    return st;
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
        chunks += chunks_of(g[i].n, kChunk);
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
    const cudaError_t e =
        launch_batch(norm_kernel, 1, kSumThreads, NormArgs{part, parts, scale, max_norm, norm_out, coef}, s);
    g_launches++;
    if (coef_out) *coef_out = coef;
    return cuda_status(e);
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
