// norm_train.cu — LayerNorm over the channels for training: the forward pass that keeps each row's mean and
// rstd = 1/√(var + eps), and the backward pass with the gradients of its vectors.
//   n = (x − mean)·rstd,  y = (n·w + b)·(1 + scale) + shift          (w, b and shift, scale each optional)
//   g = dy·(1 + scale)·w, dx = rstd·(g − mean_c(g) − n·mean_c(g·n))
//   A = Σ_rows dy·n, B = Σ_rows dy: dw = (1 + scale)·A, db = (1 + scale)·B, dscale = w·A + b·B, dshift = B.
// fp32 throughout, one rounding of y and dx to the tensors' type. The vectors' gradients are summed per CTA over its
// rows, then over the CTAs in a fixed order, so they do not depend on timing.
#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"

namespace fvsr {

namespace {

constexpr int kThreads = 256;

// The sums of a and b over the CTA, in every thread.
__device__ __forceinline__ void cta_sum2(float& a, float& b) {
    __shared__ float part[2][kThreads / 32];
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[0][threadIdx.x >> 5] = a, part[1][threadIdx.x >> 5] = b;
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) a += part[0][i], b += part[1][i];
}

template <typename T>
__device__ __forceinline__ float vec_or(const void* v, int c, float otherwise) {
    return v ? load_as_float(static_cast<const T*>(v) + c) : otherwise;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) norm_train_kernel(const NormTrainArgs a) {
    griddep_wait_then_release();
    for (int64_t r = blockIdx.x; r < a.m; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.c;
        float s = 0.0f, q = 0.0f;
        for (int c = threadIdx.x; c < a.c; c += kThreads) s += load_as_float(x + c);
        cta_sum2(s, q);
        const float mean = s / (float)a.c;
        q = 0.0f;
        for (int c = threadIdx.x; c < a.c; c += kThreads) {
            const float d = load_as_float(x + c) - mean;
            q = fmaf(d, d, q);
        }
        float unused = 0.0f;
        cta_sum2(q, unused);
        const float rstd = 1.0f / sqrtf(q / (float)a.c + a.eps);
        if (threadIdx.x == 0) a.mean[r] = mean, a.rstd[r] = rstd;
        for (int c = threadIdx.x; c < a.c; c += kThreads) {
            const float n = (load_as_float(x + c) - mean) * rstd;
            const float y = fmaf(n, vec_or<T>(a.weight, c, 1.0f), vec_or<T>(a.bias, c, 0.0f));
            store_from_float(static_cast<T*>(a.out) + r * a.c + c,
                             fmaf(y, 1.0f + vec_or<T>(a.scale, c, 0.0f), vec_or<T>(a.shift, c, 0.0f)));
        }
    }
}

template <typename T>
__device__ __forceinline__ float x_at(const NormTrainArgs& a, int64_t r, int c) {
    if (!a.x_scale) return load_as_float(static_cast<const T*>(a.x) + r * a.c + c);
    float lo, hi;
    fp8_unpack2(static_cast<const uint8_t*>(a.x)[r * fp8_ld(a.c) + c], lo, hi);
    return lo * fp8_down(a.x_scale[fp8_code_pos(r, c >> 7, fp8_scale_tiles(a.c))]);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) norm_backward_kernel(const NormTrainArgs a) {
    extern __shared__ float sums[];  // A[c], B[c]: thread t owns the channels t, t + 256, …
    griddep_wait_then_release();
    for (int c = threadIdx.x; c < 2 * a.c; c += kThreads) sums[c] = 0.0f;
    __syncthreads();
    for (int64_t r = blockIdx.x; r < a.m; r += gridDim.x) {
        const T* dy = static_cast<const T*>(a.dy) + r * a.c;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int c = threadIdx.x; c < a.c; c += kThreads) {
            const float n = (x_at<T>(a, r, c) - mean) * rstd, d = load_as_float(dy + c);
            const float g = d * ((1.0f + vec_or<T>(a.scale, c, 0.0f)) * vec_or<T>(a.weight, c, 1.0f));
            s1 += g;
            s2 = fmaf(g, n, s2);
            sums[c] = fmaf(d, n, sums[c]);
            sums[a.c + c] += d;
        }
        cta_sum2(s1, s2);
        s1 /= (float)a.c, s2 /= (float)a.c;
        for (int c = threadIdx.x; c < a.c; c += kThreads) {
            const float n = (x_at<T>(a, r, c) - mean) * rstd, d = load_as_float(dy + c);
            const float g = d * ((1.0f + vec_or<T>(a.scale, c, 0.0f)) * vec_or<T>(a.weight, c, 1.0f));
            store_from_float(static_cast<T*>(a.out) + r * a.c + c, rstd * (g - s1 - n * s2));
        }
    }
    for (int c = threadIdx.x; c < a.c; c += kThreads) {
        a.partial[(int64_t)blockIdx.x * 2 * a.c + c] = sums[c];
        a.partial[((int64_t)blockIdx.x * 2 + 1) * a.c + c] = sums[a.c + c];
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) norm_vectors_kernel(const NormTrainArgs a, int ctas) {
    griddep_wait_then_release();
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.c) return;
    float sa = 0.0f, sb = 0.0f;
    for (int i = 0; i < ctas; ++i) {
        sa += a.partial[(int64_t)i * 2 * a.c + c];
        sb += a.partial[((int64_t)i * 2 + 1) * a.c + c];
    }
    const float s1 = 1.0f + vec_or<T>(a.scale, c, 0.0f);
    if (a.dweight) a.dweight[c] = s1 * sa;
    if (a.dbias) a.dbias[c] = s1 * sb;
    if (a.dscale) a.dscale[c] = fmaf(vec_or<T>(a.weight, c, 1.0f), sa, vec_or<T>(a.bias, c, 0.0f) * sb);
    if (a.dshift) a.dshift[c] = sb;
}

template <typename T>
cudaError_t backward(const NormTrainArgs& a, cudaStream_t st) {
    const size_t smem = sizeof(float) * 2 * a.c;
    cudaError_t e = cudaFuncSetAttribute(norm_backward_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(sizeof(float) * 2 * kNormTrainMaxC));
    if (e != cudaSuccess) return e;
    const int ctas = (int)norm_backward_ctas(a.m, a.c);
    if (ctas > 0) e = launch_pdl(norm_backward_kernel<T>, dim3(ctas), dim3(kThreads), smem, st, a);
    if (e != cudaSuccess || !(a.dweight || a.dbias || a.dscale || a.dshift)) return e;
    return launch_pdl(norm_vectors_kernel<T>, dim3((a.c + kThreads - 1) / kThreads), dim3(kThreads), 0, st, a, ctas);
}

}  // namespace

int64_t norm_backward_ctas(int64_t m, int) { return m < 296 ? m : 296; }

cudaError_t launch_layernorm_train(const NormTrainArgs& a, cudaStream_t st) {
    if (a.m <= 0) return cudaSuccess;
    const dim3 grid((unsigned)(a.m < 65536 ? a.m : 65536));
    return a.dtype == FVSR_BF16 ? launch_pdl(norm_train_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, st, a)
                                : launch_pdl(norm_train_kernel<float>, grid, dim3(kThreads), 0, st, a);
}

cudaError_t launch_layernorm_backward(const NormTrainArgs& a, cudaStream_t st) {
    return a.dtype == FVSR_BF16 ? backward<__nv_bfloat16>(a, st) : backward<float>(a, st);
}

}  // namespace fvsr
