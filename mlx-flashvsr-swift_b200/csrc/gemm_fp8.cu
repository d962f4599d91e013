// gemm_fp8.cu — the linear layers on 8-bit operands: out = epilogue(x · wᵀ + bias), x (M, K) and w (N, K) in the 8-bit
// form of fp8.cuh (a scale for each block of 128 along K), fp32 sums, one rounding at the end.
#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"

namespace fvsr {

namespace {

constexpr int kTM = 64, kTN = 64, kThreads = 256;

__device__ __forceinline__ float gelu_tanh(float x) {
    return 0.5f * x * (1.0f + tanhf(0.7978845608028654f * (x + 0.044715f * x * x * x)));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) gemm_fp8_simple_kernel(const Fp8GemmArgs a) {
    __shared__ float xs[kTM][33], ws[kTN][33];
    griddep_wait_then_release();
    const int m0 = blockIdx.y * kTM, n0 = blockIdx.x * kTN;
    const int64_t ld = fp8_ld(a.K), tiles = fp8_scale_tiles(a.K);
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < (int)ld; k0 += 32) {
        for (int i = threadIdx.x; i < 64 * 16; i += kThreads) {
            const int r = i / 16, c = (i % 16) * 2;
            float lo = 0.0f, hi = 0.0f;
            if (m0 + r < a.M) {
                fp8_unpack2(*reinterpret_cast<const uint16_t*>(a.x + (m0 + r) * ld + k0 + c), lo, hi);
                const float s = fp8_down(a.x_scale[fp8_code_pos(m0 + r, k0 >> 7, tiles)]);
                lo *= s, hi *= s;
            }
            xs[r][c] = lo, xs[r][c + 1] = hi;
            lo = hi = 0.0f;
            if (n0 + r < a.N) {
                fp8_unpack2(*reinterpret_cast<const uint16_t*>(a.w + (n0 + r) * ld + k0 + c), lo, hi);
                const float s = fp8_down(a.w_scale[fp8_code_pos(n0 + r, k0 >> 7, tiles)]);
                lo *= s, hi *= s;
            }
            ws[r][c] = lo, ws[r][c + 1] = hi;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 32; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[ty * 4 + i][k], ws[tx + 16 * j][k], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
            if (m >= a.M || n >= a.N) continue;
            float y = acc[i][j] + (a.bias ? __bfloat162float(a.bias[n]) : 0.0f);
            if (a.mode == FVSR_LINEAR_GELU) y = gelu_tanh(y);
            if (a.mode == FVSR_LINEAR_GATED_RESIDUAL)
                y = fmaf(__bfloat162float(a.gate[n]), y, load_as_float(static_cast<const T*>(a.resid) + m * a.N + n));
            store_from_float(static_cast<T*>(a.out) + m * a.N + n, y);
        }
}

}  // namespace

cudaError_t launch_gemm_fp8(const Fp8GemmArgs& a, void*, cudaStream_t st) {
    const dim3 grid((a.N + kTN - 1) / kTN, (a.M + kTM - 1) / kTM);
    return a.out_dtype == FVSR_BF16 ? launch_pdl(gemm_fp8_simple_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, st, a)
                                    : launch_pdl(gemm_fp8_simple_kernel<float>, grid, dim3(kThreads), 0, st, a);
}

}  // namespace fvsr
