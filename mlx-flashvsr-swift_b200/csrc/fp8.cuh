// fp8.cuh — the 8-bit tensor form shared by the quantiser, the 8-bit linear layers and LayerNorm's backward pass.
//
// A (rows, cols) tensor is held as e4m3 values in rows of ld = cols rounded up to 128 bytes (padding zero) and one
// e8m0 scale code for each block of 128 values along a row: value = e4m3 · 2^(code − 127). The code is the smallest at
// which every |x| of the block is at most 448 · 2^(code − 127) (e4m3's largest), so scaling is exact and e4m3's
// rounding is the only one. Codes are stored as the tensor core's block-scaled MMA wants them in tensor memory: the
// 128 rows × 4 blocks of a tile are 512 bytes, the code of row r, block b at (r % 32)·16 + (r % 128) / 32·4 + b % 4 of
// tile (r / 128, b / 4), tiles row-major; rows and blocks beyond the tensor's have code 0.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace fvsr {

__host__ __device__ inline int64_t fp8_ld(int64_t cols) { return (cols + 127) / 128 * 128; }
__host__ __device__ inline int64_t fp8_scale_tiles(int64_t cols) { return (cols + 511) / 512; }
__host__ __device__ inline int64_t fp8_scale_bytes(int64_t rows, int64_t cols) {
    return (rows + 127) / 128 * fp8_scale_tiles(cols) * 512;
}
__host__ __device__ inline int64_t fp8_code_pos(int64_t row, int64_t block, int64_t tiles) {
    return ((row >> 7) * tiles + (block >> 2)) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (block & 3);
}

// The code of a block whose largest magnitude has these fp32 bits (sign clear): e = ceil(log2(amax / 448)) from the
// exponent field and a comparison of the fraction with 448's (1.75 · 2^8); 255 (NaN) when the block holds an infinity
// or a NaN, which then reads back as NaN throughout.
__device__ __forceinline__ uint32_t fp8_code(uint32_t amax_bits) {
    const int field = (int)(amax_bits >> 23);
    if (field >= 255) return 255u;
    const int code = field - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return code < 0 ? 0u : (uint32_t)code;
}
// 2^(127 − code), the exact factor that brings a block's values into e4m3's range (NaN for code 255).
__device__ __forceinline__ float fp8_up(uint32_t code) {
    return __uint_as_float(code == 255u ? 0x7FC00000u : (254u - code) << 23);
}
// 2^(code − 127), the factor that reads them back (code 0 is the subnormal 2^−127).
__device__ __forceinline__ float fp8_down(uint32_t code) {
    return __uint_as_float(code == 0u ? 0x00400000u : code == 255u ? 0x7FC00000u : code << 23);
}
// Two fp32 values rounded to e4m3 (to nearest, ties to even), lo in the low byte.
__device__ __forceinline__ uint32_t fp8_pack2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two e4m3 values as fp32 (exact: every e4m3 value is an fp16 value).
__device__ __forceinline__ void fp8_unpack2(uint32_t two, float& lo, float& hi) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    lo = f.x, hi = f.y;
}

__device__ __forceinline__ float load_as_float(const float* p) { return *p; }
__device__ __forceinline__ float load_as_float(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_from_float(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_from_float(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Multiprocessors of the current device (asked for once per device).
inline int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
    return n;
}
// Lets `kernel` take `bytes` of dynamic shared memory on the current device (once per kernel and device: kernel is a
// template argument so that each has its own record).
template <auto kernel>
cudaError_t allow_smem(size_t bytes) {
    static std::atomic<int> allowed[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && (size_t)allowed[dev].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) allowed[dev].store((int)bytes, std::memory_order_relaxed);
    return e;
}

// ---- launchers ----
// x (rows, cols) fp32 or bf16 → its 8-bit form (q, scale) and / or the 8-bit form of its transpose (qt, scale_t);
// either pair may be NULL. square: one scale for each 128 × 128 square instead of each row's 128 values.
cudaError_t launch_quantize_fp8(int64_t rows, int64_t cols, const void* x, int dtype, bool square, uint8_t* q,
                                uint8_t* scale, uint8_t* qt, uint8_t* scale_t, cudaStream_t st);
cudaError_t launch_fp8_codes(int64_t rows, int64_t cols, const uint8_t* scale, uint8_t* out, cudaStream_t st);
cudaError_t launch_dequantize_fp8(int64_t rows, int64_t cols, const uint8_t* q, const uint8_t* scale, void* out,
                                  int dtype, cudaStream_t st);

// out (M, N) = epilogue(x · wᵀ + bias) on 8-bit operands (gemm_fp8.cu, gemv_fp8.cu).
struct Fp8GemmArgs {
    int M, N, K;
    const uint8_t* x;         // (M, ld(K)) e4m3
    const uint8_t* x_scale;
    const uint8_t* w;         // (N, ld(K)) e4m3
    const uint8_t* w_scale;
    const __nv_bfloat16* bias;  // (N) or NULL
    const __nv_bfloat16* gate;  // (N), gated residual only
    const void* resid;          // (M, N) in out's dtype, gated residual only
    void* out;
    int mode, out_dtype;
};
// How a product is cut: `splits` parts of the sum over K, part_blocks blocks of 128 each (a multiple of 4: whole tiles of
// codes) except the last; more than one part, or a bf16 output's sum of more than one chain, leaves fp32 partial products
// (splits, M, ld) in the workspace.
struct Fp8GemmPlan {
    int splits, part_blocks;
    int64_t partial_ld;
    size_t partial_bytes;
};
Fp8GemmPlan plan_gemm_fp8(int M, int N, int K);
// Up to kFewTokens rows of x, without a workspace: x in a.x / a.x_scale, or bf16 in xb (gemv_fp8.cu).
constexpr int kFewTokens = 16;
cudaError_t launch_gemv_fp8(const Fp8GemmArgs& a, const __nv_bfloat16* xb, cudaStream_t st);
cudaError_t launch_gemm_fp8(const Fp8GemmArgs& a, const Fp8GemmPlan& plan, float* partial, cudaStream_t st);

// LayerNorm for training (norm_train.cu).
struct NormTrainArgs {
    int64_t m;
    int c, dtype;                    // of x / dy, the vectors, out / dx
    const void* x;
    const uint8_t* x_scale;          // non-NULL: x is the 8-bit form (backward only)
    const void *weight, *bias, *shift, *scale;
    float eps;
    void* out;                       // y or dx
    float *mean, *rstd;
    const void* dy;
    float *dweight, *dbias, *dshift, *dscale;
    float* partial;                  // norm_backward_ctas × 2 × c
};
cudaError_t launch_layernorm_train(const NormTrainArgs& a, cudaStream_t st);
cudaError_t launch_layernorm_backward(const NormTrainArgs& a, cudaStream_t st);
// CTAs of the backward pass, each leaving 2 · c partial sums.
int norm_backward_ctas(int64_t m, int c);
constexpr int kNormTrainMaxC = 8192;

}  // namespace fvsr
