// quant_fp8.cu — a tensor into its 8-bit form (fp8.cuh) and back, and into the 8-bit form of its transpose: the form the
// activations of the DiT block's linear layers are kept in between the forward and the backward pass, and the operands
// of the 8-bit linear layers (blocks along the channels for the forward and input-gradient products, blocks along the
// tokens for the weight gradient, 128 × 128 squares for weights, whose transpose has the same scales).
//
// One CTA per 128 × 128 tile: the tile is staged once in shared memory, so both orientations cost one read of x.
#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"

namespace fvsr {

namespace {

constexpr int kT = 128, kPitch = kT + 1, kThreads = 256;

// Writes one orientation of the staged tile: line l (a row of the form) holds tile element (l, i) at
// tile[l·sl + i·si]. lines = how many of the 128 lines exist; line0 / block = the tile's place in the form.
__device__ void emit(const float* tile, int sl, int si, const uint32_t* codes, int lines, int64_t line0, int64_t block,
                     int64_t blocks, int64_t ld, uint8_t* q, uint8_t* scale) {
    for (int i = threadIdx.x; i < kT * (kT / 4); i += kThreads) {
        const int l = i / (kT / 4), c = (i % (kT / 4)) * 4;
        if (l >= lines) break;
        const float up = fp8_up(codes[l]);
        const float* p = tile + l * sl + c * si;
        const uint32_t lo = fp8_pack2(p[0] * up, p[si] * up), hi = fp8_pack2(p[2 * si] * up, p[3 * si] * up);
        *reinterpret_cast<uint32_t*>(q + (line0 + l) * ld + block * kT + c) = lo | (hi << 16);
    }
    const int64_t tiles = (blocks + 3) / 4;
    for (int l = threadIdx.x; l < kT; l += kThreads) {
        scale[fp8_code_pos(line0 + l, block, tiles)] = (uint8_t)(l < lines ? codes[l] : 0u);
        if (block == blocks - 1)  // the rest of the last tile of codes
            for (int64_t b = blocks; b < 4 * tiles; ++b) scale[fp8_code_pos(line0 + l, b, tiles)] = 0;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_kernel(int64_t rows, int64_t cols, const T* __restrict__ x,
                                                            int square, uint8_t* __restrict__ q,
                                                            uint8_t* __restrict__ scale, uint8_t* __restrict__ qt,
                                                            uint8_t* __restrict__ scale_t) {
    extern __shared__ float tile[];  // [128][129]
    __shared__ uint32_t row_code[kT], col_code[kT], warp_max[kThreads / 32];
    griddep_wait_then_release();
    const int64_t rt = (rows + kT - 1) / kT, ct = (cols + kT - 1) / kT;
    for (int64_t t = blockIdx.x; t < rt * ct; t += gridDim.x) {
        const int64_t r0 = t / ct * kT, c0 = t % ct * kT;
        const int nr = (int)min((int64_t)kT, rows - r0), nc = (int)min((int64_t)kT, cols - c0);
        __syncthreads();
        for (int i = threadIdx.x; i < kT * kT; i += kThreads) {
            const int r = i / kT, c = i % kT;
            tile[r * kPitch + c] = r < nr && c < nc ? load_as_float(x + (r0 + r) * cols + c0 + c) : 0.0f;
        }
        __syncthreads();
        {   // threads 0..127: a row each, 128..255: a column each
            const int l = threadIdx.x % kT;
            const bool col = threadIdx.x >= kT;
            const float* p = tile + (col ? l : l * kPitch);
            const int step = col ? kPitch : 1;
            uint32_t m = 0;
            for (int i = 0; i < kT; ++i) m = max(m, __float_as_uint(p[i * step]) & 0x7FFFFFFFu);
            if (square) {
                m = __reduce_max_sync(0xffffffffu, m);
                if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
                __syncthreads();
                for (int i = 0; i < kThreads / 32; ++i) m = max(m, warp_max[i]);
            }
            (col ? col_code : row_code)[l] = fp8_code(m);
        }
        __syncthreads();
        if (q) emit(tile, kPitch, 1, row_code, nr, r0, c0 / kT, ct, ct * kT, q, scale);
        if (qt) emit(tile, 1, kPitch, col_code, nc, c0, r0 / kT, rt, rt * kT, qt, scale_t);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(int64_t rows, int64_t cols, const uint8_t* __restrict__ q,
                                                              const uint8_t* __restrict__ scale, T* __restrict__ out) {
    griddep_wait_then_release();
    const int64_t n = rows * cols, ld = fp8_ld(cols), tiles = fp8_scale_tiles(cols);
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
        const int64_t r = i / cols, c = i % cols;
        float lo, hi;
        fp8_unpack2(q[r * ld + c], lo, hi);
        store_from_float(out + i, lo * fp8_down(scale[fp8_code_pos(r, c >> 7, tiles)]));
    }
}

int sm_count() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n;
}

}  // namespace

cudaError_t launch_quantize_fp8(int64_t rows, int64_t cols, const void* x, int dtype, bool square, uint8_t* q,
                                uint8_t* scale, uint8_t* qt, uint8_t* scale_t, cudaStream_t st) {
    const int64_t tiles = (rows + kT - 1) / kT * ((cols + kT - 1) / kT);
    const size_t smem = sizeof(float) * kT * kPitch;
    const int grid = (int)(tiles < (1 << 30) ? tiles : (1 << 30));
    auto go = [&](auto kernel, auto* p) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        return launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, st, rows, cols, p, square ? 1 : 0, q, scale, qt,
                          scale_t);
    };
    return dtype == FVSR_BF16 ? go(quantize_kernel<__nv_bfloat16>, static_cast<const __nv_bfloat16*>(x))
                              : go(quantize_kernel<float>, static_cast<const float*>(x));
}

cudaError_t launch_dequantize_fp8(int64_t rows, int64_t cols, const uint8_t* q, const uint8_t* scale, void* out,
                                  int dtype, cudaStream_t st) {
    const int64_t blocks = (rows * cols + kThreads - 1) / kThreads, most = (int64_t)sm_count() * 8;
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    return dtype == FVSR_BF16 ? launch_pdl(dequantize_kernel<__nv_bfloat16>, grid, dim3(kThreads), 0, st, rows, cols, q,
                                           scale, static_cast<__nv_bfloat16*>(out))
                              : launch_pdl(dequantize_kernel<float>, grid, dim3(kThreads), 0, st, rows, cols, q, scale,
                                           static_cast<float*>(out));
}

}  // namespace fvsr
