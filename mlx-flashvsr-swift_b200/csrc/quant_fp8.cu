// quant_fp8.cu — a tensor into its 8-bit form (fp8.cuh) and back, and into the 8-bit form of its transpose: the form the
// activations of the DiT block's linear layers are kept in between the forward and the backward pass, and the operands
// of the 8-bit linear layers (blocks along the channels for the forward and input-gradient products, blocks along the
// tokens for the weight gradient, 128 × 128 squares for weights, whose transpose has the same scales).
//
// Both directions move bytes and do little else. quantize_kernel: one CTA of 8 warps per 128 × 128 tile, which each warp
// reads 16 rows of with 128-bit loads, all in flight at once, and keeps in registers; a row's largest magnitude is a
// shuffle over the lanes that hold it. The row form is written from the registers. For the transposed form the tile goes
// through shared memory once, as stored: a warp then owns 32 rows and a lane two neighbouring columns of them, so that
// reads are free of bank conflicts and a lane writes 32 consecutive bytes of each of its two lines. Either way x is read
// once for both forms.
#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"
#include "sm100.cuh"

namespace fvsr {

namespace {

using sm100::bf2_to_f;
using sm100::pack_bf16x2;

constexpr int kT = 128, kThreads = 256;

// Elements of T in a 16-byte load, as the pieces of a tile row a lane holds.
template <typename T>
struct Piece {
    static constexpr int kElems = 16 / (int)sizeof(T);
    static constexpr int kLanes = kT / kElems;              // lanes of a row
    static constexpr int kRowsPerLoad = 32 / kLanes;        // rows a warp covers with one load
    static constexpr int kLoads = 16 / kRowsPerLoad;        // loads for a warp's 16 rows
};

__device__ __forceinline__ void unpack(const uint4& u, float (&f)[8], const __nv_bfloat16*) {
    bf2_to_f(u.x, f[0], f[1]), bf2_to_f(u.y, f[2], f[3]), bf2_to_f(u.z, f[4], f[5]), bf2_to_f(u.w, f[6], f[7]);
}
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[4], const float*) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
}
// The largest magnitude of a piece, as fp32 bits (an integer maximum: a NaN's bits are above infinity's).
__device__ __forceinline__ uint32_t piece_max(const uint4& u, const __nv_bfloat16*) {
    const uint32_t m = 0x7FFF7FFFu;
    const uint32_t a = __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
    return max(a & 0xFFFF0000u, a << 16);
}
__device__ __forceinline__ uint32_t piece_max(const uint4& u, const float*) {
    const uint32_t m = 0x7FFFFFFFu;
    return max(max(u.x & m, u.y & m), max(u.z & m, u.w & m));
}

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    return fp8_pack2(a, b) | (fp8_pack2(c, d) << 16);
}

// kVec: rows are 16-byte aligned and their lengths whole pieces; else element by element.
template <typename T, bool kVec>
__device__ __forceinline__ uint4 load_piece(const T* row, int64_t c, int64_t cols) {
    if (kVec) return c < cols ? __ldcs(reinterpret_cast<const uint4*>(row + c)) : make_uint4(0, 0, 0, 0);
    alignas(16) T v[Piece<T>::kElems];
#pragma unroll
    for (int i = 0; i < Piece<T>::kElems; ++i) v[i] = c + i < cols ? row[c + i] : T(0.0f);
    return *reinterpret_cast<const uint4*>(v);
}

// The codes of a line (form row) beyond its last block, up to the end of the last tile of codes, are zero.
__device__ __forceinline__ void put_code(uint8_t* scale, int64_t line, int64_t block, int64_t blocks, uint32_t code) {
    const int64_t tiles = (blocks + 3) >> 2;
    uint8_t* p = scale + fp8_code_pos(line, block, tiles);
    *p = (uint8_t)code;
    if (block == blocks - 1)
        for (int i = 1; i < 4 - (int)(block & 3); ++i) p[i] = 0;
}

template <typename T, bool kVec, bool kTrans>
__global__ void __launch_bounds__(kThreads) quantize_kernel(int64_t rows, int64_t cols, const T* __restrict__ x,
                                                            int square, uint8_t* __restrict__ q,
                                                            uint8_t* __restrict__ scale, uint8_t* __restrict__ qt,
                                                            uint8_t* __restrict__ scale_t) {
    using P = Piece<T>;
    extern __shared__ uint4 tile4[];  // kTrans: the tile, [128][128] of T
    __shared__ uint32_t warp_max[kThreads / 32], col_max[4][kT];
    griddep_wait_then_release();
    const int64_t ct = (cols + kT - 1) / kT, rt = (rows + kT - 1) / kT;
    const int64_t rb = blockIdx.x / ct, cb = blockIdx.x % ct, r0 = rb * kT, c0 = cb * kT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane / P::kLanes, piece = lane % P::kLanes;
    uint4 v[P::kLoads];
#pragma unroll
    for (int i = 0; i < P::kLoads; ++i) {
        const int64_t r = r0 + warp * 16 + i * P::kRowsPerLoad + sub;
        v[i] = r < rows ? load_piece<T, kVec>(x + r * cols, c0 + piece * P::kElems, cols) : make_uint4(0, 0, 0, 0);
    }
    uint32_t top[P::kLoads];
#pragma unroll
    for (int i = 0; i < P::kLoads; ++i) {
        top[i] = piece_max(v[i], x);
#pragma unroll
        for (int o = P::kLanes / 2; o >= 1; o >>= 1) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
        if (kTrans) tile4[(warp * 16 + i * P::kRowsPerLoad + sub) * P::kLanes + piece] = v[i];
    }
    if (square) {
        uint32_t m = top[0];
#pragma unroll
        for (int i = 1; i < P::kLoads; ++i) m = max(m, top[i]);
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0) warp_max[warp] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) m = max(m, warp_max[i]);
#pragma unroll
        for (int i = 0; i < P::kLoads; ++i) top[i] = m;
    }
    if (q) {
        const int64_t ld = ct * kT;
#pragma unroll
        for (int i = 0; i < P::kLoads; ++i) {
            const int64_t r = r0 + warp * 16 + i * P::kRowsPerLoad + sub;
            const uint32_t code = fp8_code(top[i]);
            const float up = fp8_up(code);
            float f[P::kElems];
            unpack(v[i], f, x);
            if (r < rows) {
                uint8_t* p = q + r * ld + c0 + piece * P::kElems;
                if constexpr (P::kElems == 8)
                    *reinterpret_cast<uint2*>(p) = make_uint2(pack4(f[0] * up, f[1] * up, f[2] * up, f[3] * up),
                                                              pack4(f[4] * up, f[5] * up, f[6] * up, f[7] * up));
                else
                    *reinterpret_cast<uint32_t*>(p) = pack4(f[0] * up, f[1] * up, f[2] * up, f[3] * up);
            }
            if (piece == 0) put_code(scale, r, cb, ct, r < rows ? code : 0u);
        }
    }
    if constexpr (kTrans) {
        // lane: columns 2·cp, 2·cp + 1 of the 32 rows [32·quarter, +32)
        __syncthreads();
        const int quarter = warp & 3, cp = (warp >> 2) * 32 + lane;
        const int64_t ld = rt * kT;
        float a[32], b[32];
        uint32_t ma = 0, mb = 0;
        const T* tile = reinterpret_cast<const T*>(tile4) + (quarter * 32) * kT + 2 * cp;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if constexpr (sizeof(T) == 2) {
                bf2_to_f(*reinterpret_cast<const uint32_t*>(tile + i * kT), a[i], b[i]);
            } else {
                const float2 t = *reinterpret_cast<const float2*>(tile + i * kT);
                a[i] = t.x, b[i] = t.y;
            }
            ma = max(ma, __float_as_uint(a[i]) & 0x7FFFFFFFu);
            mb = max(mb, __float_as_uint(b[i]) & 0x7FFFFFFFu);
        }
        if (square) {
            ma = mb = top[0];
        } else {
            *reinterpret_cast<uint2*>(&col_max[quarter][2 * cp]) = make_uint2(ma, mb);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint2 m = *reinterpret_cast<const uint2*>(&col_max[i][2 * cp]);
                ma = max(ma, m.x), mb = max(mb, m.y);
            }
        }
        const int64_t line = c0 + 2 * cp;
        const uint32_t code_a = fp8_code(ma), code_b = fp8_code(mb);
        auto emit = [&](const float (&f)[32], float up, int64_t l) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                w[i] = pack4(f[4 * i] * up, f[4 * i + 1] * up, f[4 * i + 2] * up, f[4 * i + 3] * up);
            uint4* p = reinterpret_cast<uint4*>(qt + l * ld + r0 + quarter * 32);
            p[0] = make_uint4(w[0], w[1], w[2], w[3]);
            p[1] = make_uint4(w[4], w[5], w[6], w[7]);
        };
        if (line < cols) emit(a, fp8_up(code_a), line);
        if (line + 1 < cols) emit(b, fp8_up(code_b), line + 1);
        if (quarter == 0) {
            put_code(scale_t, line, rb, rt, line < cols ? code_a : 0u);
            put_code(scale_t, line + 1, rb, rt, line + 1 < cols ? code_b : 0u);
        }
    }
}

// A warp takes 512 columns of a row: a lane 16 values, and the four codes of the row's tile as one word. kRows rows at
// once keep enough loads in flight.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(int64_t rows, int64_t cols, const uint8_t* __restrict__ q,
                                                              const uint8_t* __restrict__ scale, T* __restrict__ out) {
    constexpr int kRows = 4;
    griddep_wait_then_release();
    const int64_t ld = fp8_ld(cols), tiles = fp8_scale_tiles(cols);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t items = (rows + kRows - 1) / kRows * tiles;
    for (int64_t it = (int64_t)blockIdx.x * (kThreads / 32) + warp; it < items; it += (int64_t)gridDim.x * (kThreads / 32)) {
        const int64_t tile = it % tiles, r0 = it / tiles * kRows, c = tile * 512 + lane * 16;
        uint4 v[kRows];
        uint32_t word[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const bool here = r0 + i < rows && c < cols;
            v[i] = here ? __ldcs(reinterpret_cast<const uint4*>(q + (r0 + i) * ld + c)) : make_uint4(0, 0, 0, 0);
            word[i] = here ? *reinterpret_cast<const uint32_t*>(scale + fp8_code_pos(r0 + i, tile * 4, tiles)) : 0u;
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (r0 + i >= rows || c >= cols) continue;
            const float down = fp8_down((word[i] >> (8 * (lane >> 3))) & 255u);
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            float f[16];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                fp8_unpack2(w[j >> 1] >> (16 * (j & 1)), f[2 * j], f[2 * j + 1]);
                f[2 * j] *= down, f[2 * j + 1] *= down;
            }
            T* p = out + (r0 + i) * cols + c;
            if (kVec) {
#pragma unroll
                for (int j = 0; j < 16; j += Piece<T>::kElems) {
                    if (c + j >= cols) break;
                    if constexpr (sizeof(T) == 2)
                        *reinterpret_cast<uint4*>(p + j) =
                            make_uint4(pack_bf16x2(f[j], f[j + 1]), pack_bf16x2(f[j + 2], f[j + 3]),
                                       pack_bf16x2(f[j + 4], f[j + 5]), pack_bf16x2(f[j + 6], f[j + 7]));
                    else
                        *reinterpret_cast<float4*>(p + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (c + j < cols) store_from_float(p + j, f[j]);
            }
        }
    }
}

int sm_count() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        n = 148;
    return n;
}

template <typename T, bool kVec, bool kTrans>
cudaError_t quantize(int64_t rows, int64_t cols, const T* x, bool square, uint8_t* q, uint8_t* scale, uint8_t* qt,
                     uint8_t* scale_t, cudaStream_t st) {
    auto kernel = quantize_kernel<T, kVec, kTrans>;
    const size_t smem = kTrans ? sizeof(T) * kT * kT : 0;
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    const int64_t tiles = (rows + kT - 1) / kT * ((cols + kT - 1) / kT);
    return launch_pdl(kernel, dim3((unsigned)tiles), dim3(kThreads), smem, st, rows, cols, x, square ? 1 : 0, q, scale,
                      qt, scale_t);
}

template <typename T>
cudaError_t quantize_t(int64_t rows, int64_t cols, const T* x, bool square, uint8_t* q, uint8_t* scale, uint8_t* qt,
                       uint8_t* scale_t, cudaStream_t st) {
    const bool vec = cols % Piece<T>::kElems == 0;
    if (qt) return vec ? quantize<T, true, true>(rows, cols, x, square, q, scale, qt, scale_t, st)
                       : quantize<T, false, true>(rows, cols, x, square, q, scale, qt, scale_t, st);
    return vec ? quantize<T, true, false>(rows, cols, x, square, q, scale, qt, scale_t, st)
               : quantize<T, false, false>(rows, cols, x, square, q, scale, qt, scale_t, st);
}

template <typename T>
cudaError_t dequantize_t(int64_t rows, int64_t cols, const uint8_t* q, const uint8_t* scale, T* out, cudaStream_t st) {
    const bool vec = cols % Piece<T>::kElems == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const int64_t items = (rows + 3) / 4 * fp8_scale_tiles(cols), blocks = (items + 7) / 8, most = (int64_t)sm_count() * 8;
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    return vec ? launch_pdl(dequantize_kernel<T, true>, grid, dim3(kThreads), 0, st, rows, cols, q, scale, out)
               : launch_pdl(dequantize_kernel<T, false>, grid, dim3(kThreads), 0, st, rows, cols, q, scale, out);
}

}  // namespace

cudaError_t launch_quantize_fp8(int64_t rows, int64_t cols, const void* x, int dtype, bool square, uint8_t* q,
                                uint8_t* scale, uint8_t* qt, uint8_t* scale_t, cudaStream_t st) {
    return dtype == FVSR_BF16
               ? quantize_t(rows, cols, static_cast<const __nv_bfloat16*>(x), square, q, scale, qt, scale_t, st)
               : quantize_t(rows, cols, static_cast<const float*>(x), square, q, scale, qt, scale_t, st);
}

cudaError_t launch_dequantize_fp8(int64_t rows, int64_t cols, const uint8_t* q, const uint8_t* scale, void* out,
                                  int dtype, cudaStream_t st) {
    return dtype == FVSR_BF16 ? dequantize_t(rows, cols, q, scale, static_cast<__nv_bfloat16*>(out), st)
                              : dequantize_t(rows, cols, q, scale, static_cast<float*>(out), st);
}

}  // namespace fvsr
