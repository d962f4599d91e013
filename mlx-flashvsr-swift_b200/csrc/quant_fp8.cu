// quant_fp8.cu — a tensor into its 8-bit form (fp8.cuh) and back, and into the 8-bit form of its transpose: the form the
// activations of the DiT block's linear layers are kept in between the forward and the backward pass, and the operands
// of the 8-bit linear layers (blocks along the channels for the forward and input-gradient products, blocks along the
// tokens for the weight gradient, 128 × 128 squares for weights, whose transpose has the same scales).
//
// Both directions move bytes, and the instructions spent on each decide how near they come to memory's rate.
// quantize_kernel: one CTA of 8 warps per 128 × 128 tile, which each warp reads 16 rows of with 128-bit loads, all in
// flight at once, and keeps in registers. The rows' largest magnitudes are found together: a butterfly in which each step
// halves the rows a lane still holds (8 shuffles for 16 rows instead of 32), after which a row's code is computed once
// and handed back with one shuffle. The row form is written from the registers. For the transposed form the tile goes
// through shared memory once, as stored. bf16 comes back through transposing matrix loads whose row addresses are chosen
// so that a lane receives 16 consecutive rows of one column (16 bytes of its line, four lanes a 64-byte run); a warp owns
// 16 whole columns, so their maxima need no further exchange. fp32 is read by columns: a warp owns 32 rows, a lane two
// neighbouring columns of them. Either way x is read once for both forms.
// One B200, bf16 (share of the copy rate, 6533 GB/s): 30,720 × 1536 to rows 23.7 µs (0.91), to both forms 38.0 (0.76), back
// 23.9 (0.91); at 17,280 rows 14.5, 20.4 and 13.7. Reading the tile by columns for the transposed bf16 form took 25.1
// instead of 20.4, a dequantising lane that owns 32 consecutive output bytes 19.3 instead of 13.7. Rows off the 16-byte grid
// (17,280 × 1531) to rows 20.6, to both forms 29.3, back 24: shifts, and sectors that two accesses share. fp32, 17,280 × 1536:
// to rows 31 (0.65), to both forms 38 (0.64), back 22 (0.92); its pieces are four values, and 64 KB of tile and the columns
// held in registers leave the transposed form three CTAs an SM.
#include <type_traits>

#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"
#include "sm100.cuh"
#include "unaligned.cuh"

namespace fvsr {

namespace {

using namespace sm100;

constexpr int kT = 128, kThreads = 256;
constexpr uint32_t kAbs = 0x7FFFFFFFu;

// Elements of T in a 16-byte load, as the pieces of a tile row a lane holds.
template <typename T>
struct Piece {
    static constexpr int kElems = 16 / (int)sizeof(T);
    static constexpr int kLanes = kT / kElems;              // lanes of a row
    static constexpr int kRowsPerLoad = 32 / kLanes;        // rows a warp covers with one load
    static constexpr int kLoads = 16 / kRowsPerLoad;        // loads for a warp's 16 rows
    using Held = std::conditional_t<sizeof(T) == 2, uint2, uint32_t>;  // the piece in 8 bits
};

__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {  // of |bf16| pairs, NaN above all
    uint32_t r;
    asm("{\n\t.reg .b32 t;\n\tabs.bf16x2 t, %2;\n\tmax.NaN.bf16x2 %0, %1, t;\n\t}" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// The largest magnitude of a piece, as fp32 bits (an integer maximum: a NaN's bits are above infinity's).
__device__ __forceinline__ uint32_t piece_max(const uint4& u, const __nv_bfloat16*) {
    const uint32_t a = max_abs2(max_abs2(max_abs2(max_abs2(0u, u.x), u.y), u.z), u.w);
    return max(a & 0xFFFF0000u, a << 16);
}
__device__ __forceinline__ uint32_t piece_max(const uint4& u, const float*) {
    return max(max(u.x & kAbs, u.y & kAbs), max(u.z & kAbs, u.w & kAbs));
}
// Four values, as two pairs already scaled, in e4m3.
__device__ __forceinline__ uint32_t pack4(uint64_t a, uint64_t b) {
    float x, y, z, w;
    uf2(a, x, y);
    uf2(b, z, w);
    return fp8_pack2(x, y) | (fp8_pack2(z, w) << 16);
}
__device__ __forceinline__ uint64_t bf_pair(uint32_t u) {
    float lo, hi;
    bf2_to_f(u, lo, hi);
    return f2(lo, hi);
}
__device__ __forceinline__ void put_piece(uint8_t* p, const uint4& u, uint64_t up, const __nv_bfloat16*) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack4(fmul2(bf_pair(u.x), up), fmul2(bf_pair(u.y), up)),
                                              pack4(fmul2(bf_pair(u.z), up), fmul2(bf_pair(u.w), up)));
}
__device__ __forceinline__ void put_piece(uint8_t* p, const uint4& u, uint64_t up, const float*) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&u);
    *reinterpret_cast<uint32_t*>(p) = pack4(fmul2(v.x, up), fmul2(v.y, up));
}

// Where the 16-byte word `w` of tile row r stands in shared memory. bf16: the words of the eight rows that one matrix
// load takes (equal but for bits 0, 4 and 5 of the row) lie in different banks.
template <typename T>
__device__ __forceinline__ int tile_word(int r, int w) {
    return r * Piece<T>::kLanes + (sizeof(T) == 2 ? w ^ ((r & 1) | (r >> 3 & 6)) : w);
}
// kVec: rows are 16-byte aligned and their lengths whole pieces; else bf16 from the one or two aligned words that hold the
// piece, fp32 (whose pieces are four elements) element by element.
template <typename T, bool kVec>
__device__ __forceinline__ uint4 load_piece(const T* p, int left) {
    if constexpr (kVec) {
        return left > 0 ? __ldcs(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
    } else if constexpr (sizeof(T) == 2) {
        const uint32_t off = reinterpret_cast<uintptr_t>(p) & 15;
        const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p) - off);
        const uint4 none = make_uint4(0, 0, 0, 0), a = left > 0 ? from[0] : none,
                    b = (int)off + min(left, 8) * 2 > 16 ? from[1] : none;
        uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, o[4];
        shift_bytes<2, 4>(w, off, o);
        if (left < 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = 2 * i + 1 < left ? o[i] : 2 * i < left ? o[i] & 0xFFFFu : 0u;
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    } else {
        alignas(16) T v[Piece<T>::kElems];
#pragma unroll
        for (int i = 0; i < Piece<T>::kElems; ++i) v[i] = i < left ? p[i] : T(0.0f);
        return *reinterpret_cast<const uint4*>(v);
    }
}

// The code of a line (form row); those beyond its last block, up to the end of the last tile of codes, are zero.
__device__ __forceinline__ void put_code(uint8_t* scale, int64_t line, int64_t block, int64_t blocks, uint32_t code) {
    uint8_t* p = scale + fp8_code_pos(line, block, (blocks + 3) >> 2);
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
    const uint32_t ct = (uint32_t)((cols + kT - 1) / kT);
    const uint32_t rb = blockIdx.x / ct, cb = blockIdx.x % ct;
    const int64_t r0 = (int64_t)rb * kT, c0 = (int64_t)cb * kT;
    const int nr = (int)min((int64_t)kT, rows - r0), nc = (int)min((int64_t)kT, cols - c0);  // of the tile
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane / P::kLanes, c = lane % P::kLanes * P::kElems, row = warp * 16 + sub;  // row of load 0
    griddep_wait_then_release();
    uint4 v[P::kLoads];
    const T* src = x + (r0 + row) * cols + c0 + c;
#pragma unroll
    for (int i = 0; i < P::kLoads; ++i)
        v[i] = load_piece<T, kVec>(src + (int64_t)(i * P::kRowsPerLoad) * cols, row + i * P::kRowsPerLoad < nr ? nc - c : 0);
    uint32_t top[P::kLoads];
#pragma unroll
    for (int i = 0; i < P::kLoads; ++i) {
        top[i] = piece_max(v[i], x);
        if (kTrans) tile4[tile_word<T>(row + i * P::kRowsPerLoad, lane % P::kLanes)] = v[i];
    }
    // After the butterfly the lanes 2i and 2i + 1 of a row's lanes hold the maximum of load i's row.
#pragma unroll
    for (int half = P::kLoads / 2, bit = P::kLanes / 2; half >= 1; half /= 2, bit /= 2) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const uint32_t keep = up ? top[i + half] : top[i], give = up ? top[i] : top[i + half];
            top[i] = max(keep, __shfl_xor_sync(0xffffffffu, give, bit));
        }
    }
    uint32_t most = max(top[0], __shfl_xor_sync(0xffffffffu, top[0], 1));
    if (square) {
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) warp_max[warp] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) most = max(most, warp_max[i]);
    }
    if (q) {
        const uint32_t code = fp8_code(most);
        const float up = fp8_up(code);
        const int64_t ld = (int64_t)ct * kT;
        uint8_t* dst = q + (r0 + row) * ld + c0 + c;
#pragma unroll
        for (int i = 0; i < P::kLoads; ++i) {
            const float u = __shfl_sync(0xffffffffu, up, (lane & ~(P::kLanes - 1)) | (2 * i));
            if (row + i * P::kRowsPerLoad < nr) put_piece(dst + (int64_t)(i * P::kRowsPerLoad) * ld, v[i], f2(u, u), x);
        }
        const int mine = row + (lane % P::kLanes >> 1) * P::kRowsPerLoad;
        if (!(lane & 1)) put_code(scale, r0 + mine, cb, ct, mine < nr ? code : 0u);
    }
    if constexpr (kTrans && sizeof(T) == 2) {
        __syncthreads();
        const int64_t rt = (rows + kT - 1) / kT, ld = rt * kT;
        // matrix 4h + m (h = which of a lane's row pairs 0..3 or 4..7, m of one load) has as its row 2j + e tile row
        // 16j + 2(4h + m) + e, so lane 4·col + j receives rows 16j .. 16j + 15 of its column over the eight matrices
        const int j2 = lane & 7, m = lane >> 3;
        const int src_row = 16 * (j2 >> 1) + 2 * m + (j2 & 1);
#pragma unroll
        for (int group = 0; group < 2; ++group) {
            const int w = warp * 2 + group, col = w * 8 + (lane >> 2);  // of the tile
            uint32_t u[2][8];  // [rows 0..63, 64..127][row pair]
            uint32_t most2 = 0;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t* d = u[half] + 4 * h;
                    const uint32_t at = smem_u32(tile4 + tile_word<T>(64 * half + src_row + 8 * h, w));
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                                 : "r"(at));
#pragma unroll
                    for (int i = 0; i < 4; ++i) most2 = max_abs2(most2, d[i]);
                }
            uint32_t top2 = max(most2 & 0xFFFF0000u, most2 << 16);
            top2 = max(top2, __shfl_xor_sync(0xffffffffu, top2, 1));
            top2 = max(top2, __shfl_xor_sync(0xffffffffu, top2, 2));
            const uint32_t code = fp8_code(square ? most : top2);
            const float f = fp8_up(code);
            const uint64_t up = f2(f, f);
            uint8_t* p = qt + (c0 + col) * ld + r0 + 16 * (lane & 3);
            if (col < nc) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[i] = pack4(fmul2(bf_pair(u[half][2 * i]), up), fmul2(bf_pair(u[half][2 * i + 1]), up));
                    *reinterpret_cast<uint4*>(p + 64 * half) = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
            if ((lane & 3) == 0) put_code(scale_t, c0 + col, rb, rt, col < nc ? code : 0u);
        }
    } else if constexpr (kTrans) {
        // lane: columns 2·cp, 2·cp + 1 of the 32 rows [32·quarter, +32)
        __syncthreads();
        const int quarter = warp & 3, cp = (warp >> 2) * 32 + lane;
        const int64_t rt = (rows + kT - 1) / kT, ld = rt * kT;
        const T* tile = reinterpret_cast<const T*>(tile4) + (quarter * 32) * kT + 2 * cp;
        uint32_t ma = 0, mb = 0;
        uint64_t w[32];  // a row's two columns
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            w[i] = *reinterpret_cast<const uint64_t*>(tile + i * kT);
            ma = max(ma, (uint32_t)w[i] & kAbs), mb = max(mb, (uint32_t)(w[i] >> 32) & kAbs);
        }
        if (square) {
            ma = mb = most;
        } else {
            *reinterpret_cast<uint2*>(&col_max[quarter][2 * cp]) = make_uint2(ma, mb);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint2 m = *reinterpret_cast<const uint2*>(&col_max[i][2 * cp]);
                ma = max(ma, m.x), mb = max(mb, m.y);
            }
        }
        const uint32_t code_a = fp8_code(ma), code_b = fp8_code(mb);
        const uint64_t up = f2(fp8_up(code_a), fp8_up(code_b));
        uint32_t a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float fa[4], fb[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) uf2(fmul2(w[4 * i + j], up), fa[j], fb[j]);
            a[i] = fp8_pack2(fa[0], fa[1]) | (fp8_pack2(fa[2], fa[3]) << 16);
            b[i] = fp8_pack2(fb[0], fb[1]) | (fp8_pack2(fb[2], fb[3]) << 16);
        }
        // Neighbouring lanes swap halves, so that one store of a warp fills whole 32-byte sectors: of the lines of the
        // even lane (then of the odd one) the even lane writes the first 16 bytes and the odd lane the rest.
        const bool odd = lane & 1;
        uint8_t* p = qt + (c0 + 2 * (cp & ~1)) * ld + r0 + quarter * 32 + (odd ? 16 : 0);
        auto put = [&](const uint32_t (&v)[8], int line) {
            uint32_t got[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) got[i] = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[4 + i], 1);
            const uint4 mine = odd ? make_uint4(v[4], v[5], v[6], v[7]) : make_uint4(v[0], v[1], v[2], v[3]);
            const uint4 theirs = make_uint4(got[0], got[1], got[2], got[3]);
            const int first = 2 * (cp & ~1) + line;  // in the tile: the even lane's line, and two further the odd lane's
            if (first < nc) *reinterpret_cast<uint4*>(p + line * ld) = odd ? theirs : mine;
            if (first + 2 < nc) *reinterpret_cast<uint4*>(p + (line + 2) * ld) = odd ? mine : theirs;
        };
        put(a, 0);
        put(b, 1);
        if (quarter == 0) {
            put_code(scale_t, c0 + 2 * cp, rb, rt, 2 * cp < nc ? code_a : 0u);
            put_code(scale_t, c0 + 2 * cp + 1, rb, rt, 2 * cp + 1 < nc ? code_b : 0u);
        }
    }
}

// A warp takes 512 columns of four rows: a lane 16 bytes' worth of output at a time, next to its neighbours', and the four
// codes of a row's tile as one word.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(int64_t rows, int64_t cols, const uint8_t* __restrict__ q,
                                                              const uint8_t* __restrict__ scale, T* __restrict__ out) {
    constexpr int kRows = 4, kElems = Piece<T>::kElems, kSteps = 512 / (32 * kElems);
    using Word = typename Piece<T>::Held;
    const int64_t ld = fp8_ld(cols);
    const uint32_t tiles = (uint32_t)fp8_scale_tiles(cols);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t it = (uint64_t)blockIdx.x * (kThreads / 32) + warp;
    const int64_t tile = it % tiles, r0 = it / tiles * kRows, c = tile * 512 + lane * kElems;
    const int here = (int)min((int64_t)kRows, rows - r0), left = (int)min(cols - tile * 512, (int64_t)512) - lane * kElems;
    griddep_wait_then_release();
    Word v[kRows][kSteps];
    uint32_t word[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint8_t* p = q + (r0 + i) * ld + c;
        word[i] = i < here ? *reinterpret_cast<const uint32_t*>(scale + fp8_code_pos(r0 + i, tile * 4, tiles)) : 0u;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            v[i][j] = Word{};
            if (i < here && j * 32 * kElems < left) v[i][j] = __ldcs(reinterpret_cast<const Word*>(p + j * 32 * kElems));
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (i >= here) break;
        T* p = out + (r0 + i) * cols + c;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            const int at = j * 32 * kElems;
            if (at >= left + (kVec ? 0 : lane * kElems)) break;  // else the whole warp's
            const int block = (lane * kElems + at) >> 7;
            const float down = fp8_down((word[i] >> (8 * block)) & 255u);
            const uint32_t w[2] = {reinterpret_cast<const uint32_t*>(&v[i][j])[0],
                                   kElems == 8 ? reinterpret_cast<const uint32_t*>(&v[i][j])[kElems == 8] : 0u};
            float f[kElems];
#pragma unroll
            for (int e = 0; e < kElems; e += 2) {
                fp8_unpack2(w[e >> 2] >> (16 * ((e >> 1) & 1)), f[e], f[e + 1]);
                f[e] *= down, f[e + 1] *= down;
            }
            if constexpr (kVec && kElems == 8) {
                *reinterpret_cast<uint4*>(p + at) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                                               pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
            } else if constexpr (kVec) {
                *reinterpret_cast<float4*>(p + at) = make_float4(f[0], f[1], f[2], f[3]);
            } else {
                uint32_t u[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    u[e] = kElems == 8 ? pack_bf16x2(f[(2 * e) % kElems], f[(2 * e + 1) % kElems]) : __float_as_uint(f[e % kElems]);
                store_unaligned<T, 4>(p - lane * kElems + at, min(32 * kElems, left + lane * kElems - at), u);
            }
        }
    }
}

// A thread takes one row's four codes of a tile.
__global__ void __launch_bounds__(kThreads) codes_kernel(int64_t rows, int64_t blocks, const uint8_t* __restrict__ scale,
                                                         uint8_t* __restrict__ out) {
    griddep_wait_then_release();
    const int64_t tiles = (blocks + 3) >> 2, items = rows * tiles;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < items; i += (int64_t)gridDim.x * kThreads) {
        const int64_t r = i / tiles, b = i % tiles * 4;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(scale + fp8_code_pos(r, b, tiles));
        for (int j = 0; j < 4 && b + j < blocks; ++j) out[r * blocks + b + j] = (uint8_t)(w >> (8 * j));
    }
}

template <typename T, bool kVec, bool kTrans>
cudaError_t quantize(int64_t rows, int64_t cols, const T* x, bool square, uint8_t* q, uint8_t* scale, uint8_t* qt,
                     uint8_t* scale_t, cudaStream_t st) {
    constexpr auto kernel = quantize_kernel<T, kVec, kTrans>;
    const size_t smem = kTrans ? sizeof(T) * kT * kT : 0;
    if (smem > 48 * 1024) {
        cudaError_t e = allow_smem<kernel>(smem);
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
    const int64_t items = (rows + 3) / 4 * fp8_scale_tiles(cols);
    const dim3 grid((unsigned)((items + 7) / 8));
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

cudaError_t launch_fp8_codes(int64_t rows, int64_t cols, const uint8_t* scale, uint8_t* out, cudaStream_t st) {
    const int64_t need = (rows * fp8_scale_tiles(cols) + kThreads - 1) / kThreads, most = (int64_t)sm_count() * 8;
    return launch_pdl(codes_kernel, dim3((unsigned)(need < most ? need : most)), dim3(kThreads), 0, st, rows,
                      (cols + 127) / 128, scale, out);
}

cudaError_t launch_dequantize_fp8(int64_t rows, int64_t cols, const uint8_t* q, const uint8_t* scale, void* out,
                                  int dtype, cudaStream_t st) {
    return dtype == FVSR_BF16 ? dequantize_t(rows, cols, q, scale, static_cast<__nv_bfloat16*>(out), st)
                              : dequantize_t(rows, cols, q, scale, static_cast<float*>(out), st);
}

}  // namespace fvsr
