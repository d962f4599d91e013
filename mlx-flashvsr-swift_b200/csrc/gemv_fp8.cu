// gemv_fp8.cu — the linear layers on 8-bit operands for a few tokens (M up to 16: the time embedding's layers, a single
// token), out = epilogue(x · wᵀ + bias) in one launch without a workspace; x in the 8-bit form or bf16, quantised here.
//
// Bound by reading w once (N·K bytes) and by latency. A CTA takes 16 rows of w (output columns) and its warps the blocks
// of 128 along K in turn; w streams from memory straight into registers, the next block's loads in flight under this
// one's arithmetic. e4m3 values are fp16 values, so they are multiplied exactly on fp16 tensor-core instructions
// (m16n8k16: 16 rows of w against 8 tokens, fp32 sums); which of a block's 128 positions an instruction's k index means
// does not matter as long as both operands agree, so a lane reads 16 consecutive bytes of a row and uses them as they
// come. Each block's sum is scaled by its two powers of two and added in fp32; the warps' sums are added in order.
// One B200, from bf16: 1 × 9216 × 1536 6.8 µs, 16 tokens 9.2 (17 tokens on the tiled kernel: 7.7 from 8-bit x, and 2 to
// quantise it); 1 × 1536 × 1536 3.4, 16 tokens 5.0 (17: 7.5 and 2). Hence the limit of 16.
#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"
#include "fp8_epilogue.cuh"
#include "sm100.cuh"

namespace fvsr {

namespace {

using namespace sm100;

constexpr int kRows = 16;  // of w per CTA

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four e4m3 values as two fp16 pairs.
__device__ __forceinline__ void to_f16(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
}

// A lane's 32 values of a block: 16 from position 16·(lane % 4) and 16 from 64 further, in 8 bits.
struct Held {
    uint4 u[2];
    __device__ __forceinline__ uint32_t word(int i) const {
        const uint4& v = u[i >> 2];
        return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
    }
};

// 2^(code − 127) in two factors near its root (NaN for code 255): the scales of two blocks may meet beyond fp32's range on
// either side (2^118 · 2^-118) while what they scale is within it. lo and hi of two codes are multiplied apart, the sum of
// the products then by each: every step is exact unless the result itself is not. (Sum · 2^(code − 127) · 2^(code' − 127)
// was infinite there.)
struct Scale {
    float lo, hi;
};
__device__ __forceinline__ Scale scale_of(uint32_t code) {
    const uint32_t half = code >> 1;
    return {__uint_as_float(code == 255u ? 0x7FC00000u : (half + 63u) << 23), __uint_as_float((code - half + 64u) << 23)};
}
__device__ __forceinline__ Scale operator*(const Scale& a, const Scale& b) { return {a.lo * b.lo, a.hi * b.hi}; }

// x as bf16: the block of token row `x` (K values) quantised by the four lanes that share it. left: values of the row
// from the lane's first on. kVec: 16-byte aligned rows of whole eights.
template <bool kVec>
__device__ __forceinline__ Held quantize_block(const __nv_bfloat16* x, int left, uint32_t& code) {
    float f[32];
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < 4; ++h) {  // eight values each, at 0, 8, 64 and 72
        const int at = (h & 1) * 8 + (h >> 1) * 64;
        if constexpr (kVec) {
            const uint4 u = at < left ? *reinterpret_cast<const uint4*>(x + at) : make_uint4(0, 0, 0, 0);
            bf2_to_f(u.x, f[8 * h], f[8 * h + 1]), bf2_to_f(u.y, f[8 * h + 2], f[8 * h + 3]);
            bf2_to_f(u.z, f[8 * h + 4], f[8 * h + 5]), bf2_to_f(u.w, f[8 * h + 6], f[8 * h + 7]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[8 * h + e] = at + e < left ? __bfloat162float(x[at + e]) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[8 * h + e]) & 0x7FFFFFFFu);
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    code = fp8_code(top);
    const float up = fp8_up(code);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        w[i] = fp8_pack2(f[4 * i] * up, f[4 * i + 1] * up) | (fp8_pack2(f[4 * i + 2] * up, f[4 * i + 3] * up) << 16);
    Held h;
    h.u[0] = make_uint4(w[0], w[1], w[2], w[3]);
    h.u[1] = make_uint4(w[4], w[5], w[6], w[7]);
    return h;
}

// kTokens: 8 or 16. kX: 0 = x in 8 bits, 1 = bf16 with 16-byte rows, 2 = bf16.
template <typename T, int kMode, int kTokens, int kX>
__global__ void __launch_bounds__(512) gemv_fp8_kernel(const Fp8GemmArgs a, const __nv_bfloat16* __restrict__ xb) {
    constexpr int kG = kTokens / 8;
    __shared__ float sums[16][kG][4][32];
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int n0 = blockIdx.x * kRows, kt = (a.K + 127) >> 7;
    const int64_t ld = fp8_ld(a.K), tiles = fp8_scale_tiles(a.K);
    // rows and tokens beyond the tensors' ends read the last one's; nothing of them is stored
    const int64_t row0 = min(n0 + g, a.N - 1), row1 = min(n0 + g + 8, a.N - 1);
    const uint8_t *w0 = a.w + row0 * ld + q * 16, *w1 = a.w + row1 * ld + q * 16;
    const int64_t code0 = fp8_code_pos(row0, 0, tiles), code1 = fp8_code_pos(row1, 0, tiles);
    auto code_at = [](int kb) { return (int64_t)(kb >> 2) * 512 + (kb & 3); };
    Held wa, wb;
    uint32_t ca, cb;
    auto fetch = [&](int kb) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            wa.u[h] = __ldcs(reinterpret_cast<const uint4*>(w0 + (int64_t)kb * 128 + 64 * h));
            wb.u[h] = __ldcs(reinterpret_cast<const uint4*>(w1 + (int64_t)kb * 128 + 64 * h));
        }
        ca = a.w_scale[code0 + code_at(kb)];
        cb = a.w_scale[code1 + code_at(kb)];
    };
    float acc[kG][4] = {};
    griddep_wait_then_release();
    if (warp < kt) fetch(warp);
    for (int kb = warp; kb < kt; kb += warps) {
        const Held now_a = wa, now_b = wb;
        const Scale scale_a = scale_of(ca), scale_b = scale_of(cb);
        if (kb + warps < kt) fetch(kb + warps);
        Held xs[kG];
        uint32_t code_x[kG];
#pragma unroll
        for (int t = 0; t < kG; ++t) {
            const int64_t token = min(8 * t + g, a.M - 1);
            if constexpr (kX == 0) {
                const uint8_t* p = a.x + token * ld + (int64_t)kb * 128 + q * 16;
                xs[t].u[0] = *reinterpret_cast<const uint4*>(p);
                xs[t].u[1] = *reinterpret_cast<const uint4*>(p + 64);
                code_x[t] = a.x_scale[fp8_code_pos(token, kb, tiles)];
            } else {
                const int at = kb * 128 + q * 16;
                xs[t] = quantize_block<kX == 1>(xb + token * a.K + at, a.K - at, code_x[t]);
            }
        }
        // of part, whose rows are g, g + 8 of w, tokens 2q, 2q + 1; a token's code is in lanes 4·token…
        Scale factor[kG][4];
        auto scale_factors = [&] {
#pragma unroll
            for (int t = 0; t < kG; ++t) {
                const Scale x0 = scale_of(__shfl_sync(0xffffffffu, code_x[t], 8 * q)),
                            x1 = scale_of(__shfl_sync(0xffffffffu, code_x[t], 8 * q + 4));
                factor[t][0] = scale_a * x0, factor[t][1] = scale_a * x1;
                factor[t][2] = scale_b * x0, factor[t][3] = scale_b * x1;
            }
        };
        // ahead of the products (behind them 1 x 1536 x 1536 from 8 bits took 2.97 instead of 2.67 µs), but for up to eight
        // bf16 tokens, whose quantising is what the products wait for (3.39, ahead 3.55)
        constexpr bool kAhead = kX == 0 || kG == 2;
        if (kAhead) scale_factors();
        float part[kG][4] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t a0, a1, a2, a3;
            to_f16(now_a.word(i), a0, a2);
            to_f16(now_b.word(i), a1, a3);
#pragma unroll
            for (int t = 0; t < kG; ++t) {
                uint32_t b0, b1;
                to_f16(xs[t].word(i), b0, b1);
                mma_f16(part[t], a0, a1, a2, a3, b0, b1);
            }
        }
        if (!kAhead) scale_factors();
#pragma unroll
        for (int t = 0; t < kG; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] += part[t][i] * factor[t][i].lo * factor[t][i].hi;
    }
#pragma unroll
    for (int t = 0; t < kG; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[warp][t][i][lane] = acc[t][i];
    __syncthreads();
    for (int o = threadIdx.x; o < kRows * kTokens; o += blockDim.x) {
        const int r = o & 15, token = o >> 4, n = n0 + r;
        if (token >= a.M || n >= a.N) continue;
        const int t = token >> 3, i = (r >> 3) * 2 + (token & 1), from = (r & 7) * 4 + ((token & 7) >> 1);
        float s = 0.0f;
        for (int w = 0; w < warps; ++w) s += sums[w][t][i][from];
        const int64_t at = (int64_t)token * a.N + n;
        const float bias = a.bias ? __bfloat162float(a.bias[n]) : 0.0f;
        float gate = 0.0f, add = 0.0f, y, unused;
        if (kMode == FVSR_LINEAR_GATED_RESIDUAL)
            gate = __bfloat162float(a.gate[n]), add = load_as_float(static_cast<const T*>(a.resid) + at);
        uf2(finish2<kMode, kMode == FVSR_LINEAR_GATED_RESIDUAL>(f2(s, s), f2(bias, bias), f2(gate, gate), f2(add, add), true, true), y, unused);
        store_from_float(static_cast<T*>(a.out) + at, y);
    }
}

template <typename T, int kMode, int kTokens>
cudaError_t launch_x(const Fp8GemmArgs& a, const __nv_bfloat16* xb, dim3 grid, dim3 block, cudaStream_t st) {
    if (!xb) return launch_pdl(gemv_fp8_kernel<T, kMode, kTokens, 0>, grid, block, 0, st, a, xb);
    if (a.K % 8 == 0) return launch_pdl(gemv_fp8_kernel<T, kMode, kTokens, 1>, grid, block, 0, st, a, xb);
    return launch_pdl(gemv_fp8_kernel<T, kMode, kTokens, 2>, grid, block, 0, st, a, xb);
}

template <typename T, int kMode>
cudaError_t launch_tokens(const Fp8GemmArgs& a, const __nv_bfloat16* xb, dim3 grid, dim3 block, cudaStream_t st) {
    return a.M <= 8 ? launch_x<T, kMode, 8>(a, xb, grid, block, st) : launch_x<T, kMode, 16>(a, xb, grid, block, st);
}

template <typename T>
cudaError_t launch_mode(const Fp8GemmArgs& a, const __nv_bfloat16* xb, dim3 grid, dim3 block, cudaStream_t st) {
    switch (a.mode) {
        case FVSR_LINEAR: return launch_tokens<T, FVSR_LINEAR>(a, xb, grid, block, st);
        case FVSR_LINEAR_GELU: return launch_tokens<T, FVSR_LINEAR_GELU>(a, xb, grid, block, st);
        default: return launch_tokens<T, FVSR_LINEAR_GATED_RESIDUAL>(a, xb, grid, block, st);
    }
}

}  // namespace

cudaError_t launch_gemv_fp8(const Fp8GemmArgs& a, const __nv_bfloat16* xb, cudaStream_t st) {
    // a warp for every three blocks along K, 4 to 16 of them
    const int kt = (a.K + 127) / 128, warps = kt <= 12 ? 4 : kt <= 24 ? 8 : 16;
    const dim3 grid((a.N + kRows - 1) / kRows), block(32 * warps);
    return a.out_dtype == FVSR_BF16 ? launch_mode<__nv_bfloat16>(a, xb, grid, block, st)
                                    : launch_mode<float>(a, xb, grid, block, st);
}

}  // namespace fvsr
