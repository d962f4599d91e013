// norm_train.cu — LayerNorm over the channels for training: the forward pass that keeps each row's mean and
// rstd = 1/√(var + eps), and the backward pass with the gradients of its vectors.
//   n = (x − mean)·rstd,  y = (n·w + b)·(1 + scale) + shift          (w, b and shift, scale each optional)
//   g = dy·(1 + scale)·w, dx = rstd·(g − mean_c(g) − n·mean_c(g·n))
//   A = Σ_rows dy·n, B = Σ_rows dy: dw = (1 + scale)·A, db = (1 + scale)·B, dscale = w·A + b·B, dshift = B.
// fp32 throughout, one rounding of y and dx to the tensors' type.
//
// Both passes are bound by memory, x (and dy) read once and the result written once. A thread owns eight neighbouring
// channels of every row it meets, so the vectors, and in the backward pass the sums A and B of those channels, stay in
// its registers over all rows: tpr = ⌈c / 8⌉ threads, in whole warps, work on a row, kRows rows at once to share a
// barrier, and the loads of the next kRows rows are in flight meanwhile. Narrow rows put several such groups in a CTA.
// The variance is taken about the mean in a second pass over the registers. The vectors' gradients are summed per group
// over its rows, then over the groups by a second kernel, both in a fixed order, so they do not depend on timing.
#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"
#include "sm100.cuh"

namespace fvsr {

namespace {

using sm100::bf2_to_f;
using sm100::pack_bf16x2;

// Eight values of a row as loaded: 16 bytes of bf16, 32 of fp32.
template <typename T>
struct Raw8 {
    uint4 u[sizeof(T) / 2];
};

// Whole and 16-byte aligned (kVec), or element by element with zeros beyond n values.
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* p, int n, Raw8<T>& r) {
    if (kVec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
        alignas(16) T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : T(0.0f);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(v)[i];
    }
}
__device__ __forceinline__ void as_floats(const Raw8<__nv_bfloat16>& r, float (&f)[8]) {
    bf2_to_f(r.u[0].x, f[0], f[1]), bf2_to_f(r.u[0].y, f[2], f[3]);
    bf2_to_f(r.u[0].z, f[4], f[5]), bf2_to_f(r.u[0].w, f[6], f[7]);
}
__device__ __forceinline__ void as_floats(const Raw8<float>& r, float (&f)[8]) {
    f[0] = __uint_as_float(r.u[0].x), f[1] = __uint_as_float(r.u[0].y);
    f[2] = __uint_as_float(r.u[0].z), f[3] = __uint_as_float(r.u[0].w);
    f[4] = __uint_as_float(r.u[1].x), f[5] = __uint_as_float(r.u[1].y);
    f[6] = __uint_as_float(r.u[1].z), f[7] = __uint_as_float(r.u[1].w);
}
template <bool kVec>
__device__ __forceinline__ void store8(__nv_bfloat16* p, int n, const float (&f)[8]) {
    if (kVec) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                                  pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = __float2bfloat16_rn(f[i]);
    }
}
template <bool kVec>
__device__ __forceinline__ void store8(float* p, int n, const float (&f)[8]) {
    if (kVec) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = f[i];
    }
}

template <typename T>
__device__ __forceinline__ float vec_or(const void* v, int c, float otherwise) {
    return v ? load_as_float(static_cast<const T*>(v) + c) : otherwise;
}

// The sums of v[0..N) over the tpr threads of a row group, in each of them: shuffles, then the warps' sums through
// `part` ([32 warps][N]) and a barrier of the CTA (every thread calls this the same number of times; two calls in a row
// use different buffers). In the order of the warps.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* part, int group_warp0, int warps) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (warps == 1) return;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) part[(threadIdx.x >> 5) * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.0f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += part[(group_warp0 + w) * N + i];
}

template <typename T, bool kVec, int kRows, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) norm_train_kernel(const NormTrainArgs a, int tpr) {
    __shared__ alignas(16) float part[2][32 * kRows];
    const int groups = (int)blockDim.x / tpr, g = (int)threadIdx.x / tpr, col = ((int)threadIdx.x % tpr) * 8;
    const int n = max(0, min(8, a.c - col)), warps = tpr >> 5, warp0 = g * warps;
    const int64_t step = (int64_t)gridDim.x * groups * kRows;
    const float inv_c = 1.0f / (float)a.c;
    const T* x = static_cast<const T*>(a.x);
    T* out = static_cast<T*>(a.out);
    griddep_wait_then_release();
    float gain[8], base[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = col + (i < n ? i : 0);
        const float s1 = n > 0 ? 1.0f + vec_or<T>(a.scale, c, 0.0f) : 0.0f;
        gain[i] = n > 0 ? s1 * vec_or<T>(a.weight, c, 1.0f) : 0.0f;
        base[i] = n > 0 ? fmaf(vec_or<T>(a.bias, c, 0.0f), s1, vec_or<T>(a.shift, c, 0.0f)) : 0.0f;
    }
    Raw8<T> next[kRows];
    auto fetch = [&](int64_t row0) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            next[i] = Raw8<T>{};
            if (row0 + i < a.m && n > 0) load8<T, kVec>(x + (row0 + i) * a.c + col, n, next[i]);
        }
    };
    int64_t row0 = ((int64_t)blockIdx.x * groups + g) * kRows;
    fetch(row0);
    for (int64_t cta0 = (int64_t)blockIdx.x * groups * kRows; cta0 < a.m; cta0 += step, row0 += step) {
        Raw8<T> now[kRows];
        float sum[kRows], sq[kRows], f[8];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            now[i] = next[i];
            as_floats(now[i], f);
            sum[i] = ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
        }
        fetch(row0 + step);
        group_sum<kRows>(sum, part[0], warp0, warps);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            sum[i] *= inv_c;
            as_floats(now[i], f);
            sq[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = f[j] - sum[i];
                if (kVec ? n > 0 : j < n) sq[i] = fmaf(d, d, sq[i]);
            }
        }
        group_sum<kRows>(sq, part[1], warp0, warps);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (row0 + i >= a.m) break;
            const float rstd = 1.0f / sqrtf(fmaf(sq[i], inv_c, a.eps));
            if (col == 0) a.mean[row0 + i] = sum[i], a.rstd[row0 + i] = rstd;
            if (n == 0) continue;
            as_floats(now[i], f);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = fmaf((f[j] - sum[i]) * rstd, gain[j], base[j]);
            store8<kVec>(out + (row0 + i) * a.c + col, n, f);
        }
    }
}

// kHeld: x is the 8-bit form.
template <typename T, bool kHeld, bool kVec, int kRows, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) norm_backward_kernel(const NormTrainArgs a, int tpr) {
    __shared__ alignas(16) float part[2][32 * 2 * kRows];
    const int groups = (int)blockDim.x / tpr, g = (int)threadIdx.x / tpr, col = ((int)threadIdx.x % tpr) * 8;
    const int n = max(0, min(8, a.c - col)), warps = tpr >> 5, warp0 = g * warps;
    const int64_t step = (int64_t)gridDim.x * groups * kRows, ld = fp8_ld(a.c), tiles = fp8_scale_tiles(a.c);
    const float inv_c = 1.0f / (float)a.c;
    const T *x = static_cast<const T*>(a.x), *dy = static_cast<const T*>(a.dy);
    const uint8_t* x8 = static_cast<const uint8_t*>(a.x);
    T* dx = static_cast<T*>(a.out);
    griddep_wait_then_release();
    float gain[8], sum_a[8], sum_b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = col + (i < n ? i : 0);
        gain[i] = n > 0 ? (1.0f + vec_or<T>(a.scale, c, 0.0f)) * vec_or<T>(a.weight, c, 1.0f) : 0.0f;
        sum_a[i] = sum_b[i] = 0.0f;
    }
    Raw8<T> next_dy[kRows], next_x[kHeld ? 1 : kRows];
    uint2 next_x8[kHeld ? kRows : 1];
    uint32_t next_code[kHeld ? kRows : 1];
    float next_mean[kRows], next_rstd[kRows];
    auto fetch = [&](int64_t row0) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int64_t r = row0 + i;
            const bool here = r < a.m && n > 0;
            next_dy[i] = Raw8<T>{};
            if (here) load8<T, kVec>(dy + r * a.c + col, n, next_dy[i]);
            if constexpr (kHeld) {
                next_x8[i] = here ? *reinterpret_cast<const uint2*>(x8 + r * ld + col) : make_uint2(0, 0);
                next_code[i] = here ? a.x_scale[fp8_code_pos(r, col >> 7, tiles)] : 0u;
            } else {
                next_x[i] = Raw8<T>{};
                if (here) load8<T, kVec>(x + r * a.c + col, n, next_x[i]);
            }
            next_mean[i] = here ? a.mean[r] : 0.0f;
            next_rstd[i] = here ? a.rstd[r] : 0.0f;
        }
    };
    int64_t row0 = ((int64_t)blockIdx.x * groups + g) * kRows;
    fetch(row0);
    int flip = 0;
    for (int64_t cta0 = (int64_t)blockIdx.x * groups * kRows; cta0 < a.m; cta0 += step, row0 += step, flip ^= 1) {
        float norm[kRows][8], grad[kRows][8], rstd[kRows], s[2 * kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            rstd[i] = next_rstd[i];
            as_floats(next_dy[i], grad[i]);
            if constexpr (kHeld) {
                const float down = fp8_down(next_code[i]);
                fp8_unpack2(next_x8[i].x, norm[i][0], norm[i][1]);
                fp8_unpack2(next_x8[i].x >> 16, norm[i][2], norm[i][3]);
                fp8_unpack2(next_x8[i].y, norm[i][4], norm[i][5]);
                fp8_unpack2(next_x8[i].y >> 16, norm[i][6], norm[i][7]);
#pragma unroll
                for (int j = 0; j < 8; ++j) norm[i][j] *= down;
            } else {
                as_floats(next_x[i], norm[i]);
            }
            s[2 * i] = s[2 * i + 1] = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                norm[i][j] = (norm[i][j] - next_mean[i]) * rstd[i];
                sum_a[j] = fmaf(grad[i][j], norm[i][j], sum_a[j]);
                sum_b[j] += grad[i][j];
                grad[i][j] *= gain[j];
                s[2 * i] += grad[i][j];
                s[2 * i + 1] = fmaf(grad[i][j], norm[i][j], s[2 * i + 1]);
            }
        }
        fetch(row0 + step);
        group_sum<2 * kRows>(s, part[flip], warp0, warps);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (row0 + i >= a.m || n == 0) break;
            const float c1 = s[2 * i] * inv_c, c2 = s[2 * i + 1] * inv_c;
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = rstd[i] * (grad[i][j] - c1 - norm[i][j] * c2);
            store8<kVec>(dx + (row0 + i) * a.c + col, n, f);
        }
    }
    float* mine = a.partial + ((int64_t)blockIdx.x * groups + g) * 2 * a.c + col;
    for (int i = 0; i < n; ++i) mine[i] = sum_a[i], mine[a.c + i] = sum_b[i];
}

// The groups' sums of 32 channels: 32 rows of threads take every 32nd group each, then their sums in order.
template <typename T>
__global__ void __launch_bounds__(1024) norm_vectors_kernel(const NormTrainArgs a, int groups) {
    __shared__ float sa[32][33], sb[32][33];
    griddep_wait_then_release();
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, c = blockIdx.x * 32 + tx;
    float va = 0.0f, vb = 0.0f;
    if (c < a.c) {
#pragma unroll 4
        for (int i = ty; i < groups; i += 32) {
            va += a.partial[(int64_t)i * 2 * a.c + c];
            vb += a.partial[((int64_t)i * 2 + 1) * a.c + c];
        }
    }
    sa[ty][tx] = va, sb[ty][tx] = vb;
    __syncthreads();
    if (ty != 0 || c >= a.c) return;
    va = vb = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) va += sa[i][tx], vb += sb[i][tx];
    const float s1 = 1.0f + vec_or<T>(a.scale, c, 0.0f);
    if (a.dweight) a.dweight[c] = s1 * va;
    if (a.dbias) a.dbias[c] = s1 * vb;
    if (a.dscale) a.dscale[c] = fmaf(vec_or<T>(a.weight, c, 1.0f), va, vec_or<T>(a.bias, c, 0.0f) * vb);
    if (a.dshift) a.dshift[c] = vb;
}

int sm_count() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        n = 148;
    return n;
}

// Threads of a row and of a CTA for c channels, and how many CTAs fit an SM at `regs` registers a thread.
struct Shape {
    int tpr, threads, groups;
    explicit Shape(int c) : tpr(((c + 7) / 8 + 31) / 32 * 32), groups(tpr >= 256 ? 1 : 256 / tpr) { threads = tpr * groups; }
    int per_sm(int regs) const { const int n = 65536 / regs / threads; return n < 1 ? 1 : n; }
};
int ctas_for(int64_t m, const Shape& s, int rows, int regs) {
    const int64_t need = (m + s.groups * rows - 1) / (s.groups * rows), most = (int64_t)sm_count() * s.per_sm(regs);
    return (int)(need < most ? need : most);
}
// Rows at once: forward four of bf16, two of fp32, backward two; one where 1024 threads leave 64 registers each.
constexpr int kWideC = 4096, kBackwardRows = 2;

template <typename T, bool kVec>
cudaError_t train(const NormTrainArgs& a, cudaStream_t st) {
    constexpr int kRows = sizeof(T) == 2 ? 4 : 2;
    const Shape s(a.c);
    const dim3 grid(ctas_for(a.m, s, a.c > kWideC ? 1 : kRows, 64)), block(s.threads);
    if (a.c > kWideC) return launch_pdl(norm_train_kernel<T, kVec, 1, 1024>, grid, block, 0, st, a, s.tpr);
    return launch_pdl(norm_train_kernel<T, kVec, kRows, 512>, grid, block, 0, st, a, s.tpr);
}

template <typename T, bool kHeld, bool kVec>
cudaError_t backward_rows(const NormTrainArgs& a, const Shape& s, int ctas, cudaStream_t st) {
    constexpr int kRows = kBackwardRows;
    const dim3 grid(ctas), block(s.threads);
    if (a.c > kWideC) return launch_pdl(norm_backward_kernel<T, kHeld, kVec, 1, 1024>, grid, block, 0, st, a, s.tpr);
    return launch_pdl(norm_backward_kernel<T, kHeld, kVec, kRows, 512>, grid, block, 0, st, a, s.tpr);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
cudaError_t backward(const NormTrainArgs& a, cudaStream_t st) {
    const Shape s(a.c);
    const int groups = (int)norm_backward_groups(a.m, a.c), ctas = groups / s.groups;
    cudaError_t e = cudaSuccess;
    if (ctas > 0) {
        const bool vec = a.c % 8 == 0 && aligned16(a.dy) && aligned16(a.out) && aligned16(a.x);
        if (a.x_scale)
            e = vec ? backward_rows<T, true, true>(a, s, ctas, st) : backward_rows<T, true, false>(a, s, ctas, st);
        else
            e = vec ? backward_rows<T, false, true>(a, s, ctas, st) : backward_rows<T, false, false>(a, s, ctas, st);
    }
    if (e != cudaSuccess || !(a.dweight || a.dbias || a.dscale || a.dshift)) return e;
    return launch_pdl(norm_vectors_kernel<T>, dim3((a.c + 31) / 32), dim3(1024), 0, st, a, groups);
}

}  // namespace

int64_t norm_backward_groups(int64_t m, int c) {
    const Shape s(c);
    return (int64_t)ctas_for(m, s, c > kWideC ? 1 : kBackwardRows, 128) * s.groups;
}

cudaError_t launch_layernorm_train(const NormTrainArgs& a, cudaStream_t st) {
    if (a.m <= 0) return cudaSuccess;
    const bool vec = a.c % 8 == 0 && aligned16(a.x) && aligned16(a.out);
    if (a.dtype == FVSR_BF16) return vec ? train<__nv_bfloat16, true>(a, st) : train<__nv_bfloat16, false>(a, st);
    return vec ? train<float, true>(a, st) : train<float, false>(a, st);
}

cudaError_t launch_layernorm_backward(const NormTrainArgs& a, cudaStream_t st) {
    return a.dtype == FVSR_BF16 ? backward<__nv_bfloat16>(a, st) : backward<float>(a, st);
}

}  // namespace fvsr
