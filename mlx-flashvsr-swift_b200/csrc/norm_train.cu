// norm_train.cu — LayerNorm over the channels for training: the forward pass that keeps each row's mean and
// rstd = 1/√(var + eps), and the backward pass with the gradients of its vectors.
//   n = (x − mean)·rstd,  y = (n·w + b)·(1 + scale) + shift          (w, b and shift, scale each optional)
//   g = dy·(1 + scale)·w, dx = rstd·(g − mean_c(g) − n·mean_c(g·n))
//   A = Σ_rows dy·n, B = Σ_rows dy: dw = (1 + scale)·A, db = (1 + scale)·B, dscale = w·A + b·B, dshift = B.
// fp32 throughout, one rounding of y and dx to the tensors' type.
//
// Both passes are bound by memory, x (and dy) read once and the result written once. A thread owns eight neighbouring
// channels (or twice eight) of every row it meets, so the vectors, and in the backward pass the sums A and B of those channels, stay in
// its registers over all rows: tpr = ⌈c / 8⌉ threads, in whole warps, work on a row, kRows rows at once to share a
// barrier; narrow rows put several such groups in a CTA. Rows are copied ahead into shared memory with cp.async, each
// thread its own pieces (so that no barrier guards them), kStages sets of rows deep: what is in flight costs no
// registers. Arithmetic is on pairs (f32x2), without which the backward pass would be bound by issue slots. The variance
// is taken about the mean in a second pass over the pieces. The vectors' gradients are summed per CTA over its rows,
// then over the CTAs by a second kernel, both in a fixed order, so they do not depend on timing.
// One B200, bf16 (share of the copy rate, 6533 GB/s): 17,280 × 1536 forward 22 µs (0.74), backward 37 (0.66), from the 8-bit
// form 40; 30,720 × 1536 34 (0.85), 55 (0.78) and 60; 4096 × 8192 27, 54 and 56. What keeps the backward pass from
// memory's rate is instructions: 152 for a thread's eight values of a row (194 from 8 bits).
#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"
#include "sm100.cuh"
#include "unaligned.cuh"

namespace fvsr {

namespace {

using namespace sm100;

// Asynchronous copies of 16 or 8 bytes, or as many zeros without a source (here false: src is not read).
__device__ __forceinline__ void copy_async16(void* dst, const void* src, bool here) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(here ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_async8(void* dst, const void* src, bool here) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(here ? 8 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

__device__ __forceinline__ uint64_t bf_pair(uint32_t u) {
    float lo, hi;
    bf2_to_f(u, lo, hi);
    return f2(lo, hi);
}
__device__ __forceinline__ float pair_sum(uint64_t v) {
    float lo, hi;
    uf2(v, lo, hi);
    return lo + hi;
}
__device__ __forceinline__ void to_regs(const uint4& u, uint32_t* v) { v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w; }
// Zeros from value n on.
__device__ __forceinline__ void clear_from(int n, uint64_t (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float lo, hi;
        uf2(f[i], lo, hi);
        f[i] = f2(2 * i < n ? lo : 0.0f, 2 * i + 1 < n ? hi : 0.0f);
    }
}

// Eight values of a row as stored: 16 bytes of bf16, 32 of fp32. In shared memory the pieces of kThreads threads take
// kStride 16-byte words: if rows are 16-byte aligned and c a whole number of pieces (kVec), a piece's words are split,
// [word][thread], so that a warp's accesses are contiguous; else each warp has its stretch of the row as the aligned words
// that cover it, one more than its pieces have.
template <typename T, bool kVec, int kThreads>
struct Piece {
    static constexpr int kWords = (int)sizeof(T) / 2, kRegs = kWords * 4;
    static constexpr int kWarpStride = kVec ? 32 : kWords * 32 + 1, kStride = kWords * kThreads + (kVec ? 0 : kThreads / 32);

    // Copies this thread's part of a row's piece, of which n values are there (n <= 0: zeros). p and to: kVec, its own
    // piece; else its warp's, and the words may also hold what stands beside the row.
    static __device__ __forceinline__ void fetch(const T* p, int n, uint4* to) {
        if constexpr (kVec) {
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                copy_async16(to + i * kThreads, reinterpret_cast<const uint4*>(p) + i, n > 0);
        } else {
            const int lane = threadIdx.x & 31, off = (int)(reinterpret_cast<uintptr_t>(p) & 15);
            const int bytes = n > 0 ? off + n * (int)sizeof(T) : 0;
            const char* from = reinterpret_cast<const char*>(p) - off;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const int at = lane + 32 * i;
                copy_async16(to + at, from + 16 * at, 16 * at < bytes);
            }
            if (lane == 0) copy_async16(to + 32 * kWords, from + 512 * kWords, 512 * kWords < bytes);
        }
    }
    // This thread's piece as four fp32 pairs, zeros beyond its n values; off: the warp's p's offset from 16 bytes.
    static __device__ __forceinline__ void read(const uint4* from, uint32_t off, int n, uint64_t (&f)[4]) {
        uint32_t v[kRegs];
        if constexpr (kVec) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) to_regs(from[i * kThreads], v + 4 * i);
        } else {
            uint32_t w[kRegs + 4];
            from += (threadIdx.x & 31) * kWords;
#pragma unroll
            for (int i = 0; i <= kWords; ++i) to_regs(from[i], w + 4 * i);
            shift_bytes<sizeof(T), kRegs>(w, off, v);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2)
                f[i] = bf_pair(v[i]);
            else
                f[i] = f2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
        }
        if (!kVec && n < 8) clear_from(n, f);
    }
    // kVec: p is this thread's; else its warp's, which has n values.
    static __device__ __forceinline__ void store(T* p, int n, const uint64_t (&f)[4]) {
        uint32_t v[kRegs];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo, hi;
            uf2(f[i], lo, hi);
            if constexpr (sizeof(T) == 2)
                v[i] = pack_bf16x2(lo, hi);
            else
                v[2 * i] = __float_as_uint(lo), v[2 * i + 1] = __float_as_uint(hi);
        }
        if constexpr (kVec) {
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                reinterpret_cast<uint4*>(p)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
            store_unaligned<T, kRegs>(p, n, v);
        }
    }
};
// The offset of row r from a 16-byte boundary, and so (pieces of a warp being whole multiples of 16 bytes apart) that of
// its stretches.
template <bool kVec, typename T>
__device__ __forceinline__ uint32_t row_offset(const T* base, int r, int c) {
    return kVec ? 0u : ((uint32_t)reinterpret_cast<uintptr_t>(base) + (uint32_t)r * (uint32_t)c * (uint32_t)sizeof(T)) & 15u;
}
template <typename T>
__device__ __forceinline__ float vec_or(const void* v, int c, float otherwise) {
    return v ? load_as_float(static_cast<const T*>(v) + c) : otherwise;
}

// The sums of v[0..N) over the tpr threads of a row group, in each of them (N = 1, 2 or 4). Within a warp a butterfly
// whose first steps also halve the values a lane holds; then the warps' sums through `part` ([32 warps][N]) and a barrier
// of the CTA (every thread calls this the same number of times; two calls in a row use different buffers), which each
// warp adds up by another butterfly. The order is fixed by the lanes.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* part, int group_warp0, int warps) {
    const int lane = threadIdx.x & 31;
    int bit = 16;
#pragma unroll
    for (int half = N / 2; half >= 1; half /= 2, bit /= 2) {
        const bool up = lane & bit;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float keep = up ? v[i + half] : v[i], give = up ? v[i] : v[i + half];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
        }
    }
    constexpr int kHold = 32 / N;  // lanes that now hold the same value, lane / kHold
    float s = v[0];
#pragma unroll
    for (int o = kHold / 2; o >= 1; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (warps == 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, s, i * kHold);
        return;
    }
    if (lane % kHold == 0) part[(threadIdx.x >> 5) * N + lane / kHold] = s;
    __syncthreads();
    part += group_warp0 * N;
    s = lane < warps * N ? part[lane] : 0.0f;
    for (int i = lane + 32; i < warps * N; i += 32) s += part[i];
#pragma unroll
    for (int o = 16; o >= N; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, s, i);
}

// 1 / √v: the hardware's approximation (2^-22) and one Newton step, except where that step has nothing to refine.
__device__ __forceinline__ float rsqrt_refined(float v) {
    const float r = rsqrtf(v);
    return v > 0.0f && r > 0.0f ? r * fmaf(-0.5f * v * r, r, 1.5f) : r;
}

constexpr int kStages = 3;
// Of the backward pass: with three, fp32 rings of three CTAs do not fit an SM (17280 × 1536: 94 against 90 µs), and bf16
// gains nothing by the third.
constexpr int kBackwardStages = 2;
// Rows at once: forward four of bf16, two of fp32, backward two; with two pieces a thread, forward two and one, backward
// one. Threads that the kernels' registers let an SM hold: 768 of the forward pass (80 registers), 576 of the backward
// pass (112; 512 in CTAs of 256).
constexpr int kBackwardRows = 2, kForwardThreads = 768, kBackwardThreads = 576;

// kP: pieces of eight channels a thread owns, tpr · 8 channels apart.
template <typename T, bool kVec, int kRows, int kP, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads, kForwardThreads / kMaxThreads > 1 ? kForwardThreads / kMaxThreads : 1)
    norm_train_kernel(const NormTrainArgs a, int tpr) {
    extern __shared__ uint4 ring[];  // [kStages][kRows][kP][words][kMaxThreads]
    __shared__ alignas(16) float part[2][32 * kRows];
    using P = Piece<T, kVec, kMaxThreads>;
    constexpr int kPieceWords = P::kStride, kRowWords = kP * kPieceWords;
    const int groups = (int)blockDim.x / tpr, g = (int)threadIdx.x / tpr, warps = tpr >> 5, warp0 = g * warps;
    const int col0 = ((int)threadIdx.x % tpr) * 8;
    auto col = [&](int p) { return col0 + p * tpr * 8; };
    int lens[kP];
#pragma unroll
    for (int p = 0; p < kP; ++p) lens[p] = max(0, min(8, a.c - col(p)));
    auto len = [&](int p) { return lens[p]; };  // of piece p
    // where this thread's part in the copies starts, and how much of it a row has: its own pieces, or (not kVec) its warp's
    const int at0 = kVec ? col0 : col0 & ~255;
    auto here = [&](int p) { return kVec ? len(p) : min(256, a.c - at0 - p * tpr * 8); };
    const int step = (int)gridDim.x * groups * kRows, row_first = ((int)blockIdx.x * groups + g) * kRows, m = (int)a.m;
    const int64_t c = a.c;
    const float inv_c = 1.0f / (float)a.c;
    int left = m - row_first;  // rows from the group's next ones to the end
    const T* x = static_cast<const T*>(a.x);
    int64_t fetch_at = row_first * c + at0;  // of the rows to fetch next
    auto fetch = [&](uint4* to, int rows) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int p = 0; p < kP; ++p)
                P::fetch(x + fetch_at + i * c + p * tpr * 8, i < rows ? here(p) : 0, to + i * kRowWords + p * kPieceWords);
        copy_async_commit();
        fetch_at += step * c;
    };
    griddep_wait_then_release();
    uint4* const mine = ring + (kVec ? (int)threadIdx.x : ((int)threadIdx.x >> 5) * P::kWarpStride);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) fetch(mine + s * kRows * kRowWords, left - s * step);
    uint64_t gain[kP][4], base[kP][4];
#pragma unroll
    for (int p = 0; p < kP; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float gv[2], bv[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const bool here = 2 * i + j < len(p);
                const int at = here ? col(p) + 2 * i + j : 0;
                const float s1 = 1.0f + vec_or<T>(a.scale, at, 0.0f);
                gv[j] = here ? s1 * vec_or<T>(a.weight, at, 1.0f) : 0.0f;
                bv[j] = here ? fmaf(vec_or<T>(a.bias, at, 0.0f), s1, vec_or<T>(a.shift, at, 0.0f)) : 0.0f;
            }
            gain[p][i] = f2(gv[0], gv[1]), base[p][i] = f2(bv[0], bv[1]);
        }
    int stage = 0;
    for (int cta_left = m - (int)blockIdx.x * groups * kRows; cta_left > 0; cta_left -= step, left -= step) {
        if (!kVec) __syncwarp();  // the warp has read the stage that is filled now
        fetch(mine + (stage == 0 ? kStages - 1 : stage - 1) * kRows * kRowWords, left - (kStages - 1) * step);
        copy_async_wait<kStages - 1>();
        if (!kVec) __syncwarp();  // and all its lanes' copies have arrived
        const uint4* now = mine + stage * kRows * kRowWords;
        float sum[kRows], sq[kRows];
        uint64_t f[kRows][kP][4];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            sum[i] = 0.0f;
#pragma unroll
            for (int p = 0; p < kP; ++p) {
                uint64_t(&v)[4] = f[i][p];
                P::read(now + i * kRowWords + p * kPieceWords, row_offset<kVec>(x, m - left + i, a.c), len(p), v);
                sum[i] += pair_sum(fadd2(fadd2(v[0], v[1]), fadd2(v[2], v[3])));
            }
        }
        group_sum<kRows>(sum, part[0], warp0, warps);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            sum[i] *= inv_c;
            const uint64_t minus = f2(-sum[i], -sum[i]);
            sq[i] = 0.0f;
#pragma unroll
            for (int p = 0; p < kP; ++p) {
                uint64_t q = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint64_t d = f[i][p][j] = fadd2(f[i][p][j], minus);
                    if (!kVec && 2 * j + 1 >= len(p)) {  // a piece that ends inside
                        float lo, hi;
                        uf2(d, lo, hi);
                        d = f2(2 * j < len(p) ? lo : 0.0f, 0.0f);
                    }
                    q = ffma2(d, d, q);
                }
                if (len(p) > 0) sq[i] += pair_sum(q);
            }
        }
        group_sum<kRows>(sq, part[1], warp0, warps);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (i >= left) break;
            const float rstd = rsqrt_refined(fmaf(sq[i], inv_c, a.eps));
            if (col0 == 0) a.mean[m - left + i] = sum[i], a.rstd[m - left + i] = rstd;
            const uint64_t r2 = f2(rstd, rstd);
#pragma unroll
            for (int p = 0; p < kP; ++p) {
                if (here(p) <= 0) continue;
                uint64_t(&v)[4] = f[i][p];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = ffma2(fmul2(v[j], r2), gain[p][j], base[p][j]);
                P::store(static_cast<T*>(a.out) + (int64_t)(m - left + i) * c + at0 + p * tpr * 8, here(p), v);
            }
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    copy_async_wait<0>();
}

// kHeld: x is the 8-bit form; a piece of it is 8 bytes.
template <typename T, bool kHeld, bool kVec, int kRows, int kP, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads, kBackwardThreads / kMaxThreads > 1 ? kBackwardThreads / kMaxThreads : 1)
    norm_backward_kernel(const NormTrainArgs a, int tpr) {
    constexpr int kStages = kBackwardStages;
    extern __shared__ uint4 ring[];  // [kStages][kRows][kP][words of dy][kMaxThreads], then the same of x (8 bytes if held)
    __shared__ alignas(16) float part[2][32 * 2 * kRows];
    using P = Piece<T, kVec, kMaxThreads>;
    constexpr int kPieceWords = P::kStride, kRowWords = kP * kPieceWords;
    const int groups = (int)blockDim.x / tpr, g = (int)threadIdx.x / tpr, warps = tpr >> 5, warp0 = g * warps;
    const int col0 = ((int)threadIdx.x % tpr) * 8;
    auto col = [&](int p) { return col0 + p * tpr * 8; };
    int lens[kP];
#pragma unroll
    for (int p = 0; p < kP; ++p) lens[p] = max(0, min(8, a.c - col(p)));
    auto len = [&](int p) { return lens[p]; };  // of piece p
    // where this thread's part in the copies starts, and how much of it a row has: its own pieces, or (not kVec) its warp's
    const int at0 = kVec ? col0 : col0 & ~255;
    auto here = [&](int p) { return kVec ? len(p) : min(256, a.c - at0 - p * tpr * 8); };
    const int step = (int)gridDim.x * groups * kRows, row_first = ((int)blockIdx.x * groups + g) * kRows, m = (int)a.m;
    const int64_t c = a.c, ld = fp8_ld(a.c);
    const float inv_c = -1.0f / (float)a.c;
    int left = m - row_first;  // rows from the group's next ones to the end
    const T *dy = static_cast<const T*>(a.dy), *x = static_cast<const T*>(a.x);
    const uint8_t* x8 = static_cast<const uint8_t*>(a.x);
    int64_t fetch_at = row_first * c + at0, fetch_at8 = row_first * ld + col0;  // of the rows to fetch next
    uint4* const mine = ring + (kVec ? (int)threadIdx.x : ((int)threadIdx.x >> 5) * P::kWarpStride);
    uint4* const mine_x = mine + kStages * kRows * kRowWords;
    uint2* const mine_x8 = reinterpret_cast<uint2*>(ring + kStages * kRows * kRowWords) + threadIdx.x;
    auto fetch = [&](int stage, int rows) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int p = 0; p < kP; ++p) {
                const int n = i < rows ? here(p) : 0, piece = (stage * kRows + i) * kP + p;
                P::fetch(dy + fetch_at + i * c + p * tpr * 8, n, mine + piece * kPieceWords);
                if constexpr (kHeld)
                    copy_async8(mine_x8 + piece * kMaxThreads, x8 + fetch_at8 + i * ld + p * tpr * 8, i < rows && len(p) > 0);
                else
                    P::fetch(x + fetch_at + i * c + p * tpr * 8, n, mine_x + piece * kPieceWords);
            }
        copy_async_commit();
        fetch_at += step * c;
        if (kHeld) fetch_at8 += step * ld;
    };
    // the rows' statistics (and codes) one step ahead, in registers; past the last row, that row's: its dy there is zero
    float next_mean[kRows], next_rstd[kRows];
    uint32_t next_code[kRows][kP];
    const int tile_bytes = (int)fp8_scale_tiles(a.c) * 512;
    int code_at[kP];
#pragma unroll
    for (int p = 0; p < kP; ++p) {
        const int block = min(col(p), a.c - 1) >> 7;
        code_at[p] = (block >> 2) * 512 + (block & 3);
    }
    auto fetch_row = [&](int rows) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = min(m - rows + i, m - 1);
            next_mean[i] = a.mean[r], next_rstd[i] = a.rstd[r];
#pragma unroll
            for (int p = 0; p < kP; ++p)
                if (kHeld)
                    next_code[i][p] =
                        a.x_scale[(int64_t)(r >> 7) * tile_bytes + (r & 31) * 16 + ((r >> 5) & 3) * 4 + code_at[p]];
        }
    };
    griddep_wait_then_release();
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) fetch(s, left - s * step);
    fetch_row(left);
    uint64_t gain[kP][4], sum_a[kP][4], sum_b[kP][4];
#pragma unroll
    for (int p = 0; p < kP; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float gv[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const bool here = 2 * i + j < len(p);
                const int at = here ? col(p) + 2 * i + j : 0;
                gv[j] = here ? (1.0f + vec_or<T>(a.scale, at, 0.0f)) * vec_or<T>(a.weight, at, 1.0f) : 0.0f;
            }
            gain[p][i] = f2(gv[0], gv[1]);
            sum_a[p][i] = sum_b[p][i] = 0;
        }
    int stage = 0, flip = 0;
    for (int cta_left = m - (int)blockIdx.x * groups * kRows; cta_left > 0; cta_left -= step, left -= step, flip ^= 1) {
        if (!kVec) __syncwarp();  // the warp has read the stage that is filled now
        fetch(stage == 0 ? kStages - 1 : stage - 1, left - (kStages - 1) * step);
        copy_async_wait<kStages - 1>();
        if (!kVec) __syncwarp();  // and all its lanes' copies have arrived
        uint64_t norm[kRows][kP][4], grad[kRows][kP][4];
        float rstd[kRows], s[2 * kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            rstd[i] = next_rstd[i];
            const uint64_t minus = f2(-next_mean[i], -next_mean[i]), r2 = f2(rstd[i], rstd[i]);
            s[2 * i] = s[2 * i + 1] = 0.0f;
#pragma unroll
            for (int p = 0; p < kP; ++p) {
                const int piece = (stage * kRows + i) * kP + p;
                uint64_t(&n)[4] = norm[i][p];
                uint64_t(&d)[4] = grad[i][p];
                P::read(mine + piece * kPieceWords, row_offset<kVec>(dy, m - left + i, a.c), len(p), d);
                if constexpr (kHeld) {
                    const uint2 u = mine_x8[piece * kMaxThreads];
                    const uint32_t two[4] = {u.x, u.x >> 16, u.y, u.y >> 16};
                    const float down = fp8_down(next_code[i][p]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {  // the scaling is exact: one rounding, in the subtraction
                        float lo, hi;
                        fp8_unpack2(two[j], lo, hi);
                        n[j] = ffma2(f2(lo, hi), f2(down, down), minus);
                    }
                } else {
                    P::read(mine_x + piece * kPieceWords, row_offset<kVec>(x, m - left + i, a.c), len(p), n);
#pragma unroll
                    for (int j = 0; j < 4; ++j) n[j] = fadd2(n[j], minus);
                }
                uint64_t s1 = 0, s2 = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    n[j] = fmul2(n[j], r2);
                    sum_a[p][j] = ffma2(d[j], n[j], sum_a[p][j]);
                    sum_b[p][j] = fadd2(sum_b[p][j], d[j]);
                    d[j] = fmul2(d[j], gain[p][j]);
                    s1 = fadd2(s1, d[j]);
                    s2 = ffma2(d[j], n[j], s2);
                }
                s[2 * i] += pair_sum(s1);
                if (len(p) > 0) s[2 * i + 1] += pair_sum(s2);
            }
        }
        fetch_row(left - step);
        group_sum<2 * kRows>(s, part[flip], warp0, warps);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (i >= left) break;
            const float c1 = s[2 * i] * inv_c, c2 = s[2 * i + 1] * inv_c;
            const uint64_t c1p = f2(c1, c1), c2p = f2(c2, c2), r2 = f2(rstd[i], rstd[i]);
#pragma unroll
            for (int p = 0; p < kP; ++p) {
                if (here(p) <= 0) continue;
                uint64_t f[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = fmul2(ffma2(norm[i][p][j], c2p, fadd2(grad[i][p][j], c1p)), r2);
                P::store(static_cast<T*>(a.out) + (int64_t)(m - left + i) * c + at0 + p * tpr * 8, here(p), f);
            }
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    copy_async_wait<0>();
    // the CTA's sums: the groups' in order, through the ring
    if (groups > 1) {
        __syncthreads();
        uint64_t* const held = reinterpret_cast<uint64_t*>(ring);  // [8 kP][kMaxThreads]
#pragma unroll
        for (int p = 0; p < kP; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                held[(8 * p + i) * kMaxThreads + threadIdx.x] = sum_a[p][i];
                held[(8 * p + 4 + i) * kMaxThreads + threadIdx.x] = sum_b[p][i];
            }
        __syncthreads();
        for (int o = 1; g == 0 && o < groups; ++o)
#pragma unroll
            for (int p = 0; p < kP; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sum_a[p][i] = fadd2(sum_a[p][i], held[(8 * p + i) * kMaxThreads + threadIdx.x + o * tpr]);
                    sum_b[p][i] = fadd2(sum_b[p][i], held[(8 * p + 4 + i) * kMaxThreads + threadIdx.x + o * tpr]);
                }
        if (g != 0) return;
    }
    float* to = a.partial + (int64_t)blockIdx.x * 2 * a.c;
#pragma unroll
    for (int p = 0; p < kP; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float av[2], bv[2];
            uf2(sum_a[p][i], av[0], av[1]);
            uf2(sum_b[p][i], bv[0], bv[1]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (2 * i + j < len(p)) to[col(p) + 2 * i + j] = av[j], to[a.c + col(p) + 2 * i + j] = bv[j];
        }
}

// The CTAs' sums of eight channels (a 32-byte sector): 64 rows of eight threads take every 64th CTA's each, eight at a
// time in flight (the few hundred CTAs of a full device are one round trip to L2), then their sums in a fixed order.
template <typename T>
__global__ void __launch_bounds__(512) norm_vectors_kernel(const NormTrainArgs a, int ctas) {
    __shared__ float sa[16][8], sb[16][8];
    griddep_wait_then_release();
    const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3, c = blockIdx.x * 8 + tx;
    float va = 0.0f, vb = 0.0f;
    const int64_t step = (int64_t)128 * a.c;
    const float* p = a.partial + (int64_t)ty * 2 * a.c + c;
    for (int i = c < a.c ? ty : ctas; i < ctas; i += 512) {
        float pa[8], pb[8];
#pragma unroll
        for (int j = 0; j < 8; ++j, p += step) {
            const bool here = i + 64 * j < ctas;
            pa[j] = here ? p[0] : 0.0f, pb[j] = here ? p[a.c] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) va += pa[j], vb += pb[j];
    }
#pragma unroll
    for (int o = 8; o <= 16; o *= 2) {
        va += __shfl_xor_sync(0xffffffffu, va, o);
        vb += __shfl_xor_sync(0xffffffffu, vb, o);
    }
    if ((threadIdx.x & 31) < 8) sa[threadIdx.x >> 5][tx] = va, sb[threadIdx.x >> 5][tx] = vb;
    __syncthreads();
    if (ty != 0 || c >= a.c) return;
    va = vb = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) va += sa[i][tx], vb += sb[i][tx];
    const float s1 = 1.0f + vec_or<T>(a.scale, c, 0.0f);
    if (a.dweight) a.dweight[c] = s1 * va;
    if (a.dbias) a.dbias[c] = s1 * vb;
    if (a.dscale) a.dscale[c] = fmaf(vec_or<T>(a.weight, c, 1.0f), va, vec_or<T>(a.bias, c, 0.0f) * vb);
    if (a.dshift) a.dshift[c] = vb;
}

// Pieces a thread owns, threads of a row and of a CTA for c channels, and how many CTAs share an SM. Two pieces above
// 4096 channels: one would take CTAs of over 512 threads with 64 registers each (4096 × 8192 bf16 forward 38 instead of 27
// µs, backward 59 / 54); at 1536 two are slower (forward 24 / 22, backward 40 / 37).
struct Shape {
    int pieces, tpr, threads, groups;
    explicit Shape(int c) : pieces(c > 4096 ? 2 : 1) {
        tpr = ((c + 8 * pieces - 1) / (8 * pieces) + 31) / 32 * 32;
        groups = tpr >= 256 ? 1 : 256 / tpr;
        threads = tpr * groups;
    }
    int ctas(int64_t m, int rows, int sm_threads) const {
        const int64_t need = (m + groups * rows - 1) / (groups * rows);
        const int64_t most = (int64_t)sm_count() * (sm_threads > threads ? sm_threads / threads : 1);
        return (int)(need < most ? need : most);
    }
};

template <auto kernel>
cudaError_t launch_ring(int ctas, const Shape& s, size_t ring_bytes, const NormTrainArgs& a, cudaStream_t st) {
    if (ring_bytes > 40 * 1024) {
        cudaError_t e = allow_smem<kernel>(ring_bytes);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(kernel, dim3(ctas), dim3(s.threads), ring_bytes, st, a, s.tpr);
}

template <typename T, bool kVec, int kRows, int kP, int kMaxThreads>
cudaError_t train_threads(const NormTrainArgs& a, const Shape& s, cudaStream_t st) {
    const size_t ring = (size_t)16 * kStages * kRows * kP * Piece<T, kVec, kMaxThreads>::kStride;
    return launch_ring<norm_train_kernel<T, kVec, kRows, kP, kMaxThreads>>(s.ctas(a.m, kRows, kForwardThreads), s, ring, a, st);
}

template <typename T, bool kVec, int kRows, int kP>
cudaError_t train_pieces(const NormTrainArgs& a, const Shape& s, cudaStream_t st) {
    if constexpr (kP == 1) {  // two pieces: more than 256 threads
        if (s.threads <= 192) return train_threads<T, kVec, kRows, kP, 192>(a, s, st);
        if (s.threads <= 256) return train_threads<T, kVec, kRows, kP, 256>(a, s, st);
    }
    return train_threads<T, kVec, kRows, kP, 512>(a, s, st);
}

template <typename T, bool kVec>
cudaError_t train(const NormTrainArgs& a, cudaStream_t st) {
    constexpr int kRows = sizeof(T) == 2 ? 4 : 2;
    const Shape s(a.c);
    return s.pieces == 1 ? train_pieces<T, kVec, kRows, 1>(a, s, st) : train_pieces<T, kVec, kRows / 2, 2>(a, s, st);
}

template <typename T, bool kHeld, bool kVec, int kRows, int kP, int kMaxThreads>
cudaError_t backward_threads(const NormTrainArgs& a, const Shape& s, int ctas, cudaStream_t st) {
    constexpr int kDy = 16 * Piece<T, kVec, kMaxThreads>::kStride, kX = kHeld ? 8 * kMaxThreads : kDy;
    const size_t ring = (size_t)kBackwardStages * kRows * kP * (kDy + kX);
    return launch_ring<norm_backward_kernel<T, kHeld, kVec, kRows, kP, kMaxThreads>>(ctas, s, ring, a, st);
}

template <typename T, bool kHeld, bool kVec, int kRows, int kP>
cudaError_t backward_pieces(const NormTrainArgs& a, const Shape& s, int ctas, cudaStream_t st) {
    if constexpr (kP == 1) {  // two pieces: more than 256 threads
        if (s.threads <= 192) return backward_threads<T, kHeld, kVec, kRows, kP, 192>(a, s, ctas, st);
        if (s.threads <= 256) return backward_threads<T, kHeld, kVec, kRows, kP, 256>(a, s, ctas, st);
    }
    return backward_threads<T, kHeld, kVec, kRows, kP, 512>(a, s, ctas, st);
}

template <typename T, bool kHeld, bool kVec>
cudaError_t backward_rows(const NormTrainArgs& a, const Shape& s, int ctas, cudaStream_t st) {
    return s.pieces == 1 ? backward_pieces<T, kHeld, kVec, kBackwardRows, 1>(a, s, ctas, st)
                         : backward_pieces<T, kHeld, kVec, 1, 2>(a, s, ctas, st);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
cudaError_t backward(const NormTrainArgs& a, cudaStream_t st) {
    const Shape s(a.c);
    const int ctas = norm_backward_ctas(a.m, a.c);
    cudaError_t e = cudaSuccess;
    if (ctas > 0) {
        const bool vec = a.c % 8 == 0 && aligned16(a.dy) && aligned16(a.out) && aligned16(a.x);
        if (a.x_scale)
            e = vec ? backward_rows<T, true, true>(a, s, ctas, st) : backward_rows<T, true, false>(a, s, ctas, st);
        else
            e = vec ? backward_rows<T, false, true>(a, s, ctas, st) : backward_rows<T, false, false>(a, s, ctas, st);
    }
    if (e != cudaSuccess || !(a.dweight || a.dbias || a.dscale || a.dshift)) return e;
    return launch_pdl(norm_vectors_kernel<T>, dim3((a.c + 7) / 8), dim3(512), 0, st, a, ctas);
}

}  // namespace

int norm_backward_ctas(int64_t m, int c) {
    const Shape s(c);
    return s.ctas(m, s.pieces == 1 ? kBackwardRows : 1, kBackwardThreads);
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
