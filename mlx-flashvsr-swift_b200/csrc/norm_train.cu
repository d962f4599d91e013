// norm_train.cu — LayerNorm over the channels for training: the forward pass that keeps each row's mean and
// rstd = 1/√(var + eps), and the backward pass with the gradients of its vectors.
//   n = (x − mean)·rstd,  y = (n·w + b)·(1 + scale) + shift          (w, b and shift, scale each optional)
//   g = dy·(1 + scale)·w, dx = rstd·(g − mean_c(g) − n·mean_c(g·n))
//   A = Σ_rows dy·n, B = Σ_rows dy: dw = (1 + scale)·A, db = (1 + scale)·B, dscale = w·A + b·B, dshift = B.
// fp32 throughout, one rounding of y and dx to the tensors' type.
//
// Both passes move bytes, x (and dy) read once and the result written once. A thread owns eight channels (or
// twice eight) of every row it meets, so the vectors, and in the backward pass the sums A and B of those channels, stay in
// its registers over all rows: tpr = ⌈c / 8⌉ threads, in whole warps, work on a row, kRows rows at once to share a
// barrier; narrow rows put several such groups in a CTA. Rows are copied ahead into shared memory with cp.async, each
// thread its own pieces (so that no barrier guards them), kStages sets of rows deep: what is in flight costs no
// registers. Arithmetic is on pairs (f32x2), without which the backward pass would be bound by issue slots. The variance
// is taken about the mean in a second pass over the pieces. The vectors' gradients are summed per CTA over its rows,
// then over the CTAs by a second kernel, both in a fixed order, so they do not depend on timing.
// Where rows do not start on the 16-byte grid (c not a multiple of eight, or a tensor that starts off it) all accesses but
// those at a row's two ends are still 16 aligned bytes (enum Grid below).
// One B200, µs (share of the copy rate, 6533 GB/s):   forward     backward    from the 8-bit form
//   17,280 × 1536 bf16                               22 (0.73)   37 (0.66)   40
//   30,720 × 1536 bf16                               34 (0.84)   55 (0.79)   60
//   4096 × 8192 bf16                                 28 (0.74)   54 (0.57)   56
//   17,280 × 1536 fp32                               39 (0.83)   57 (0.85)   45
//   8640 × 2048 bf16                                 17 (0.64)   28 (0.57)   29
//   4096 × 8192 bf16                                 28 (0.74)   55 (0.57)   57
//   17,280 × 1531 bf16                               33          45          66
//   17,280 × 1531 fp32                               38          62          73
// What keeps bf16 from memory's rate is neither memory nor instructions, but waits: at 17,280 × 1536 the backward pass has
// DRAM 45 % busy (from 8 bits 32 %, the forward pass 30 %) and half of its issue slots used, by 15 warps an SM (21) that its
// registers leave, which wait for their own results, for shared memory and for the barrier of every two rows. The CTAs
// divide an SM's registers evenly at 1536 channels; at 2048 and above 4096 fewer warps share it.
#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"
#include "sm100.cuh"
#include "unaligned.cuh"

#include <algorithm>

namespace fvsr {

namespace {

using namespace sm100;

// Asynchronous copies of 16 bytes, or of 8 or 4, or as many zeros without a source (here false: src is not read).
__device__ __forceinline__ void copy_async16(void* dst, const void* src, bool here) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(here ? 16 : 0)
                 : "memory");
}
template <int kBytes>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool here) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_u32(dst)), "l"(src), "n"(kBytes),
                 "r"(here ? kBytes : 0)
                 : "memory");
}
template <int kParts>
struct PartOf {
    using type = uint2;
};
template <>
struct PartOf<2> {
    using type = uint32_t;
};
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
// Zeros where the mask's bit is not set: by the bit masks of four values that shared memory holds for each of the sixteen
// cases (test and select of each value took twice the instructions, and a row's two ends hold up the rest of its threads).
__device__ __forceinline__ void fill_nibbles(uint4* nibbles) {
    const uint32_t t = threadIdx.x;
    if (t < 16)
        nibbles[t] = make_uint4(0u - (t & 1), 0u - (t >> 1 & 1), 0u - (t >> 2 & 1), 0u - (t >> 3 & 1));
    __syncthreads();
}
template <typename... Pieces>
__device__ __forceinline__ void clear_outside(const uint4* nibbles, uint32_t mask, Pieces&... pieces) {
    const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(nibbles + (mask & 15));
    const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(nibbles + (mask >> 4));
    ((pieces[0] &= a.x, pieces[1] &= a.y, pieces[2] &= b.x, pieces[3] &= b.y), ...);
}

// How a row's pieces of eight values lie against the 16-byte grid.
enum Grid {
    kWhole,    // rows start on it and are whole pieces
    kClasses,  // they do not, but all tensors' rows are off it alike: a group of threads keeps to rows that are off by the
               // same, so its threads' pieces can start on the grid, the first before the row (17,280 × 1531 bf16 forward 33
               // µs, element by element 68)
    kShifted,  // the tensors' rows are off it by different amounts, or x is the 8-bit form, whose rows are never off it:
               // pieces start at the row's start and are shifted (46 µs)
};

// A thread's eight values of a row: one 16-byte word of bf16, two of fp32, 32 words apart in the row, so that a warp's
// accesses are contiguous (with the two side by side each access took half of every sector: 17,280 × 1536 backward 92 µs);
// kShifted: side by side. In shared memory the pieces of kThreads threads take kStride words: [word][thread], or (kShifted)
// for each warp the aligned words that cover its stretch of the row, one more than its pieces have. A mask has the bits of
// a piece's values that are in the row; `part` is it, or (kShifted) how many values of the row the warp's stretch has.
template <typename T, Grid kGrid, int kThreads>
struct Piece {
    static constexpr int kWords = (int)sizeof(T) / 2, kRegs = kWords * 4, kWord = 8 / kWords;
    static constexpr int kLane = kGrid == kShifted ? 8 : kWord, kNext = kGrid == kShifted ? kWord : 32 * kWord;
    static constexpr int kWarpStride = kGrid == kShifted ? kWords * 32 + 1 : 32;
    static constexpr int kStride = kWords * kThreads + (kGrid == kShifted ? kThreads / 32 : 0);

    static __device__ __forceinline__ uint32_t of_word(uint32_t mask, int i) {
        return kWords == 1 ? mask : mask >> (i * kWord) & ((1 << kWord) - 1);
    }
    // Copies this thread's part of a row's pieces (part <= 0: zeros). p and to: of its own piece; kShifted: of its warp's
    // stretch. The words copied may also hold what stands beside the row.
    static __device__ __forceinline__ void fetch(const T* p, int part, uint4* to) {
        if constexpr (kGrid == kShifted) {
            const int lane = threadIdx.x & 31, off = (int)(reinterpret_cast<uintptr_t>(p) & 15);
            const int bytes = part > 0 ? off + part * (int)sizeof(T) : 0;
            const char* from = reinterpret_cast<const char*>(p) - off;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const int at = lane + 32 * i;
                copy_async16(to + at, from + 16 * at, 16 * at < bytes);
            }
            if (lane == 0) copy_async16(to + 32 * kWords, from + 512 * kWords, 512 * kWords < bytes);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) copy_async16(to + i * kThreads, p + i * kNext, of_word(part, i) != 0);
        }
    }
    // This thread's piece as four fp32 pairs, what is outside the mask as it stands there (zeros where it was not copied);
    // off: the warp's p's offset from 16 bytes.
    static __device__ __forceinline__ void read(const uint4* from, uint32_t off, uint64_t (&f)[4]) {
        uint32_t v[kRegs];
        if constexpr (kGrid == kShifted) {
            uint32_t w[kRegs + 4];
            from += (threadIdx.x & 31) * kWords;
#pragma unroll
            for (int i = 0; i <= kWords; ++i) to_regs(from[i], w + 4 * i);
            shift_bytes<sizeof(T), kRegs>(w, off, v);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) to_regs(from[i * kThreads], v + 4 * i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2)
                f[i] = bf_pair(v[i]);
            else
                f[i] = f2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
        }
    }
    template <typename... Pieces>
    static __device__ __forceinline__ void clear(const uint4* nibbles, uint32_t mask, Pieces&... pieces) {
        if (kGrid != kWhole && mask != 255) clear_outside(nibbles, mask, pieces...);
    }
    // p: as fetch.
    static __device__ __forceinline__ void store(T* p, int part, const uint64_t (&f)[4]) {
        uint32_t v[kRegs];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a, b;
            uf2(f[i], a, b);
            if constexpr (sizeof(T) == 2)
                v[i] = pack_bf16x2(a, b);
            else
                v[2 * i] = __float_as_uint(a), v[2 * i + 1] = __float_as_uint(b);
        }
        if constexpr (kGrid == kShifted) {
            store_unaligned<T, kRegs>(p, part, v);
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const uint32_t in = of_word(part, i);
                if (kGrid == kWhole ? in != 0 : in == (1 << kWord) - 1) {
                    *reinterpret_cast<uint4*>(p + i * kNext) =
                        make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
                } else if (kGrid == kClasses && in != 0) {
#pragma unroll
                    for (int j = 0; j < kWord; ++j) {
                        if (!(in >> j & 1)) continue;
                        if constexpr (sizeof(T) == 2)
                            reinterpret_cast<uint16_t*>(p)[j] = (uint16_t)(j & 1 ? v[j / 2] >> 16 : v[j / 2]);
                        else
                            reinterpret_cast<uint32_t*>(p)[i * kNext + j] = v[4 * i + j];
                    }
                }
            }
        }
    }
};

// The rows that a group of threads takes: those of its class, r ≡ cls (mod 2^log), `step` of them further on at a time.
struct Walk {
    int log, cls, m, first, step, cta_left;  // m: rows of the class; first, step: among them; cta_left: of no group more
    __device__ __forceinline__ Walk(int rows, int log_, int groups, int g, int at_once) : log(log_) {
        const int index = (int)blockIdx.x * groups + g, period = 1 << log;
        cls = index & (period - 1);
        m = (rows - cls + period - 1) >> log;
        first = (index >> log) * at_once;
        step = ((int)gridDim.x * groups >> log) * at_once;
        cta_left = ((rows + period - 1) >> log) - ((int)blockIdx.x * groups >> log) * at_once;
    }
    __device__ __forceinline__ int row(int i) const { return cls + (i << log); }
};

// kShifted: the offset of row r from a 16-byte boundary, and so (a warp's stretches being whole multiples of 16 bytes
// apart) that of its stretches.
template <Grid kGrid, typename T>
__device__ __forceinline__ uint32_t row_offset(const T* base, int r, int c) {
    if (kGrid != kShifted) return 0;
    return ((uint32_t)reinterpret_cast<uintptr_t>(base) + (uint32_t)r * (uint32_t)c * (uint32_t)sizeof(T)) & 15u;
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
// Of the backward pass: with three, fp32 rings of three CTAs do not fit an SM (17280 × 1536: 61 against 58 µs), and bf16
// gains nothing by the third (37.3 / 36.7).
constexpr int kBackwardStages = 2;
// Rows at once: forward four of bf16, two of fp32, backward two; with two pieces a thread, forward two and one, backward
// one. Threads that the kernels' registers let an SM hold: 768 of the forward pass (80 registers), 576 of the backward
// pass (112; 512 in CTAs of 256).
constexpr int kBackwardRows = 2, kForwardThreads = 768, kBackwardThreads = 576;

// kP: pieces of eight channels a thread owns, tpr · 8 channels apart.
template <typename T, Grid kGrid, int kRows, int kP, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads, kForwardThreads / kMaxThreads > 1 ? kForwardThreads / kMaxThreads : 1)
    norm_train_kernel(const NormTrainArgs a, int tpr, int log_period) {
    extern __shared__ uint4 ring[];  // [kStages][kRows][kP][words][kMaxThreads]
    __shared__ alignas(16) float part[2][32 * kRows];
    __shared__ uint4 nibbles[kGrid == kWhole ? 1 : 16];
    using P = Piece<T, kGrid, kMaxThreads>;
    constexpr int kPieceWords = P::kStride, kRowWords = kP * kPieceWords;
    const int groups = (int)blockDim.x / tpr, g = (int)threadIdx.x / tpr, warps = tpr >> 5, warp0 = g * warps;
    const Walk walk((int)a.m, kGrid == kClasses ? log_period : 0, groups, g, kRows);
    const int low0 = kGrid == kClasses ? (int)((uint32_t)(reinterpret_cast<uintptr_t>(a.out) / sizeof(T)) +
                                               (uint32_t)walk.cls * (uint32_t)a.c) & (P::kWord - 1) : 0;
    const int at_warp = ((int)threadIdx.x % tpr & ~31) * 8 - low0, col0 = at_warp + ((int)threadIdx.x & 31) * P::kLane;
    auto col = [&](int p, int j) {  // the channel of value j of piece p
        return col0 + p * tpr * 8 + j / P::kWord * P::kNext + j % P::kWord;
    };
    uint32_t mask[kP];
#pragma unroll
    for (int p = 0; p < kP; ++p) {
        mask[p] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mask[p] |= (uint32_t)(0 <= col(p, j) && col(p, j) < a.c) << j;
    }
    // where this thread's part in the copies starts, and what a row has there (a piece's `part`)
    const int at0 = kGrid == kShifted ? col0 & ~255 : col0;
    auto there = [&](int p) { return kGrid == kShifted ? min(256, a.c - at0 - p * tpr * 8) : (int)mask[p]; };
    const int step = walk.step, m = walk.m;  // in rows of the class
    const int64_t c = a.c, next = c << walk.log;  // from a row of the class to the next one
    const float inv_c = 1.0f / (float)a.c;
    int left = m - walk.first;  // rows of the class from the group's next ones to the end
    const T* x = static_cast<const T*>(a.x);
    int64_t fetch_at = walk.row(walk.first) * c + at0;  // of the rows to fetch next
    auto fetch = [&](uint4* to, int rows) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int p = 0; p < kP; ++p)
                P::fetch(x + fetch_at + i * next + p * tpr * 8, i < rows ? there(p) : 0,
                         to + i * kRowWords + p * kPieceWords);
        copy_async_commit();
        fetch_at += step * next;
    };
    if (kGrid != kWhole) fill_nibbles(nibbles);
    griddep_wait_then_release();
    uint4* const mine = ring + (kGrid == kShifted ? ((int)threadIdx.x >> 5) * P::kWarpStride : (int)threadIdx.x);
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
                const bool here = mask[p] >> (2 * i + j) & 1;
                const int at = here ? col(p, 2 * i + j) : 0;
                const float s1 = 1.0f + vec_or<T>(a.scale, at, 0.0f);
                gv[j] = here ? s1 * vec_or<T>(a.weight, at, 1.0f) : 0.0f;
                bv[j] = here ? fmaf(vec_or<T>(a.bias, at, 0.0f), s1, vec_or<T>(a.shift, at, 0.0f)) : 0.0f;
            }
            gain[p][i] = f2(gv[0], gv[1]), base[p][i] = f2(bv[0], bv[1]);
        }
    int stage = 0;
    for (int cta_left = walk.cta_left; cta_left > 0; cta_left -= step, left -= step) {
        if (kGrid == kShifted) __syncwarp();  // the warp has read the stage that is filled now
        fetch(mine + (stage == 0 ? kStages - 1 : stage - 1) * kRows * kRowWords, left - (kStages - 1) * step);
        copy_async_wait<kStages - 1>();
        if (kGrid == kShifted) __syncwarp();  // and all its lanes' copies have arrived
        const uint4* now = mine + stage * kRows * kRowWords;
        float sum[kRows], sq[kRows];
        uint64_t f[kRows][kP][4];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            sum[i] = 0.0f;
#pragma unroll
            for (int p = 0; p < kP; ++p) {
                uint64_t(&v)[4] = f[i][p];
                P::read(now + i * kRowWords + p * kPieceWords, row_offset<kGrid>(x, m - left + i, a.c), v);
                P::clear(nibbles, mask[p], v);
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
                uint64_t(&d)[4] = f[i][p];
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] = fadd2(d[j], minus);
                P::clear(nibbles, mask[p], d);
#pragma unroll
                for (int w = 0; w < P::kWords; ++w) {
                    uint64_t q = 0;
#pragma unroll
                    for (int j = w * P::kWord / 2; j < (w + 1) * P::kWord / 2; ++j) q = ffma2(d[j], d[j], q);
                    if (kGrid != kWhole || P::of_word(mask[p], w) != 0) sq[i] += pair_sum(q);
                }
            }
        }
        group_sum<kRows>(sq, part[1], warp0, warps);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (i >= left) break;
            const float rstd = rsqrt_refined(fmaf(sq[i], inv_c, a.eps));
            const int r = walk.row(m - left + i);
            if ((int)threadIdx.x % tpr == 0) a.mean[r] = sum[i], a.rstd[r] = rstd;
            const uint64_t r2 = f2(rstd, rstd);
#pragma unroll
            for (int p = 0; p < kP; ++p) {
                if (there(p) <= 0) continue;
                uint64_t(&v)[4] = f[i][p];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = ffma2(fmul2(v[j], r2), gain[p][j], base[p][j]);
                P::store(static_cast<T*>(a.out) + r * c + at0 + p * tpr * 8, there(p), v);
            }
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    copy_async_wait<0>();
}

// kHeld: x is the 8-bit form; a piece of it is 8 bytes.
template <typename T, bool kHeld, Grid kGrid, int kRows, int kP, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads, kBackwardThreads / kMaxThreads > 1 ? kBackwardThreads / kMaxThreads : 1)
    norm_backward_kernel(const NormTrainArgs a, int tpr, int log_period) {
    constexpr int kStages = kBackwardStages;
    // dy's and n's values beside the row are cleared under one branch, but for two pieces of fp32 each, which spill so
    // (4339 × 7415 off the grid by different amounts 119 µs instead of 108)
    constexpr bool kOneClear = kHeld || kP * sizeof(T) < 8;
    // What only the kernel's end needs is found anew there: kept, it is spilled in the loop (17,280 × 1531 bf16 from 8 bits 67
    // instead of 66 µs, fp32 79 / 73; fp32 from fp32 is faster so, off the grid by different amounts 75 / 83).
    constexpr bool kAnew = kGrid == kShifted && (kHeld || sizeof(T) == 2);
    extern __shared__ uint4 ring[];  // [kStages][kRows][kP][words of dy][kMaxThreads], then the same of x (8 bytes if held)
    __shared__ alignas(16) float part[2][32 * 2 * kRows];
    __shared__ uint4 nibbles[kGrid == kWhole ? 1 : 16];
    using P = Piece<T, kGrid, kMaxThreads>;
    constexpr int kPieceWords = P::kStride, kRowWords = kP * kPieceWords;
    const int groups = (int)blockDim.x / tpr, g = (int)threadIdx.x / tpr, warps = tpr >> 5, warp0 = g * warps;
    const Walk walk((int)a.m, kGrid == kClasses ? log_period : 0, groups, g, kRows);
    const int low0 = kGrid == kClasses ? (int)((uint32_t)(reinterpret_cast<uintptr_t>(a.out) / sizeof(T)) +
                                               (uint32_t)walk.cls * (uint32_t)a.c) & (P::kWord - 1) : 0;
    const int at_warp = ((int)threadIdx.x % tpr & ~31) * 8 - low0, col0 = at_warp + ((int)threadIdx.x & 31) * P::kLane;
    auto col = [&](int p, int j) {  // the channel of value j of piece p
        return col0 + p * tpr * 8 + j / P::kWord * P::kNext + j % P::kWord;
    };
    uint32_t mask[kP];
#pragma unroll
    for (int p = 0; p < kP; ++p) {
        mask[p] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mask[p] |= (uint32_t)(0 <= col(p, j) && col(p, j) < a.c) << j;
    }
    // where this thread's part in the copies starts, and what a row has there (a piece's `part`)
    const int at0 = kGrid == kShifted ? col0 & ~255 : col0;
    auto there = [&](int p) { return kGrid == kShifted ? min(256, a.c - at0 - p * tpr * 8) : (int)mask[p]; };
    const int step = walk.step, m = walk.m;  // in rows of the class
    const int64_t c = a.c, next = c << walk.log, ld = fp8_ld(a.c);  // next: from a row of the class to the next one
    const float inv_c = -1.0f / (float)a.c;
    int left = m - walk.first;  // rows of the class from the group's next ones to the end
    const T *dy = static_cast<const T*>(a.dy), *x = static_cast<const T*>(a.x);
    const uint8_t* x8 = static_cast<const uint8_t*>(a.x);
    int64_t fetch_at = walk.row(walk.first) * c + at0, fetch_at8 = walk.first * ld + col0;  // of the rows to fetch next
    uint4* const mine = ring + (kGrid == kShifted ? ((int)threadIdx.x >> 5) * P::kWarpStride : (int)threadIdx.x);
    uint4* const mine_x = mine + kStages * kRows * kRowWords;
    // the 8-bit form: a piece's eight bytes, or four of each of its words
    constexpr int kParts = kGrid == kShifted ? 1 : P::kWords;
    using Part = typename PartOf<kParts>::type;
    Part* const mine_x8 = reinterpret_cast<Part*>(ring + kStages * kRows * kRowWords) + threadIdx.x;
    auto fetch = [&](int stage, int rows) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int p = 0; p < kP; ++p) {
                const int n = i < rows ? there(p) : 0, piece = (stage * kRows + i) * kP + p;
                P::fetch(dy + fetch_at + i * next + p * tpr * 8, n, mine + piece * kPieceWords);
                if constexpr (kHeld)
#pragma unroll
                    for (int w = 0; w < kParts; ++w)
                        copy_async<8 / kParts>(mine_x8 + (piece * kParts + w) * kMaxThreads,
                                               x8 + fetch_at8 + i * ld + p * tpr * 8 + w * P::kNext,
                                               i < rows && (kParts == 1 ? mask[p] : P::of_word(mask[p], w)) != 0);
                else
                    P::fetch(x + fetch_at + i * next + p * tpr * 8, n, mine_x + piece * kPieceWords);
            }
        copy_async_commit();
        fetch_at += step * next;
        if (kHeld) fetch_at8 += step * ld;
    };
    // the rows' statistics (and codes) one step ahead, in registers; past the last row that row's, but rstd 0: n is zero there
    // as dy is, where −mean · rstd may be infinite
    float next_mean[kRows], next_rstd[kRows];
    uint32_t next_code[kRows][kP];
    const int tile_bytes = (int)fp8_scale_tiles(a.c) * 512;
    int code_at[kP];
#pragma unroll
    for (int p = 0; p < kP; ++p) {
        const int block = (min(col(p, 0), a.c - 1) >> 7) & -kParts;  // with two parts, the second is of the next block
        code_at[p] = (block >> 2) * 512 + (block & 3);
    }
    auto fetch_row = [&](int rows) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = min(walk.row(m - rows + i), (int)a.m - 1);
            next_mean[i] = a.mean[r], next_rstd[i] = i < rows ? a.rstd[r] : 0.0f;
#pragma unroll
            for (int p = 0; p < kP; ++p)
                if (kHeld) {
                    const uint8_t* code =
                        a.x_scale + (int64_t)(r >> 7) * tile_bytes + (r & 31) * 16 + ((r >> 5) & 3) * 4 + code_at[p];
                    next_code[i][p] = kParts == 1 ? *code : *reinterpret_cast<const uint16_t*>(code);
                }
        }
    };
    if (kGrid != kWhole) fill_nibbles(nibbles);
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
                const bool here = mask[p] >> (2 * i + j) & 1;
                const int at = here ? col(p, 2 * i + j) : 0;
                gv[j] = here ? (1.0f + vec_or<T>(a.scale, at, 0.0f)) * vec_or<T>(a.weight, at, 1.0f) : 0.0f;
            }
            gain[p][i] = f2(gv[0], gv[1]);
            sum_a[p][i] = sum_b[p][i] = 0;
        }
    int stage = 0, flip = 0;
    for (int cta_left = walk.cta_left; cta_left > 0; cta_left -= step, left -= step, flip ^= 1) {
        if (kGrid == kShifted) __syncwarp();  // the warp has read the stage that is filled now
        fetch(stage == 0 ? kStages - 1 : stage - 1, left - (kStages - 1) * step);
        copy_async_wait<kStages - 1>();
        if (kGrid == kShifted) __syncwarp();  // and all its lanes' copies have arrived
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
                P::read(mine + piece * kPieceWords, row_offset<kGrid>(dy, m - left + i, a.c), d);
                if constexpr (!kOneClear) P::clear(nibbles, mask[p], d);
                if constexpr (kHeld) {
                    uint32_t u[2];
                    float down[2];
                    if constexpr (kParts == 1) {
                        const uint2 both = mine_x8[piece * kMaxThreads];
                        u[0] = both.x, u[1] = both.y, down[0] = down[1] = fp8_down(next_code[i][p]);
                    } else {
                        u[0] = mine_x8[piece * 2 * kMaxThreads], u[1] = mine_x8[(piece * 2 + 1) * kMaxThreads];
                        down[0] = fp8_down(next_code[i][p] & 255u), down[1] = fp8_down(next_code[i][p] >> 8);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {  // the scaling is exact: one rounding, in the subtraction
                        float lo, hi;
                        fp8_unpack2(u[j >> 1] >> (16 * (j & 1)), lo, hi);
                        n[j] = ffma2(f2(lo, hi), f2(down[j >> 1], down[j >> 1]), minus);
                    }
                } else {
                    P::read(mine_x + piece * kPieceWords, row_offset<kGrid>(x, m - left + i, a.c), n);
#pragma unroll
                    for (int j = 0; j < 4; ++j) n[j] = fadd2(n[j], minus);
                }
                // n after the subtraction: zero beside the row, not −mean · rstd
                if constexpr (kOneClear)
                    P::clear(nibbles, mask[p], d, n);
                else
                    P::clear(nibbles, mask[p], n);
                uint64_t s1 = 0, s2 = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // a word beside the row (bf16: the whole piece, below): n as P::clear leaves it
                    const bool none = kGrid == kWhole && P::kWords == 2 && P::of_word(mask[p], 2 * j / P::kWord) == 0;
                    n[j] = fmul2(n[j], none ? 0 : r2);
                    sum_a[p][j] = ffma2(d[j], n[j], sum_a[p][j]);
                    sum_b[p][j] = fadd2(sum_b[p][j], d[j]);
                    d[j] = fmul2(d[j], gain[p][j]);
                    s1 = fadd2(s1, d[j]);
                    s2 = ffma2(d[j], n[j], s2);
                }
                s[2 * i] += pair_sum(s1);
                if (kGrid != kWhole || P::kWords == 2 || mask[p] != 0) s[2 * i + 1] += pair_sum(s2);
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
                if (there(p) <= 0) continue;
                uint64_t f[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = fmul2(ffma2(norm[i][p][j], c2p, fadd2(grad[i][p][j], c1p)), r2);
                P::store(static_cast<T*>(a.out) + walk.row(m - left + i) * c + at0 + p * tpr * 8, there(p), f);
            }
        }
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    copy_async_wait<0>();
    // the CTA's sums: its only group's, or the groups' in order, through the ring (by channel: the pieces of groups of
    // different classes lie differently)
    float* to = a.partial + (int64_t)blockIdx.x * 2 * a.c;
    int tid = threadIdx.x;
    if constexpr (kAnew) asm volatile("" : "+r"(tid));  // not the tid that g, col0 and the masks are known for
    float* const own = groups > 1 ? reinterpret_cast<float*>(ring) + tid / tpr * 2 * a.c : to;
    auto end_col = [&](int p, int j) { return kAnew ? tid % tpr * 8 + p * tpr * 8 + j : col(p, j); };
    if (groups > 1) __syncthreads();
#pragma unroll
    for (int p = 0; p < kP; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float av[2], bv[2];
            uf2(sum_a[p][i], av[0], av[1]);
            uf2(sum_b[p][i], bv[0], bv[1]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (const int at = end_col(p, 2 * i + j); kAnew ? at < a.c : mask[p] >> (2 * i + j) & 1)
                    own[at] = av[j], own[a.c + at] = bv[j];
        }
    if (groups == 1) return;
    __syncthreads();
    const float* held = reinterpret_cast<const float*>(ring);
    for (int i = threadIdx.x; i < 2 * a.c; i += blockDim.x) {
        float sum = held[i];
        for (int o = 1; o < groups; ++o) sum += held[o * 2 * a.c + i];
        to[i] = sum;
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
// µs, backward 59 / 54); below two are slower (1536: forward 26 / 22, backward 50 / 37; 4096: 33 / 32 and 52 / 49).
struct Shape {
    int pieces, tpr, threads, groups, log_period;
    // word: values in 16 bytes. kClasses: up to word − 1 values more in front of a row, and rows are alike again after
    // word / gcd(c, word).
    Shape(int c, Grid grid, int word) : log_period(0) {
        if (grid == kClasses)
            while (((int64_t)c << log_period) % word) ++log_period;
        const int n = c + (grid == kClasses ? word - 1 : 0);
        pieces = n > 4096 ? 2 : 1;
        tpr = ((n + 8 * pieces - 1) / (8 * pieces) + 31) / 32 * 32;
        groups = tpr >= 256 ? 1 : 256 / tpr;
        threads = tpr * groups;
    }
    // As many groups of threads of each class (a power of two, as `groups` is).
    int ctas(int64_t m, int rows, int sm_threads) const {
        const int64_t period = (int64_t)1 << log_period, unit = period > groups ? period / groups : 1;
        const int64_t sets = ((m + period - 1) / period + rows - 1) / rows * period;
        const int64_t need = ((sets + groups - 1) / groups + unit - 1) / unit * unit;
        const int64_t most = (int64_t)sm_count() * (sm_threads > threads ? sm_threads / threads : 1) / unit * unit;
        return (int)(need < most ? need : most);
    }
    int backward_ctas(int64_t m) const { return ctas(m, pieces == 1 ? kBackwardRows : 1, kBackwardThreads); }
};

// Offsets from the 16-byte grid decide; with kClasses a row may need more threads than a CTA has here (above 8185 channels).
template <typename T>
Grid grid_of(int c, const void* x, const void* y, const void* z, bool held) {
    auto off = [](const void* p) { return (int)(reinterpret_cast<uintptr_t>(p) & 15); };
    if (c % 8 == 0 && !(off(x) || off(y) || off(z))) return kWhole;
    const bool alike = off(x) == off(y) && off(y) == off(z);
    return !held && alike && Shape(c, kClasses, 16 / sizeof(T)).threads <= 512 ? kClasses : kShifted;
}

template <auto kernel>
cudaError_t launch_ring(int ctas, const Shape& s, size_t ring_bytes, const NormTrainArgs& a, cudaStream_t st) {
    if (ring_bytes > 40 * 1024) {
        cudaError_t e = allow_smem<kernel>(ring_bytes);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(kernel, dim3(ctas), dim3(s.threads), ring_bytes, st, a, s.tpr, s.log_period);
}

template <typename T, Grid kGrid, int kRows, int kP, int kMaxThreads>
cudaError_t train_threads(const NormTrainArgs& a, const Shape& s, cudaStream_t st) {
    const size_t ring = (size_t)16 * kStages * kRows * kP * Piece<T, kGrid, kMaxThreads>::kStride;
    return launch_ring<norm_train_kernel<T, kGrid, kRows, kP, kMaxThreads>>(s.ctas(a.m, kRows, kForwardThreads), s, ring, a,
                                                                            st);
}

template <typename T, Grid kGrid, int kRows, int kP>
cudaError_t train_pieces(const NormTrainArgs& a, const Shape& s, cudaStream_t st) {
    if constexpr (kP == 1) {  // two pieces: more than 256 threads
        if (s.threads <= 192) return train_threads<T, kGrid, kRows, kP, 192>(a, s, st);
        if (s.threads <= 256) return train_threads<T, kGrid, kRows, kP, 256>(a, s, st);
    }
    return train_threads<T, kGrid, kRows, kP, 512>(a, s, st);
}

template <typename T, Grid kGrid>
cudaError_t train_grid(const NormTrainArgs& a, cudaStream_t st) {
    constexpr int kRows = sizeof(T) == 2 ? 4 : 2;
    const Shape s(a.c, kGrid, 16 / sizeof(T));
    return s.pieces == 1 ? train_pieces<T, kGrid, kRows, 1>(a, s, st) : train_pieces<T, kGrid, kRows / 2, 2>(a, s, st);
}

template <typename T>
cudaError_t train(const NormTrainArgs& a, cudaStream_t st) {
    const Grid grid = grid_of<T>(a.c, a.x, a.out, a.out, false);
    return grid == kWhole ? train_grid<T, kWhole>(a, st)
                          : grid == kClasses ? train_grid<T, kClasses>(a, st) : train_grid<T, kShifted>(a, st);
}

template <typename T, bool kHeld, Grid kGrid, int kRows, int kP, int kMaxThreads>
cudaError_t backward_threads(const NormTrainArgs& a, const Shape& s, cudaStream_t st) {
    constexpr int kDy = 16 * Piece<T, kGrid, kMaxThreads>::kStride, kX = kHeld ? 8 * kMaxThreads : kDy;
    const size_t ring = (size_t)kBackwardStages * kRows * kP * (kDy + kX);
    return launch_ring<norm_backward_kernel<T, kHeld, kGrid, kRows, kP, kMaxThreads>>(s.backward_ctas(a.m), s, ring, a, st);
}

template <typename T, bool kHeld, Grid kGrid, int kRows, int kP>
cudaError_t backward_pieces(const NormTrainArgs& a, const Shape& s, cudaStream_t st) {
    if constexpr (kP == 1) {  // two pieces: more than 256 threads
        if (s.threads <= 192) return backward_threads<T, kHeld, kGrid, kRows, kP, 192>(a, s, st);
        if (s.threads <= 256) return backward_threads<T, kHeld, kGrid, kRows, kP, 256>(a, s, st);
    }
    return backward_threads<T, kHeld, kGrid, kRows, kP, 512>(a, s, st);
}

template <typename T, bool kHeld, Grid kGrid>
cudaError_t backward_grid(const NormTrainArgs& a, const Shape& s, cudaStream_t st) {
    return s.pieces == 1 ? backward_pieces<T, kHeld, kGrid, kBackwardRows, 1>(a, s, st)
                         : backward_pieces<T, kHeld, kGrid, 1, 2>(a, s, st);
}

template <typename T>
cudaError_t backward(const NormTrainArgs& a, cudaStream_t st) {
    const bool held = a.x_scale;
    const Grid grid = grid_of<T>(a.c, a.dy, a.out, held ? a.out : a.x, held);
    const Shape s(a.c, grid, 16 / sizeof(T));
    cudaError_t e = cudaSuccess;
    if (a.m > 0) {
        if (held)
            e = grid == kWhole ? backward_grid<T, true, kWhole>(a, s, st) : backward_grid<T, true, kShifted>(a, s, st);
        else
            e = grid == kWhole ? backward_grid<T, false, kWhole>(a, s, st)
                               : grid == kClasses ? backward_grid<T, false, kClasses>(a, s, st)
                                                  : backward_grid<T, false, kShifted>(a, s, st);
    }
    if (e != cudaSuccess || !(a.dweight || a.dbias || a.dscale || a.dshift)) return e;
    return launch_pdl(norm_vectors_kernel<T>, dim3((a.c + 7) / 8), dim3(512), 0, st, a, a.m > 0 ? s.backward_ctas(a.m) : 0);
}

}  // namespace

// Of any grid and type.
int norm_backward_ctas(int64_t m, int c) {
    int most = 0;
    for (int word = 4; word <= 8; word += 4)
        for (const Grid grid : {kShifted, kClasses}) most = std::max(most, Shape(c, grid, word).backward_ctas(m));
    return most;
}

cudaError_t launch_layernorm_train(const NormTrainArgs& a, cudaStream_t st) {
    if (a.m <= 0) return cudaSuccess;
    return a.dtype == FVSR_BF16 ? train<__nv_bfloat16>(a, st) : train<float>(a, st);
}

cudaError_t launch_layernorm_backward(const NormTrainArgs& a, cudaStream_t st) {
    return a.dtype == FVSR_BF16 ? backward<__nv_bfloat16>(a, st) : backward<float>(a, st);
}

}  // namespace fvsr
