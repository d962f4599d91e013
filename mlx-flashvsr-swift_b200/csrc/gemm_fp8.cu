// gemm_fp8.cu — the linear layers on 8-bit operands: out = epilogue(x · wᵀ + bias), x (M, K) and w (N, K) in the 8-bit
// form of fp8.cuh (a scale for each block of 128 along K), fp32 sums, one rounding at the end.
//
//   out[m][n] = epi(Σ_b 2^(ex[m][b] + ew[n][b]) · Σ_{k in block b} x8[m][k]·w8[n][k] + bias[n])
//
// The scales are powers of two in the layout tensor memory wants, so the tensor core applies them itself
// (tcgen05 kind::mxf8f6f4, one scale for 32 values along K): the four MMAs of a 128-wide block name the same byte of the
// scale words, and one 512-byte copy to tensor memory serves 128 rows × 4 blocks. Nothing is promoted or rescaled in
// registers, and a weight gradient (a scale for each row and block on both sides) costs what a forward product does.
//
// Persistent kernel over CTA pairs (clusters of two CTAs, one TPC): a pair walks 256 × 256 output tiles, CTA r of it
// loading rows [m0 + 128r, +128) of x and [n0 + 128r, +128) of w per 128-wide K step (32 KB a stage, 5 stages) and, every
// fourth step, the codes of its 128 rows of x and of all 256 rows of w. Warp roles (320 threads per CTA):
//   warp 0      TMA producer;
//   warp 1      TMEM owner and, in the even CTA, the issuer of the scale copies and MMAs (M 256, N 256, K 32);
//   warps 2..9  epilogue: thread = output row = TMEM lane, each half of the warps 128 of the tile's columns, 32 at a time
//               through shared memory in the layout a TMA store takes (16-byte words swizzled, so that the threads'
//               writes meet no bank conflicts). The residual, where there is one, arrives by TMA in the place the result
//               is written to. (Stores straight from the threads, a row each and 32 rows an instruction, cost 13 % of
//               the whole product at K = 1536.) Rows that are not 16-byte aligned take the same way through shared
//               memory and are read and written a row at a time, a lane a column.
// The first two warps walk the tiles as whole warps and issue under elect_one: issued by `lane == 0`, a step's four MMAs
// and its wait took 720 cycles instead of the MMAs' 512, whatever the ring's depth.
// Tensor memory (512 columns): accumulator 0 in [0, 256), accumulator 1 in [240, 496), the scales in [496, 508). The two
// accumulators share 16 columns, which an epilogue reads first and releases (ovl) before anything else, so the next
// tile's MMAs start some hundred cycles into the epilogue and run beside the rest of it.
// The epilogue's signals that an accumulator is free carry no release at cluster scope, which waited for its stores (a
// tile took 1900 cycles longer: 162 instead of 138 us below).
// Measured on operands of zeros, which leave the clock at its highest: 17280 × 8960 × 1536 138 us = 3442 TFLOP/s, with GELU 153;
// 17280 × 1536 × 8960 129 us = 3694. 4 stages 151, 150 and 148 us; groups of 8 tile rows 146, 152 and 130. On random
// values the clock falls to 1.5 GHz at 1000 W and energy decides: 180 us = 2644 TFLOP/s, 195 and (gated) 183.
// Not kept, measured before the two lines above held: 256 × 384 tiles in two accumulators of 192 columns, and sixteen
// epilogue warps (each slower than 256 × 256 and eight, but GELU with sixteen).
//
// The tensor core adds to its fp32 accumulator by truncation, an error that grows with the number of additions and, where
// the products have one sign, is a bias. Measured in one chain, relative to the result, zero-mean / one-signed operands:
// K = 4096 2.2e-7 / 1.5e-6, 8960 6e-7 / 4.4e-6, 17280 1.3e-6 / 1.1e-5, 65536 5e-6 / 6e-5, 262144 4.3e-5 / 4.2e-4 (sums that
// round, in torch: 8e-8 / 2.3e-7 at 4096). For an fp32 output the sum is therefore taken in chains of 4096, which the
// epilogue adds up with rounding, in the output itself (2.3e-7 / 1.5e-6 whatever K): the accumulators alternate between
// chains as between tiles. A bf16 output, whose rounding is 3.9e-3, is one chain up to 65536 (1/64 of that); beyond, its
// chains are added up in an fp32 plane of the workspace, as the partial sums below are.
// When the tiles are fewer than half the pairs, the sum over K is cut into parts (whole tiles of codes, 512 wide) that
// leave fp32 partial products; a second kernel adds them in order and applies the epilogue.
// Every wait is bounded (4 s); on expiry the kernel raises its abort and device timeout words, skips the rest of its
// work and fvsr_device_check reports FVSR_ETIMEOUT.
#include "../../include/fvsr_lcsa.h"
#include "common.cuh"
#include "fp8.cuh"
#include "fp8_epilogue.cuh"
#include "sm100.cuh"
#include "unaligned.cuh"

namespace fvsr {

__device__ int g_gemm_fp8_timeout = 0;

namespace {

using namespace sm100;

constexpr int kBM = 256, kBN = 256, kBK = 128, kStages = 5;
constexpr uint32_t kHalfBytes = 128 * kBK;       // 16 KB: one CTA's rows of x or of w per K step
constexpr uint32_t kStageBytes = 2 * kHalfBytes;
constexpr uint32_t kScaleBytes = 3 * 512;        // x's 128 rows, w's 256 rows, four blocks
constexpr int kThreads = 320;
constexpr int kEpiWarps = 8, kEpiThreads = 32 * kEpiWarps;
constexpr int kChainBlocks = 32, kLongChainBlocks = 512;  // of 128: the longest chains of an fp32 and of a bf16 output
constexpr uint64_t kWaitLimitNs = 4000000000ull;
constexpr uint32_t kIdesc = idesc_mxf8(kBM, kBN);
constexpr uint32_t kAcc1 = 240, kTmemScale = 496;
constexpr uint32_t kChunkRoom = 4096;            // an epilogue warp's chunks: 2 of 32 × 32 bf16 or 1 of fp32
constexpr int kBarFull = 0, kBarEmpty = kStages, kBarAccFull = 2 * kStages, kBarAccEmpty = 2 * kStages + 2,
              kBarOvl = 2 * kStages + 4, kBarSrc = 2 * kStages + 5, kNumBars = kBarSrc + 2 * kEpiWarps;
constexpr uint32_t kOffChunks = kStages * kStageBytes;
constexpr uint32_t kOffScale = kOffChunks + kEpiWarps * kChunkRoom;
constexpr uint32_t kOffBar = kOffScale + kStages * kScaleBytes;
constexpr uint32_t kOffTmemSlot = kOffBar + 8 * kNumBars;
constexpr uint32_t kOffAbort = kOffTmemSlot + 4;
constexpr uint32_t kOffCols = (kOffAbort + 4 + 15) & ~15u;  // bias[256], gate[256] as fp32, of this tile and the next
constexpr uint32_t kSmemBytes = 1024 + kOffCols + 4 * kBN * 4;
static_assert(kSmemBytes <= 232448, "shared memory");

struct Work {
    int mt, nt, kt, splits, part_blocks, chain_blocks;
    int tma;  // rows of out (and resid) are 16-byte aligned
};

template <typename T, int kMode>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_fp8_sm100_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                          const __grid_constant__ CUtensorMap tmXS, const __grid_constant__ CUtensorMap tmWS,
                          const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmResid,
                          const Fp8GemmArgs a, const Work wk) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = (int)(blockIdx.x >> 1), npairs = (int)(gridDim.x >> 1);
    const int items = wk.mt * wk.nt * wk.splits;
    volatile uint32_t* abort_word = reinterpret_cast<volatile uint32_t*>(smem + kOffAbort);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kOffTmemSlot);
    auto bar = [&](int i) { return sbase + kOffBar + 8u * (uint32_t)i; };
    auto wait = [&](int b, uint32_t parity) {
        return mbar_wait(bar(b), parity & 1u, abort_word, &g_gemm_fp8_timeout, kWaitLimitNs);
    };
    // for a whole warp
    auto wait_all = [&](int b, uint32_t parity) { return __all_sync(0xffffffffu, wait(b, parity)) != 0; };
    // item → output tile (columns fastest) and blocks [kb0, kb1) of K
    auto place = [&](int t, int& m0, int& n0, int& kb0, int& kb1) {
        const int tile = t / wk.splits, part = t % wk.splits;
        m0 = tile / wk.nt * kBM, n0 = tile % wk.nt * kBN;
        kb0 = part * wk.part_blocks, kb1 = min(kb0 + wk.part_blocks, wk.kt);
    };
    if (threadIdx.x == 0) {
        for (int st = 0; st < kStages; ++st) {
            mbar_init(bar(kBarFull + st), 1);
            mbar_init(bar(kBarEmpty + st), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar(kBarAccFull + b), 1);
            mbar_init(bar(kBarAccEmpty + b), 2 * kEpiWarps);
        }
        mbar_init(bar(kBarOvl), kEpiWarps);
        for (int b = 0; b < 2 * kEpiWarps; ++b) mbar_init(bar(kBarSrc + b), 1);
        *abort_word = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmX);
        prefetch_tmap(&tmW);
        prefetch_tmap(&tmXS);
        prefetch_tmap(&tmWS);
        prefetch_tmap(&tmOut);
    }
    griddep_wait_then_release();
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_slot), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();  // both CTAs' barriers are initialised and their TMEM allocated before any remote signal
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ---------------- TMA producer: rows past the tensors' ends read as zeros with scale code 0 ----------------
        {
            const bool issuer = elect_one();
            uint32_t it = 0;
            bool ok = true;
            for (int t = pair; ok && t < items; t += npairs) {
                int m0, n0, kb0, kb1;
                place(t, m0, n0, kb0, kb1);
                m0 += 128 * (int)rank;
                const int nr = n0 + 128 * (int)rank;
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int st = (int)(it % kStages);
                    if (it >= kStages && !(ok = wait_all(kBarEmpty + st, it / kStages - 1))) break;
                    const uint32_t dst = sbase + (uint32_t)st * kStageBytes;
                    const uint32_t sdst = sbase + kOffScale + (uint32_t)st * kScaleBytes;
                    const uint32_t full0 = mapa_shared(bar(kBarFull + st), 0);
                    const bool scales = (kb & 3) == 0;
                    if (!issuer) continue;
                    if (rank == 0) mbar_expect_tx(bar(kBarFull + st), 2 * (kStageBytes + (scales ? kScaleBytes : 0)));
                    tma_load_2d_pair(dst, &tmX, kb * kBK, m0, full0);
                    tma_load_2d_pair(dst + kHalfBytes, &tmW, kb * kBK, nr, full0);
                    if (scales) {
                        const int g = kb >> 2, kt4 = (wk.kt + 3) >> 2;
                        tma_load_2d_pair(sdst, &tmXS, 0, (m0 >> 7) * kt4 + g, full0);
                        tma_load_2d_pair(sdst + 512, &tmWS, 0, (n0 >> 7) * kt4 + g, full0);
                        tma_load_2d_pair(sdst + 1024, &tmWS, 0, ((n0 >> 7) + 1) * kt4 + g, full0);
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer: one lane of the even CTA, its warp walking the tiles with it ----------------
        if (rank == 0) {
            const bool issuer = elect_one();
            uint32_t it = 0;
            bool ok = true;
            int lt = 0;
            for (int t = pair; ok && t < items; t += npairs) {
                int m0, n0, kb0, kb1;
                place(t, m0, n0, kb0, kb1);
                for (int cb = kb0; ok && cb < kb1; cb += wk.chain_blocks, ++lt) {
                    const int acc = lt & 1, ce = min(cb + wk.chain_blocks, kb1);
                    if (lt >= 2 && !(ok = wait_all(kBarAccEmpty + acc, (uint32_t)((lt >> 1) - 1)))) break;
                    if (lt >= 1 && !(ok = wait_all(kBarOvl, (uint32_t)(lt - 1)))) break;
                    tc_fence_after();
                    const uint32_t d = tmem + (acc ? kAcc1 : 0u), sf = tmem + kTmemScale;
                    for (int kb = cb; kb < ce; ++kb, ++it) {
                        const int st = (int)(it % kStages);
                        if (!(ok = wait_all(kBarFull + st, it / kStages))) break;
                        tc_fence_after();
                        if (!issuer) continue;
                        const uint32_t sa = sbase + (uint32_t)st * kStageBytes;
                        if ((kb & 3) == 0) {
                            const uint32_t sc = sbase + kOffScale + (uint32_t)st * kScaleBytes;
                            tmem_cp_scales_pair(sf, scale_desc(sc));
                            tmem_cp_scales_pair(sf + 4, scale_desc(sc + 512));
                            tmem_cp_scales_pair(sf + 8, scale_desc(sc + 1024));
                        }
                        const uint64_t ad = smem_desc(sa, 16, 1024);
                        const uint64_t bd = smem_desc(sa + kHalfBytes, 16, 1024);
                        const uint32_t idesc = kIdesc | idesc_sf_id((uint32_t)kb & 3u);
#pragma unroll
                        for (int kk = 0; kk < kBK / 32; ++kk)
                            mma_mxf8_pair(d, ad + (uint64_t)(2 * kk), bd + (uint64_t)(2 * kk), idesc, sf, sf + 4,
                                          (kb > cb || kk > 0) ? 1u : 0u);
                        mma_commit_both(bar(kBarEmpty + st));
                    }
                    if (ok && issuer) mma_commit_both(bar(kBarAccFull + acc));
                }
            }
        }
    } else {
        // ---------------- epilogue: this CTA's 128 rows; thread = row = TMEM lane, half = which 128 columns ----------------
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int et = threadIdx.x - 64;
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * (kBN / 2));
        // a thread's column of bias and gate, for the tile's 256 columns: fetched for the next tile under this one's work
        float* const cols = reinterpret_cast<float*>(smem + kOffCols);
        float next_bias = 0.0f, next_gate = 0.0f;
        auto fetch_cols = [&](int t) {
            int m0, n0, kb0, kb1;
            place(t, m0, n0, kb0, kb1);
            const int c = n0 + et;
            next_bias = next_gate = 0.0f;
            if (t < items && c < a.N) {
                if (a.bias) next_bias = __bfloat162float(a.bias[c]);
                if (kMode == FVSR_LINEAR_GATED_RESIDUAL) next_gate = __bfloat162float(a.gate[c]);
            }
        };
        auto put_cols = [&](int buffer) {
            cols[buffer * 2 * kBN + et] = next_bias;
            if (kMode == FVSR_LINEAR_GATED_RESIDUAL) cols[buffer * 2 * kBN + kBN + et] = next_gate;
        };
        const uint32_t acc_empty0 = mapa_shared(bar(kBarAccEmpty), 0), ovl0 = mapa_shared(bar(kBarOvl), 0);
        const bool leader = elect_one();  // issues the warp's copies and signals
        constexpr bool kBf16 = sizeof(T) == 2;
        constexpr bool kAdds = !kBf16 || kMode == FVSR_LINEAR_GATED_RESIDUAL;  // something may be added to the products
        constexpr int kRoom = kBf16 ? 2 : 1;  // chunks in flight
        constexpr uint32_t kRowBytes = 32 * sizeof(T), kChunkBytes = 32 * kRowBytes;
        uint8_t* const chunks = smem + kOffChunks + (uint32_t)(warp - 2) * kChunkRoom;
        const uint32_t swizzle = (kBf16 ? (uint32_t)lane >> 1 & 3u : (uint32_t)lane & 7u) << 4;
        const int src_bar = kBarSrc + 2 * (warp - 2);
        uint32_t src_phase = 0;  // bit b: parity of the next wait on chunk place b
        int lt = 0, buffer = 0;
        bool ok = true;
        fetch_cols(pair);
        put_cols(0);
        for (int t = pair; t < items; t += npairs, buffer ^= 1) {
            int m0, n0, kb0, kb1;
            place(t, m0, n0, kb0, kb1);
            named_barrier_sync(1, kEpiThreads);  // the tile's columns are there, the other buffer's are done with
            const float *bias_s = cols + buffer * 2 * kBN, *gate_s = bias_s + kBN;
            fetch_cols(t + npairs);
            const int row0 = m0 + 128 * (int)rank + quarter * 32, plane = t % wk.splits;
            const int c0 = n0 + half * (kBN / 2);
            const float *bcol = bias_s + half * (kBN / 2), *gcol = gate_s + half * (kBN / 2);
            for (int cb = kb0; cb < kb1; cb += wk.chain_blocks, ++lt) {
                const int acc = lt & 1;
                const bool first = cb == kb0, last = cb + wk.chain_blocks >= kb1;
                // something to add: the chains before (an fp32 output's), the residual
                const bool src = kAdds && (kMode == FVSR_LINEAR_GATED_RESIDUAL || !first);
                // accumulator 0 from its last chunk to its first, accumulator 1 from its first: the shared columns come first
                auto chunk = [&](int i) { return acc ? i : kBN / 64 - 1 - i; };
                auto live = [&](int c) { return row0 < a.M && c0 + 32 * c < a.N; };
                auto fetch = [&](int i) {  // by the leader: the values to add to chunk i into its place
                    const int c = chunk(i);
                    if (!live(c)) return;
                    const uint32_t b = bar(src_bar + i % kRoom);
                    mbar_expect_tx(b, kChunkBytes);
                    tma_load_3d(smem_u32(chunks + (i % kRoom) * kChunkBytes), first ? &tmResid : &tmOut, c0 + 32 * c,
                                row0, plane, b);
                };
                if (wk.tma && src && ok && leader) {
                    if (first) bulk_wait_read<0>();
                    else bulk_wait<0>();  // the chain before is in memory
                    for (int i = 0; i < kRoom; ++i) fetch(i);
                }
                if (ok) ok = __all_sync(0xffffffffu, wait(kBarAccFull + acc, (uint32_t)(lt >> 1)));
                if (!ok) continue;
                tc_fence_after();
                const uint32_t tbase = lane_base + (acc ? kAcc1 : 0u);
                auto emit = [&](const uint32_t* v, int i) {
                    const int c = chunk(i);
                    const float *bias = bcol + 32 * c, *gate = gcol + 32 * c;
                    auto fetch_next = [&] {  // by the leader, once this chunk's place is free again
                        if (src && i + kRoom < kBN / 64) {
                            bulk_wait_read<0>();
                            fetch(i + kRoom);
                        }
                    };
                    if (!live(c)) {
                        if (wk.tma && leader) {
                            bulk_commit();  // keeps the groups' count
                            fetch_next();
                        }
                        return;
                    }
                    const int place_i = i % kRoom;
                    uint8_t* const room = chunks + place_i * kChunkBytes;
                    uint8_t* const mine = room + (uint32_t)lane * kRowBytes;
                    // without TMA: lane = column, row by row (each element always the same lane's)
                    const int rows = min(32, a.M - row0);
                    const bool col_here = c0 + 32 * c + lane < a.N;
                    const int64_t corner = (int64_t)row0 * a.N + c0 + 32 * c + lane;
                    auto element = [&](int r) {
                        const uint32_t byte = (uint32_t)lane * (uint32_t)sizeof(T);
                        const uint32_t word = (byte >> 4) ^ (kBf16 ? (uint32_t)r >> 1 & 3u : (uint32_t)r & 7u);
                        return reinterpret_cast<T*>(room + (uint32_t)r * kRowBytes + (word << 4) + (byte & 15u));
                    };
                    if (wk.tma && src) {
                        const bool here = wait(src_bar + place_i, src_phase >> place_i);
                        src_phase ^= 1u << place_i;
                        if (!__all_sync(0xffffffffu, here)) ok = false;
                    } else if (wk.tma) {
                        if (leader) bulk_wait_read<kRoom - 1>();
                        __syncwarp();
                    } else if (src && first) {
                        // the residual: lane = row, which reads the aligned words that hold its 32 values (9492 × 2527 × 94
                        // bf16 66 µs, lane = column 75; 17,280 × 1537 × 1536 87 / 93)
                        const T* p = static_cast<const T*>(a.resid) + (int64_t)(row0 + lane) * a.N + c0 + 32 * c;
                        const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15);
                        const int end = lane < rows ? off + min(32, a.N - (c0 + 32 * c)) * (int)sizeof(T) : 0;
                        const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p) - off);
                        __syncwarp();
#pragma unroll 1
                        for (int h = 0; h < (int)sizeof(T) / 2; ++h) {  // 64 bytes at a time
                            uint32_t got[20], o[16];
#pragma unroll
                            for (int i = 0; i < 5; ++i) {
                                const uint4 u = 64 * h + 16 * i < end ? from[4 * h + i] : make_uint4(0, 0, 0, 0);
                                got[4 * i] = u.x, got[4 * i + 1] = u.y, got[4 * i + 2] = u.z, got[4 * i + 3] = u.w;
                            }
                            shift_bytes<sizeof(T), 16>(got, (uint32_t)off, o);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                *reinterpret_cast<uint4*>(mine + (((uint32_t)(4 * h + i) << 4) ^ swizzle)) =
                                    make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                    } else if (src) {
                        const T* from = static_cast<const T*>(a.out) + corner;
                        __syncwarp();
#pragma unroll 1
                        for (int r0 = 0; r0 < 32; r0 += 16) {
                            T got[16];  // in flight at once
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                got[r] = col_here && r0 + r < rows ? from[(int64_t)(r0 + r) * a.N] : T(0.0f);
#pragma unroll
                            for (int r = 0; r < 16; ++r) *element(r0 + r) = got[r];
                        }
                        __syncwarp();
                    } else {
                        __syncwarp();
                    }
                    constexpr int kPairs = 8 / sizeof(T);  // of a 16-byte word
#pragma unroll
                    for (int w = 0; w < 16 / kPairs; ++w) {
                        uint4* at = reinterpret_cast<uint4*>(mine + (((uint32_t)w << 4) ^ swizzle));
                        uint64_t add[kPairs] = {}, y[kPairs];
                        if (src) {
                            if constexpr (kBf16) {
                                const uint4 u = *at;
                                const uint32_t p[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                                for (int e = 0; e < kPairs; ++e) {
                                    float lo, hi;
                                    bf2_to_f(p[e & 3], lo, hi);
                                    add[e] = f2(lo, hi);
                                }
                            } else {
                                const ulonglong2 u = *reinterpret_cast<const ulonglong2*>(at);
                                add[0] = u.x, add[kPairs - 1] = u.y;
                            }
                        }
#pragma unroll
                        for (int e = 0; e < kPairs; ++e) {
                            const int i = 2 * (w * kPairs + e);
                            y[e] = finish2<kMode, kAdds>(f2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])),
                                                  *reinterpret_cast<const uint64_t*>(bias + i),
                                                  *reinterpret_cast<const uint64_t*>(gate + i), add[e],
                                                  kBf16 || first, kBf16 || last);
                        }
                        if constexpr (kBf16) {
                            uint32_t p[4];
#pragma unroll
                            for (int e = 0; e < kPairs; ++e) {
                                float lo, hi;
                                uf2(y[e], lo, hi);
                                p[e & 3] = pack_bf16x2(lo, hi);
                            }
                            *at = make_uint4(p[0], p[1], p[2], p[3]);
                        } else {
                            *reinterpret_cast<ulonglong2*>(at) = make_ulonglong2(y[0], y[kPairs - 1]);
                        }
                    }
                    if (wk.tma) {
                        fence_async_shared();
                        __syncwarp();
                        if (leader) {
                            tma_store_3d(&tmOut, c0 + 32 * c, row0, plane, smem_u32(room));
                            bulk_commit();
                            fetch_next();
                        }
                    } else {
                        __syncwarp();
                        T* to = static_cast<T*>(a.out) + corner;
                        if (col_here)
#pragma unroll 8
                            for (int r = 0; r < rows; ++r) to[(int64_t)r * a.N] = *element(r);
                    }
                };
                uint32_t va[32], vb[32];
                tmem_ld32(tbase + 32u * (uint32_t)chunk(0), va);
                tmem_ld_wait(va);
                if (half != acc) {  // this half held the shared columns: half 1 of accumulator 0, half 0 of accumulator 1
                    tc_fence_before();
                    __syncwarp();
                    if (leader) mbar_arrive_remote(ovl0);
                }
#pragma unroll
                for (int i = 0; i < kBN / 64; i += 2) {
                    tmem_ld32(tbase + 32u * (uint32_t)chunk(i + 1), vb);
                    emit(va, i);
                    tmem_ld_wait(vb);
                    if (i + 2 < kBN / 64) tmem_ld32(tbase + 32u * (uint32_t)chunk(i + 2), va);
                    if (i + 2 == kBN / 64) {  // the accumulator is in registers
                        tc_fence_before();
                        __syncwarp();
                        if (leader) mbar_arrive_remote(acc_empty0 + 8u * (uint32_t)acc);
                    }
                    emit(vb, i + 1);
                    if (i + 2 < kBN / 64) tmem_ld_wait(va);
                }
            }
            put_cols(buffer ^ 1);
        }
        if (wk.tma && leader) bulk_wait<0>();
    }
    tc_fence_before();
    cluster_sync();  // no signal to the other CTA and no MMA on this CTA's shared memory is still in flight
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

// out = epilogue(Σ partial products in order + bias), a thread four columns of a row.
template <typename T, int kMode>
__global__ void __launch_bounds__(256) gemm_fp8_join_kernel(const Fp8GemmArgs a, const float* __restrict__ partial,
                                                            int splits, int64_t ld) {
    griddep_wait_then_release();
    const int quads = (int)(ld >> 2);
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / quads;
    if (row >= a.M) return;
    const int col = (int)(i % quads) * 4, left = min(4, a.N - col);
    const int64_t plane = (int64_t)a.M * ld;
    const float* p = partial + row * ld + col;
    float4 s = *reinterpret_cast<const float4*>(p);
#pragma unroll 4
    for (int k = 1; k < splits; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(p + k * plane);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    T* out = static_cast<T*>(a.out) + row * a.N + col;
    const T* resid = static_cast<const T*>(a.resid) + row * a.N + col;
    float b[4] = {}, g[4] = {}, r[4] = {}, y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (e >= left) break;
        if (a.bias) b[e] = __bfloat162float(a.bias[col + e]);
        if (kMode == FVSR_LINEAR_GATED_RESIDUAL) g[e] = __bfloat162float(a.gate[col + e]), r[e] = load_as_float(resid + e);
    }
    uf2(finish2<kMode, kMode == FVSR_LINEAR_GATED_RESIDUAL>(f2(s.x, s.y), f2(b[0], b[1]), f2(g[0], g[1]), f2(r[0], r[1]), true, true), y[0], y[1]);
    uf2(finish2<kMode, kMode == FVSR_LINEAR_GATED_RESIDUAL>(f2(s.z, s.w), f2(b[2], b[3]), f2(g[2], g[3]), f2(r[2], r[3]), true, true), y[2], y[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) store_from_float(out + e, y[e]);
}

struct Maps {
    CUtensorMap x, w, xs, ws, out, resid;
};

template <typename T, int kMode>
cudaError_t launch_tiles(const Fp8GemmArgs& args, const Work& wk, const Maps& m, cudaStream_t st) {
    constexpr auto kernel = gemm_fp8_sm100_kernel<T, kMode>;
    cudaError_t e = allow_smem<kernel>(kSmemBytes);
    if (e != cudaSuccess) return e;
    const int items = wk.mt * wk.nt * wk.splits, pairs = sm_count() / 2;
    return launch_pdl(kernel, dim3(2 * (items < pairs ? items : pairs)), dim3(kThreads), kSmemBytes, st, m.x, m.w, m.xs,
                      m.ws, m.out, m.resid, args, wk);
}

template <typename T>
cudaError_t launch_mode(const Fp8GemmArgs& args, const Work& wk, const Maps& m, cudaStream_t st) {
    switch (args.mode) {
        case FVSR_LINEAR: return launch_tiles<T, FVSR_LINEAR>(args, wk, m, st);
        case FVSR_LINEAR_GELU: return launch_tiles<T, FVSR_LINEAR_GELU>(args, wk, m, st);
        default: return launch_tiles<T, FVSR_LINEAR_GATED_RESIDUAL>(args, wk, m, st);
    }
}

template <typename T>
cudaError_t launch_join(const Fp8GemmArgs& a, const Fp8GemmPlan& p, const float* partial, cudaStream_t st) {
    const dim3 grid((unsigned)(((int64_t)a.M * (p.partial_ld >> 2) + 255) / 256)), block(256);
    switch (a.mode) {
        case FVSR_LINEAR: return launch_pdl(gemm_fp8_join_kernel<T, FVSR_LINEAR>, grid, block, 0, st, a, partial, p.splits, p.partial_ld);
        case FVSR_LINEAR_GELU: return launch_pdl(gemm_fp8_join_kernel<T, FVSR_LINEAR_GELU>, grid, block, 0, st, a, partial, p.splits, p.partial_ld);
        default: return launch_pdl(gemm_fp8_join_kernel<T, FVSR_LINEAR_GATED_RESIDUAL>, grid, block, 0, st, a, partial, p.splits, p.partial_ld);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

Fp8GemmPlan plan_gemm_fp8(int M, int N, int K) {
    Fp8GemmPlan p{1, 0, 0, 0};
    const int kt = (K + kBK - 1) / kBK, groups = (kt + 3) / 4;
    const int64_t tiles = (int64_t)((M + kBM - 1) / kBM) * ((N + kBN - 1) / kBN);
    const int pairs = sm_count() / 2;
    // Parts of at least 1024 along K: with 512 the join costs more than it gives (777 × 1000 × 1100 12.3 against 10.8 us,
    // 17 × 9216 × 1536 11.5 / 10.0, but 17 × 1536 × 1536 9.2 / 9.8); with 1536 the parts get too few (17 × 1536 × 8960
    // 11.1 against 12.5 us, 300 × 300 × 4000 12.6 / 14.9).
    int splits = tiles * 2 <= pairs ? (int)(pairs / tiles) : 1;
    if (splits > groups / 2) splits = groups < 2 ? 1 : groups / 2;
    const int per = (groups + splits - 1) / splits;
    p.splits = (groups + per - 1) / per;
    p.part_blocks = 4 * per;
    if (p.splits > 1 || kt > kLongChainBlocks) {
        p.partial_ld = (N + 3) / 4 * 4;  // 16-byte rows
        p.partial_bytes = (size_t)p.splits * M * p.partial_ld * sizeof(float);
    }
    return p;
}

cudaError_t launch_gemm_fp8(const Fp8GemmArgs& args, const Fp8GemmPlan& plan, float* partial, cudaStream_t st) {
    const bool bf16 = args.out_dtype == FVSR_BF16;
    Work wk;
    wk.mt = (args.M + kBM - 1) / kBM;
    wk.nt = (args.N + kBN - 1) / kBN;
    wk.kt = (args.K + kBK - 1) / kBK;
    wk.splits = plan.splits;
    wk.part_blocks = plan.part_blocks;
    wk.chain_blocks = bf16 ? kLongChainBlocks : kChainBlocks;
    const bool parts = plan.splits > 1 || (bf16 && wk.kt > kLongChainBlocks);  // by way of the workspace
    const bool gated = args.mode == FVSR_LINEAR_GATED_RESIDUAL;
    wk.tma = parts || ((int64_t)args.N * (bf16 ? 2 : 4) % 16 == 0 && aligned16(args.out) && (!gated || aligned16(args.resid)));
    Maps m;
    const int64_t ld = fp8_ld(args.K), kt4 = fp8_scale_tiles(args.K);
    bool made = make_byte_map(&m.x, args.x, args.M, ld, 128) && make_byte_map(&m.w, args.w, args.N, ld, 128) &&
                make_scale_map(&m.xs, args.x_scale, ((int64_t)args.M + 127) / 128 * kt4) &&
                make_scale_map(&m.ws, args.w_scale, ((int64_t)args.N + 127) / 128 * kt4);
    m.out = m.resid = m.x;  // not used without tma
    if (parts)  // with the rows' padding: the join reads it (beyond w's last row the products are zeros)
        made = made && make_chunk_map(&m.out, partial, false, plan.splits, args.M, plan.partial_ld, plan.partial_ld);
    else if (wk.tma)
        made = made && make_chunk_map(&m.out, args.out, bf16, 1, args.M, args.N, args.N) &&
               (!gated || make_chunk_map(&m.resid, args.resid, bf16, 1, args.M, args.N, args.N));
    if (!made) return cudaErrorInvalidValue;
    if (!parts) return bf16 ? launch_mode<__nv_bfloat16>(args, wk, m, st) : launch_mode<float>(args, wk, m, st);
    Fp8GemmArgs sums = args;
    sums.bias = nullptr;
    sums.mode = FVSR_LINEAR;
    cudaError_t e = launch_tiles<float, FVSR_LINEAR>(sums, wk, m, st);
    if (e != cudaSuccess) return e;
    return bf16 ? launch_join<__nv_bfloat16>(args, plan, partial, st) : launch_join<float>(args, plan, partial, st);
}

cudaError_t read_and_clear_gemm_fp8_error(int* flag) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_gemm_fp8_timeout, sizeof(int));
    if (e != cudaSuccess) return e;
    if (v) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_gemm_fp8_timeout, &zero, sizeof(int));
    }
    *flag = v;
    return e;
}

}  // namespace fvsr
