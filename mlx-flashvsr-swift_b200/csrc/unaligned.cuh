// unaligned.cuh — a warp's contiguous stretch of a row whose first element is not on a 16-byte boundary, moved by aligned
// 16-byte accesses and shifts in registers. Each lane owns kRegs words of four bytes of the stretch, next to its
// neighbours'. Element by element, lanes 16 or 32 bytes apart, the same stretch takes eight (fp32: four) times the memory
// instructions, each touching every sector of it again: LayerNorm's passes over 17,280 × 1531 bf16 took 68 and 92 µs so
// (this way 46 and 63), reading an 8-bit tensor of that size back as bf16 82 (24).
#pragma once
#include "common.cuh"

namespace fvsr {

// Bytes [shift, shift + 4·kRegs) of w; shift < 16 and a multiple of the element's size. By halves: two selects and, for
// 2-byte elements, a funnel shift a word.
template <int kElemBytes, int kRegs>
__device__ __forceinline__ void shift_bytes(uint32_t (&w)[kRegs + 4], uint32_t shift, uint32_t (&out)[kRegs]) {
    const bool eight = shift & 8, four = shift & 4;
#pragma unroll
    for (int i = 0; i < kRegs + 2; ++i) w[i] = eight ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < kRegs + 1; ++i) w[i] = four ? w[i + 1] : w[i];
#pragma unroll
    for (int i = 0; i < kRegs; ++i)
        out[i] = kElemBytes == 4 ? w[i] : __funnelshift_r(w[i], w[i + 1], (shift & 2) * 8);
}

// The warp's elements [0, n) to p on, v being this lane's: the 16-byte words that lie wholly in them as such, each from
// its lane's elements and the last ones of the lane below, what is left at the two ends element by element. Every lane
// of the warp calls this with the same p and n.
template <typename T, int kRegs>
__device__ __forceinline__ void store_unaligned(T* p, int n, const uint32_t (&v)[kRegs]) {
    constexpr int kSize = sizeof(T), kWord = 16 / kSize, kElems = kRegs * 4 / kSize;
    const int lane = threadIdx.x & 31, off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / kSize);  // in elements
    uint32_t o[kRegs];
    if (off == 0) {
#pragma unroll
        for (int i = 0; i < kRegs; ++i) o[i] = v[i];
    } else {
        uint32_t w[kRegs + 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __shfl_up_sync(0xffffffffu, v[kRegs - 4 + i], 1);
#pragma unroll
        for (int i = 0; i < kRegs; ++i) w[4 + i] = v[i];
        shift_bytes<kSize, kRegs>(w, 16 - off * kSize, o);
    }
    const int first = lane * kElems - off;  // of o
    T* to = p + first;
#pragma unroll
    for (int i = 0; i < kRegs / 4; ++i)
        if (first + i * kWord >= 0 && first + (i + 1) * kWord <= n)
            reinterpret_cast<uint4*>(to)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    const int head = off == 0 ? 0 : kWord - off, tail = max(head, (n + off) / kWord * kWord - off);
    if ((lane == 0 && head > 0) || lane * kElems + kElems > tail) {
#pragma unroll
        for (int i = 0; i < kElems; ++i) {
            const int e = lane * kElems + i;
            const uint32_t u = v[i * kSize / 4];
            if (e < n && (e < head || e >= tail)) {
                if constexpr (kSize == 4)
                    reinterpret_cast<uint32_t*>(p)[e] = u;
                else
                    reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(i & 1 ? u >> 16 : u);
            }
        }
    }
}

}  // namespace fvsr
