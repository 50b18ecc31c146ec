// lm_store.cuh - 32 rows of results that a warp holds, a row per lane, out to memory in whole lines.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace lm {
namespace {

// The lanes' rows of 128 bytes into 4 KB of shared memory: a row's 16-byte piece c goes to place c ^ (row % 8), so that neither side meets itself in a bank.
__device__ __forceinline__ void turn_rows(unsigned char* blk, const uint32_t (&w)[32], int lane) {
#pragma unroll
    for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(blk + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
}

// and from there to y, rows `pitch` bytes apart, `cols` numbers of BYTES each.  wide: y, pitch and cols are multiples of 16 bytes
template <int BYTES>
__device__ __forceinline__ void store_turned(const unsigned char* blk, char* y, size_t pitch, int rows, int cols, bool wide, int lane) {
    if (wide) {                                               // a row per eight lanes
        const int rr = lane >> 3, ch = lane & 7;
        uint4 u[8];
#pragma unroll
        for (int g = 0; g < 8; ++g) u[g] = *reinterpret_cast<const uint4*>(blk + (4 * g + rr) * 128 + ((ch ^ ((4 * g + rr) & 7)) << 4));
        const bool in = ch * (16 / BYTES) < cols;
#pragma unroll
        for (int g = 0; g < 8; ++g)
            if (in && 4 * g + rr < rows) *reinterpret_cast<uint4*>(y + (4 * g + rr) * pitch + 16 * ch) = u[g];
        return;
    }
    // A row per warp, eight rows in flight, a 4-byte word per lane.  Where a row of 16-bit numbers begins half way into a word of memory, a lane's word is made of the
    // second number of the lane in front and its own first one.
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += 8) {
        uint32_t u[8];
#pragma unroll
        for (int g = 0; g < 8; ++g) u[g] = *reinterpret_cast<const uint32_t*>(blk + (r0 + g) * 128 + (((lane >> 2) ^ g) << 4) + 4 * (lane & 3));
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            char* const row = y + (r0 + g) * pitch;
            if constexpr (BYTES == 4) {
                if (r0 + g < rows && lane < cols) *reinterpret_cast<uint32_t*>(row + 4 * lane) = u[g];
            } else {
                const uint32_t front = __shfl_up_sync(0xffffffffu, u[g], 1);
                if (r0 + g >= rows) continue;
                const int off = (int)(reinterpret_cast<uintptr_t>(row) >> 1 & 1), c = 2 * lane - off;
                const uint32_t word = off ? __funnelshift_r(front, u[g], 16) : u[g];
                if (c >= 0 && c + 1 < cols) *reinterpret_cast<uint32_t*>(row + 2 * c) = word;
                // what stands alone at either end: the first number, the last one (of 64: a second store of the last lane)
                const bool front_end = c < 0, back_end = c == cols - 1, last = off && lane == 31 && cols == 64;
                if (front_end || back_end || last)
                    *reinterpret_cast<uint16_t*>(row + 2 * (front_end ? 0 : back_end ? c : 63)) = (uint16_t)(front_end ? u[g] : back_end ? word : u[g] >> 16);
            }
        }
    }
}

}  // namespace
}  // namespace lm
