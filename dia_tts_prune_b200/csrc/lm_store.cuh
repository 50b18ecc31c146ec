// lm_store.cuh - results that two warps hold, 32 rows of them, out to memory in whole lines.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace lm {
namespace {

// A panel is 32 rows of 256 bytes in shared memory, filled by two warps (a row per lane, 128 bytes each) and stored by them, 16 rows each: sectors of memory that a row
// does not fill alone cost a read, so a warp writes long rows (4096 x 16383 bf16 results of 256 channels, 128 bytes of a row at a time 123 us, 256 bytes 72; fp32 130 and 87).
constexpr int kPanelBytes = 32 * 256;

// a row's 16-byte piece c (0 .. 15) goes to place c ^ (row % 8) of its half, so that neither side meets itself in a bank
__device__ __forceinline__ int panel_at(int row, int piece) { return row * 256 + (piece & 8) * 16 + (((piece & 7) ^ (row & 7)) << 4); }

__device__ __forceinline__ void fill_panel(unsigned char* panel, int half, const uint32_t (&w)[32], int lane) {
#pragma unroll
    for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(panel + panel_at(lane, 8 * half + c)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
}

// the two warps of a panel (quarter: 0 .. 3) meet
__device__ __forceinline__ void panel_sync(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); }

// Rows 16 half .. of the panel to y (of row 0), `pitch` bytes apart, `cols` numbers of BYTES each.  wide: y, pitch and cols are multiples of 16 bytes.
template <int BYTES>
__device__ __forceinline__ void store_panel(const unsigned char* panel, char* y, size_t pitch, int half, int rows, int cols, bool wide, int lane) {
    const int sub = lane >> 4, ch = lane & 15, len = cols * BYTES;           // a row per sixteen lanes
    if (wide) {
        uint4 u[8];
#pragma unroll
        for (int g = 0; g < 8; ++g) u[g] = *reinterpret_cast<const uint4*>(panel + panel_at(16 * half + 2 * g + sub, ch));
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            const int r = 16 * half + 2 * g + sub;
            if (16 * ch < len && r < rows) *reinterpret_cast<uint4*>(y + r * pitch + 16 * ch) = u[g];
        }
        return;
    }
    if constexpr (BYTES == 4) {                               // a word per lane, two stores a row (in aligned pieces as below 1024 x 16383 results of 256 channels took 30 us, not 26)
#pragma unroll 1
        for (int r0 = 16 * half; r0 < min(16 * half + 16, rows); r0 += 4) {
            uint32_t u[4][2];
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int h = 0; h < 2; ++h) u[g][h] = *reinterpret_cast<const uint32_t*>(panel + panel_at(r0 + g, 8 * h + (lane >> 2)) + 4 * (lane & 3));
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (r0 + g < rows && 32 * h + lane < cols) *reinterpret_cast<uint32_t*>(y + (r0 + g) * pitch + 128 * h + 4 * lane) = u[g][h];
        }
    } else {
        // Rows of 16-bit numbers that begin anywhere, eight in flight: a lane takes 16 aligned bytes of memory, which lie across two pieces of the panel; what stands alone at
        // either end of the row goes number by number.
#pragma unroll 1
        for (int g0 = 0; g0 < 8; g0 += 4) {
            if (16 * half + 2 * g0 >= rows) break;
            uint4 w[4];
            uint16_t alone[4];
            int from[4], at[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int r = 16 * half + 2 * (g0 + g) + sub, s = (int)(reinterpret_cast<uintptr_t>(y + r * pitch) & 15), lead = s ? 16 - s : 0;
                const auto word = [&](int b) { return *reinterpret_cast<const uint32_t*>(panel + panel_at(r, b >> 4 & 15) + (b & 12)); };
                from[g] = 16 * ch + lead;                     // the lane's bytes of the row
                const int b = from[g] & 252;
                w[g] = make_uint4(word(b), word(b + 4), word(b + 8), word(b + 12));
                const uint32_t behind = word(b + 16);
                if (from[g] & 2)
                    w[g] = make_uint4(__funnelshift_r(w[g].x, w[g].y, 16), __funnelshift_r(w[g].y, w[g].z, 16), __funnelshift_r(w[g].z, w[g].w, 16), __funnelshift_r(w[g].w, behind, 16));
                const int front = min(lead, len), back = front + ((len - front) & ~15);      // bytes in front of the whole ones, and up to their end
                at[g] = 2 * ch < front ? 2 * ch : back + 2 * ch - front;
                alone[g] = *reinterpret_cast<const uint16_t*>(panel + panel_at(r, at[g] >> 4 & 15) + (at[g] & 15));
                if (r >= rows) from[g] = at[g] = len;
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                char* const row = y + (16 * half + 2 * (g0 + g) + sub) * pitch;
                if (from[g] + 16 <= len) *reinterpret_cast<uint4*>(row + from[g]) = w[g];
                if (at[g] < len) *reinterpret_cast<uint16_t*>(row + at[g]) = alone[g];
            }
        }
    }
    __syncwarp();
}

}  // namespace
}  // namespace lm
