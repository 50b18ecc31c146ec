// lm_mxfp4.cu - microscaled 4-bit numbers: rounding rows to them, their values, and products on the tensor cores' own 4-bit path.
//
// Rounding (OCP Microscaling Formats, version 1.0): a block of 32 channels has the scale 2^e, e = floor(log2(largest magnitude)) - 2 (2 is the exponent of the largest
// E2M1 number, 6), at least 2^-127; its elements are x 2^-e to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (half way: to the even code), 6 beyond.  Both steps are exact
// but for that last one, so every implementation of the rule has the same bits.
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_split.h"
#include "engine_internal.h"
#include "gemm_tcgen05.h"
#include "lm_mxfp4.h"
#include "lm_store.cuh"
#include "tensor_cores.cuh"

namespace lm {
namespace {

using namespace dia;

// ---- rounding and values -------------------------------------------------------------------------------------------------------------------

// Eight neighbouring channels of a row as they lie in memory.  WIDE: rows of whole 16 bytes whose channels are a multiple of eight, all eight are there or none; else those
// at or beyond `n` are zero.  ONCE: an SM reads them once, so that L1 does without them (32768 x 2048 fp32 rounded in 42 us, not 48), and no kernel writes them meanwhile (the
// read-only path; a kernel that starts before its predecessor has ended does without it).  (Fetching and widening are apart: widened at once, a load is waited for before the
// next one goes out.)
template <int TYPE, bool WIDE, bool ONCE>
struct Eight {
    static __device__ __forceinline__ uint4 load(const uint4* p) {
        if constexpr (!ONCE) return *p;
        uint4 v;
        asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
        return v;
    }
    uint4 w[TYPE == kTypeF32 ? 2 : 1];
    __device__ __forceinline__ void fetch(const void* row, int k, int n) {
        constexpr int kWords = TYPE == kTypeF32 ? 2 : 1;
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                w[i] = n > 0 ? load(reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(row) + (size_t)k * (TYPE == kTypeF32 ? 4 : 2)) + i) : make_uint4(0u, 0u, 0u, 0u);
        } else {
            uint32_t u[4 * kWords];
#pragma unroll
            for (int e = 0; e < 4 * kWords; ++e) {
                if (TYPE == kTypeF32) {
                    u[e] = e < n ? reinterpret_cast<const uint32_t*>(row)[k + e] : 0u;
                } else {
                    const uint32_t lo = 2 * e < n ? reinterpret_cast<const uint16_t*>(row)[k + 2 * e] : 0u, hi = 2 * e + 1 < n ? reinterpret_cast<const uint16_t*>(row)[k + 2 * e + 1] : 0u;
                    u[e] = lo | hi << 16;
                }
            }
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
        }
    }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
        const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
        if constexpr (TYPE == kTypeF32) {
            const uint4 h = w[TYPE == kTypeF32];
            v[0] = __uint_as_float(u[0]); v[1] = __uint_as_float(u[1]); v[2] = __uint_as_float(u[2]); v[3] = __uint_as_float(u[3]);
            v[4] = __uint_as_float(h.x); v[5] = __uint_as_float(h.y); v[6] = __uint_as_float(h.z); v[7] = __uint_as_float(h.w);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (TYPE == kTypeBf16) {
                    v[2 * e] = __uint_as_float(u[e] << 16);
                    v[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
                    v[2 * e] = f.x;
                    v[2 * e + 1] = f.y;
                }
            }
        }
    }
};
inline int wide_rows(const void* x, int type, long long ld, int K) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld * type_bytes(type) % 16 == 0 && K % 8 == 0; }

// The codes of eight channels and their block's scale, where the four lanes of a group of four hold the block's 32 channels.
__device__ __forceinline__ uint32_t round_block(const float (&v)[8], uint32_t& scale) {
    uint32_t most = 0;                                        // magnitudes as bits: an infinity or a NaN is the largest
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const uint32_t exponent = most >> 23;
    scale = most >= 0x7f800000u ? 255u : exponent > 2u ? exponent - 2u : 0u;
    if (scale == 255u) return 0u;
    const float f = __uint_as_float((254u - scale) << 23);    // 2^(127 - scale)
    uint32_t codes;
    asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c3, %8, %7;\n\t"
        "mov.b32 %0, {c0, c1, c2, c3};\n\t}"
        : "=r"(codes)
        : "f"(v[0] * f), "f"(v[1] * f), "f"(v[2] * f), "f"(v[3] * f), "f"(v[4] * f), "f"(v[5] * f), "f"(v[6] * f), "f"(v[7] * f));
    return codes;
}

// A CTA takes 128 rows x 256 channels, a warp 16 rows of them, a lane eight channels (four neighbours a block): kAhead rows are on their way at a time, eight loads, and the
// scales leave as the two pieces that they are.  early: the successor, a product of these rows, may start now (a product asks for its weights before this kernel has ended:
// they are never what it writes).  Rows behind the last one of a piece get scales of zero.  Bound: memory, instructions next (32768 x 2048 bf16, 170 MB: 31 us; 75 with an index
// per eight channels, whose scales went out byte by byte; fp32, 304 MB: 42, and 48 with eight rows on their way, whose registers leave fewer warps).
constexpr int kQuantThreads = 256;
template <int TYPE, bool WIDE>
__global__ void __launch_bounds__(kQuantThreads) mxfp4_quantize_kernel(const void* __restrict__ x, long long ld, int rows, int K, uint32_t* __restrict__ codes,
                                                                       uint8_t* __restrict__ scales, int early) {
    if (early) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ __align__(16) uint8_t staged[2 * kMxScaleBytes];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pieces = (K + 127) / 128, c0 = blockIdx.x * 32 + lane, k = 8 * c0;
    const long long row0 = (long long)blockIdx.y * 128 + warp * 16;
    const bool kept = c0 < pieces * 16;                       // (a row's codes go on to the end of its last piece)
    constexpr int kAhead = TYPE == kTypeF32 ? 4 : 8;
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += kAhead) {
        Eight<TYPE, WIDE, true> x8[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const long long r = row0 + r0 + j;
            x8[j].fetch(reinterpret_cast<const char*>(x) + r * ld * (TYPE == kTypeF32 ? 4 : 2), k, r < rows ? K - k : 0);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int in = warp * 16 + r0 + j;
            const long long r = row0 + r0 + j;
            float v[8];
            x8[j].widen(v);
            uint32_t scale;
            const uint32_t code = round_block(v, scale);
            if (kept && r < rows) codes[r * (pieces * 16) + c0] = code;
            if ((lane & 3) == 0) staged[(lane >> 4) * kMxScaleBytes + (in & 31) * 16 + (in >> 5) * 4 + ((lane >> 2) & 3)] = (uint8_t)scale;
        }
    }
    __syncthreads();
    const int piece = 2 * blockIdx.x + (threadIdx.x >> 5);
    if (threadIdx.x < 64 && piece < pieces)
        reinterpret_cast<uint4*>(scales + ((size_t)blockIdx.y * pieces + piece) * kMxScaleBytes)[lane] = reinterpret_cast<const uint4*>(staged)[threadIdx.x];
}

// four neighbouring numbers of a row, those at or beyond `n` left out.  wide: one store of them all
template <int TYPE>
__device__ __forceinline__ void put4(void* y, size_t at, float4 v, int n, bool wide) {
    const float f[4] = {v.x, v.y, v.z, v.w};
    if constexpr (TYPE == kTypeF32) {
        float* const o = reinterpret_cast<float*>(y) + at;
        if (wide) {
            *reinterpret_cast<float4*>(o) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) if (e < n) o[e] = f[e];
        }
    } else {
        uint16_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = TYPE == kTypeBf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(f[e])) : __half_as_ushort(__float2half_rn(f[e]));
        uint16_t* const o = reinterpret_cast<uint16_t*>(y) + at;
        if (wide) {
            *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(h);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) if (e < n) o[e] = h[e];
        }
    }
}

__device__ __forceinline__ float2 two_values(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 c;\n\t.reg .b16 w;\n\tcvt.u16.u32 w, %1;\n\tcvt.u8.u16 c, w;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}" : "=r"(h) : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float scale_value(uint32_t scale) { return __uint_as_float(scale == 255u ? 0x7fffffffu : scale ? scale << 23 : 0x00400000u); }

// The same shares; a lane takes four neighbouring channels of either half, so that whole lines of float32 are stored.
template <int TYPE>
__global__ void __launch_bounds__(kQuantThreads) mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int K,
                                                                         void* __restrict__ out, int wide) {
    __shared__ __align__(16) uint8_t staged[2 * kMxScaleBytes];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pieces = (K + 127) / 128;
    const long long row0 = (long long)blockIdx.y * 128 + warp * 16;
    if (threadIdx.x < 64 && 2 * (int)blockIdx.x + warp < pieces)
        reinterpret_cast<uint4*>(staged)[threadIdx.x] = reinterpret_cast<const uint4*>(scales + ((size_t)blockIdx.y * pieces + 2 * blockIdx.x + warp) * kMxScaleBytes)[lane];
    __syncthreads();
    const int n = (int)min(16LL, rows - row0);
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += 4) {
        uint32_t code[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int piece = 2 * blockIdx.x + h;
                code[j][h] = r0 + j < n && piece < pieces ? reinterpret_cast<const uint16_t*>(codes + (row0 + r0 + j) * (pieces * 64) + piece * 64)[lane] : 0u;
            }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int in = warp * 16 + r0 + j, k = (2 * blockIdx.x + h) * 128 + 4 * lane;
                if (r0 + j >= n || k >= K) continue;
                const float f = scale_value(staged[h * kMxScaleBytes + (in & 31) * 16 + (in >> 5) * 4 + (lane >> 3)]);
                const float2 a = two_values(code[j][h] & 255u), b = two_values(code[j][h] >> 8);
                put4<TYPE>(out, (size_t)(row0 + r0 + j) * K + k, make_float4(a.x * f, a.y * f, b.x * f, b.y * f), K - k, wide);
            }
    }
}

// ---- the product -----------------------------------------------------------------------------------------------------------------------------

constexpr int kBM = 128, kBN = 128, kStageK = 256;            // rows of A and of W in a tile, channels of a stage
constexpr int kCodeTile = 128 * 128;                          // 128 rows x 256 channels, 16 KB
constexpr int kStageBytes = 2 * kCodeTile + 2 * 1024;         // A, W, their scales
constexpr int kStages = 5;
constexpr int kFewThreads = 320, kWarps4 = 8, kThreads4 = 64 + 32 * kWarps4;
constexpr int kTurnBytes = kWarps4 * 4096;
constexpr int kSmem4 = kStages * kStageBytes + kTurnBytes + 1024 + 256;

// scales of 128 rows x 128 channels in shared memory: 8 rows of 16 bytes after one another, no swizzle
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
    const uint32_t lo = (smem_addr & 0x3FFFFu) >> 4, hi = (128u >> 4) | (1u << 14);
    return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_mxfp4(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t a_scales, uint32_t b_scales, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
}
// instruction descriptor: E2M1 operands, both K-major, scales in UE8M0, M = 128; which two of a piece's four scales an MMA of 64 channels takes
__device__ __forceinline__ uint32_t mx_idesc(int n, int half) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | (1u << 27) | ((uint32_t)(2 * half) << 29) | ((uint32_t)(2 * half) << 4);
}

struct TiledProduct {
    const uint8_t *a_scales, *w_scales;
    void* y;
    int M, N, K;
    int* ran_out;
    unsigned polls;
};

// columns of a panel of results (see lm_store.cuh)
template <int TYPE>
struct Out {
    static constexpr int kBytes = TYPE == kTypeF32 ? 4 : 2, kPanel = 256 / kBytes;
};
__device__ __forceinline__ uint32_t pack16(int type, float lo, float hi) {
    if (type == kTypeBf16) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&b);
    }
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// The warp's half of a panel of an accumulator (from: its first column of the warp's 32 rows)
template <int TYPE>
__device__ __forceinline__ void panel_half(uint32_t from, int half, uint32_t (&w)[32]) {
    if constexpr (TYPE == kTypeF32) {
        tmem_columns32(from + 32 * half, w);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    } else {
        uint32_t v[2][32];
        tmem_columns32(from + 64 * half, v[0]);
        tmem_columns32(from + 64 * half + 32, v[1]);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int e = 0; e < 32; ++e) w[e] = pack16(TYPE, __uint_as_float(v[e >> 4][2 * e & 31]), __uint_as_float(v[e >> 4][(2 * e & 31) + 1]));
    }
}
// The warp's half (w) of a panel to rows row0 .. and columns n0 .. of the result, by the two warps of a quarter.
template <int TYPE>
__device__ __forceinline__ void put_out(uint32_t (&w)[32], unsigned char* panel, const TiledProduct& p, int row0, int rows, int n0, int quarter, int half, int lane, bool ok, bool wide) {
    if (!ok) {
#pragma unroll
        for (int e = 0; e < 32; ++e) w[e] = TYPE == kTypeF16 ? 0x7e007e00u : 0x7fff7fffu;                         // (no result: NaN as one number or two)
    }
    fill_panel(panel, half, w, lane);
    panel_sync(quarter);
    const size_t pitch = (size_t)p.N * Out<TYPE>::kBytes;
    store_panel<Out<TYPE>::kBytes>(panel, reinterpret_cast<char*>(p.y) + (row0 * pitch + (size_t)n0 * Out<TYPE>::kBytes), pitch, half, rows, min(Out<TYPE>::kPanel, p.N - n0), wide, lane);
    panel_sync(quarter);
}
template <int TYPE>
__device__ __forceinline__ bool whole_pieces(const TiledProduct& p) { return p.N * Out<TYPE>::kBytes % 16 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0; }

// One CTA per SM walks 128 x 128 tiles.
//   warp 0    one lane: a stage's codes (TMA, 128-byte swizzle) and scales (plain bulk copies)
//   warp 1    one elected lane: the stage's scales into tensor memory, then its MMAs of 64 channels
//   warps 2-9 take a finished accumulator out through shared memory while the next tile fills the other (four of them took up to twice as long, rows that begin anywhere)
template <int TYPE>
__global__ void __launch_bounds__(kThreads4, 1)
mxfp4_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ TiledProduct p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* turn = smem + kStages * kStageBytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(turn + kTurnBytes);
    uint64_t* empty = full + kStages;
    uint64_t* t_full = empty + kStages;
    uint64_t* t_empty = t_full + 2;
    uint64_t* done = t_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pieces = (p.K + 127) / 128, n_stage = (pieces + 1) / 2;
    const int tiles_m = (p.M + kBM - 1) / kBM, n_tiles = tiles_m * ((p.N + kBN - 1) / kBN);

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&t_full[i], 1); mbar_init(&t_empty[i], kWarps4); }
        mbar_init(done, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            // a stage's weights, which do not wait for the kernel that rounds the rows, and its rows (t, s: its tile and place there)
            const auto weights = [&](unsigned at, int t, int s) {
                unsigned char* const dst = smem + at * kStageBytes;
                const uint32_t sc = kMxScaleBytes * min(2, pieces - 2 * s);
                const int tn = t / tiles_m;
                mbar_arrive_expect_tx(&full[at], 2 * kCodeTile + 2 * sc);
                tma_load_2d(smem_u32(dst + kCodeTile), &map_w, smem_u32(&full[at]), s * (kStageK / 2), tn * kBN);
                bulk_g2s(dst + 2 * kCodeTile + 1024, p.w_scales + ((size_t)tn * pieces + 2 * s) * kMxScaleBytes, sc, &full[at]);
            };
            const auto rows = [&](unsigned at, int t, int s) {
                unsigned char* const dst = smem + at * kStageBytes;
                const int tm = t % tiles_m;
                tma_load_2d(smem_u32(dst), &map_a, smem_u32(&full[at]), s * (kStageK / 2), tm * kBM);
                bulk_g2s(dst + 2 * kCodeTile, p.a_scales + ((size_t)tm * pieces + 2 * s) * kMxScaleBytes, kMxScaleBytes * min(2, pieces - 2 * s), &full[at]);
            };
            unsigned i = 0;
            int t = blockIdx.x, s = 0;
            const auto next = [&]() {
                ++i;
                if (++s == n_stage) s = 0, t += gridDim.x;
            };
            while (i < kStages && t < n_tiles) { weights(i, t, s); next(); }
            const unsigned ahead = i;
            asm volatile("griddepcontrol.wait;" ::: "memory");
            i = 0; t = blockIdx.x; s = 0;
            while (i < ahead) { rows(i, t, s); next(); }
            for (; t < n_tiles; next()) {
                const unsigned at = i % kStages;
                if (!lane_wait(&empty[at], ((i / kStages) & 1u) ^ 1u, p.polls)) { ok = false; break; }
                weights(at, t, s);
                rows(at, t, s);
            }
            copies_landed(full, kStages, i);
        }
    } else if (warp == 1) {
        const uint32_t idesc[2] = {mx_idesc(kBN, 0), mx_idesc(kBN, 1)};
        unsigned i = 0, it = 0;
        for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x, ++it) {
            if (!pair_wait(&t_empty[it & 1u], ((it >> 1) & 1u) ^ 1u, p.polls)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t d = tmem + (it & 1u) * kBN;
            for (int s = 0; s < n_stage; ++s, ++i) {
                const unsigned at = i % kStages;
                if (!pair_wait(&full[at], (i / kStages) & 1u, p.polls)) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t base = smem_u32(smem + at * kStageBytes);
                const uint64_t adesc = umma_desc(base), bdesc = umma_desc(base + kCodeTile);
                const uint32_t sa = tmem + 2 * kBN + (i & 3u) * 16, sb = sa + 8;
                const int here = min(2, pieces - 2 * s);
                if (elect_one_sync()) {
                    for (int c = 0; c < here; ++c) {
                        scales_to_tmem(sa + 4 * c, scale_desc(base + 2 * kCodeTile + c * kMxScaleBytes));
                        scales_to_tmem(sb + 4 * c, scale_desc(base + 2 * kCodeTile + 1024 + c * kMxScaleBytes));
                    }
                    for (int c = 0; c < here; ++c)
#pragma unroll
                        for (int j = 0; j < 2; ++j)           // 64 channels: 32 bytes, 2 descriptor units
                            umma_mxfp4(d, adesc + 4 * c + 2 * j, bdesc + 4 * c + 2 * j, idesc[j], sa + 4 * c, sb + 4 * c, (s | c | j) != 0 ? 1u : 0u);
                    umma_commit(&empty[at]);
                    if (s == n_stage - 1) umma_commit(&t_full[it & 1u]);
                }
                __syncwarp();
            }
        }
        mmas_ended<false>(done);
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2;       // (a warp reads the 32 lanes of its number mod 4)
        unsigned char* const panel = turn + q * kPanelBytes;
        const bool wide = whole_pieces<TYPE>(p);
        unsigned it = 0;
        for (int t = blockIdx.x; t < n_tiles; t += gridDim.x, ++it) {
            const int n0 = t / tiles_m * kBN, row0 = t % tiles_m * kBM + q * 32, rows = min(32, p.M - row0);
            ok = ok && pair_wait(&t_full[it & 1u], (it >> 1) & 1u, p.polls);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int c = 0; c < kBN && n0 + c < p.N && rows > 0; c += Out<TYPE>::kPanel) {
                uint32_t w[32];
                panel_half<TYPE>(tmem + ((uint32_t)(q * 32) << 16) + (it & 1u) * kBN + c, half, w);
                put_out<TYPE>(w, panel, p, row0, rows, n0 + c, q, half, lane, ok, wide);
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&t_empty[it & 1u]);
        }
    }
    if (!ok && lane == 0 && p.ran_out) {
        *reinterpret_cast<volatile int*>(p.ran_out) = 1;
        __threadfence_system();
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// The same on pairs of SMs: a cluster of two CTAs owns a 256 x 256 tile, an MMA of the pair multiplies the 256 rows of both by the 256 columns of both, so an SM takes 32 KB
// of codes from L2 for 512 cycles of MMAs where the kernel above takes as much for 256.  Each SM needs the scales of its own 128 rows and of all 256 columns.  Two accumulators
// and the scales of two stages are 576 columns of tensor memory, which has 512: the second accumulator begins on the last 64 columns of the first, and whichever is taken out
// hands these over first.  (192 columns a tile, accumulators apart: 4096 x 16384 x 4096 133 us here 104, 2048 channels 75 / 60.)
//   warp 0    one lane per CTA: codes and scales (TMA) of its halves; every byte of both CTAs counts on the leader's barrier
//   warp 1    leader only: a stage's scales into the tensor memory of both, then the pair's MMAs; commits to the barriers of both
//   warps 2-9 take the CTA's 128 rows of a finished accumulator out
// Bound: what the SMs take from L2, 12 TB/s (4096 x 16384 x 4096, us with 8 of waiting for the rows: 104; without MMAs 96, without loading scales 97, without taking results
// out 98).
constexpr int kPairN = 256, kPairShift = 192, kPairStages = 5, kPairWarps = 8, kPairThreads = 64 + 32 * kPairWarps;
constexpr int kPairCodes = kCodeTile + kPairN / 2 * 128, kPairStage = kPairCodes + 3 * 1024;
constexpr int kPairSmem = kPairStages * kPairStage + kPairWarps * 4096 + 1024 + 256;
static_assert(kPairStage % 1024 == 0 && kPairSmem <= 227 * 1024, "shared memory");

__device__ __forceinline__ void scales_to_tmem_pair(uint32_t tmem, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_mxfp4_pair(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t a_scales, uint32_t b_scales, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
}

template <int TYPE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
mxfp4_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_as,
                  const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ TiledProduct p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* turn = smem + kPairStages * kPairStage;
    uint64_t* full = reinterpret_cast<uint64_t*>(turn + kPairWarps * 4096);  // (the leader's alone)
    uint64_t* empty = full + kPairStages;
    uint64_t* t_full = empty + kPairStages;
    uint64_t* t_early = t_full + 2;                                          // (these two the leader's alone)
    uint64_t* t_empty = t_early + 2;
    PairEnd* end = reinterpret_cast<PairEnd*>(t_empty + 2);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(end + 1);
    static_assert((2 * kPairStages + 6) * 8 + sizeof(PairEnd) + 4 <= 256, "barrier region");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int pieces = (p.K + 127) / 128, n_stage = (pieces + 1) / 2;
    const int tiles_m = (p.M + 255) / 256, n_tiles = tiles_m * ((p.N + kPairN - 1) / kPairN);

    if (threadIdx.x == 0) {
        for (int i = 0; i < kPairStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&t_full[i], 1); mbar_init(&t_early[i], 2 * kPairWarps); mbar_init(&t_empty[i], 2 * kPairWarps); }
        pair_begin(end);
        fence_mbar_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            // a stage's weights, which do not wait for the kernel that rounds the rows, and its rows (t, s: its tile and place there)
            const auto weights = [&](unsigned at, int t, int s) {
                const int n0 = t / tiles_m * kPairN;
                const uint32_t bar = at_rank(&full[at], 0), dst = smem_u32(smem + at * kPairStage);
                if (rank == 0) mbar_arrive_expect_tx(&full[at], 2u * kPairStage);
                tma_load_2d_pair(dst + kCodeTile, &map_w, bar, s * (kStageK / 2), n0 + (int)rank * (kPairN / 2));
                tma_load_2d_pair(dst + kPairCodes + 1024, &map_ws, bar, s * (2 * kMxScaleBytes / 4), n0 / 128);
            };
            const auto rows = [&](unsigned at, int t, int s) {
                const int m = t % tiles_m * 2 + (int)rank;
                const uint32_t bar = at_rank(&full[at], 0), dst = smem_u32(smem + at * kPairStage);
                tma_load_2d_pair(dst, &map_a, bar, s * (kStageK / 2), m * 128);
                tma_load_2d_pair(dst + kPairCodes, &map_as, bar, s * (2 * kMxScaleBytes / 4), m);
            };
            unsigned i = 0;
            int t = pair, s = 0;
            const auto next = [&]() {
                ++i;
                if (++s == n_stage) s = 0, t += pairs;
            };
            while (i < kPairStages && t < n_tiles) { weights(i, t, s); next(); }
            const unsigned ahead = i;
            asm volatile("griddepcontrol.wait;" ::: "memory");
            i = 0; t = pair; s = 0;
            while (i < ahead) { rows(i, t, s); next(); }
            for (; t < n_tiles; next()) {
                const unsigned at = i % kPairStages;
                if (!lane_wait(&empty[at], ((i / kPairStages) & 1u) ^ 1u, p.polls)) { ok = false; break; }
                weights(at, t, s);
                rows(at, t, s);
            }
            // (the leader's last commits arrive here: not after this CTA has gone)
            for (unsigned j = i > (unsigned)kPairStages ? i - kPairStages : 0; j < i && ok; ++j) ok = lane_wait(&empty[j % kPairStages], (j / kPairStages) & 1u, p.polls);
            pair_issued(end, rank, i);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t two = mx_idesc(kPairN, 0) ^ (3u << 27), idesc[2] = {two, two | (mx_idesc(0, 1) ^ mx_idesc(0, 0))};      // M = 256
            unsigned i = 0, it = 0;
            for (int t = pair; t < n_tiles && ok; t += pairs, ++it) {
                if (!pair_wait(&t_empty[it & 1u], ((it >> 1) & 1u) ^ 1u, p.polls) || (it && !pair_wait(&t_early[(it & 1u) ^ 1u], ((it - 1) >> 1) & 1u, p.polls))) { ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = tmem + (it & 1u) * kPairShift;
                for (int s = 0; s < n_stage; ++s, ++i) {
                    const unsigned at = i % kPairStages;
                    if (!pair_wait(&full[at], (i / kPairStages) & 1u, p.polls)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t base = smem_u32(smem + at * kPairStage);
                    const uint64_t adesc = umma_desc(base), bdesc = umma_desc(base + kCodeTile);
                    const uint32_t sa = tmem + kPairShift + kPairN + (i & 1u) * 32, sb = sa + 8;
                    const int here = min(2, pieces - 2 * s);
                    if (elect_one_sync()) {
                        for (int c = 0; c < here; ++c) {
                            scales_to_tmem_pair(sa + 4 * c, scale_desc(base + kPairCodes + c * kMxScaleBytes));
                            scales_to_tmem_pair(sb + 8 * c, scale_desc(base + kPairCodes + 1024 + c * kMxScaleBytes));
                            scales_to_tmem_pair(sb + 8 * c + 4, scale_desc(base + kPairCodes + 2048 + c * kMxScaleBytes));
                        }
                        for (int c = 0; c < here; ++c)
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                umma_mxfp4_pair(d, adesc + 4 * c + 2 * j, bdesc + 4 * c + 2 * j, idesc[j], sa + 4 * c, sb + 8 * c, (s | c | j) != 0 ? 1u : 0u);
                        umma_commit_pair(&empty[at]);
                        if (s == n_stage - 1) umma_commit_pair(&t_full[it & 1u]);
                    }
                    __syncwarp();
                }
            }
            mmas_ended<true>(&end->done);
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2;
        unsigned char* const panel = turn + q * kPanelBytes;
        const bool wide = whole_pieces<TYPE>(p);
        constexpr int kPanels = kPairN / Out<TYPE>::kPanel;
        unsigned it = 0;
        for (int t = pair; t < n_tiles; t += pairs, ++it) {
            const int n0 = t / tiles_m * kPairN, row0 = t % tiles_m * 256 + (int)rank * 128 + q * 32, rows = min(32, p.M - row0);
            ok = ok && pair_wait(&t_full[it & 1u], (it >> 1) & 1u, p.polls);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            // (relaxed: a release would wait for this warp's stores of earlier tiles to be seen, with which the MMAs have nothing to do; 1024 channels took 66 us, not 46)
            const auto taken = [&](uint64_t* bar) {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(at_rank(bar, 0)) : "memory");
            };
            // the panel that the next tile's accumulator lies on goes first
#pragma unroll 1
            for (int i = 0; i < kPanels; ++i) {
                const int c = (it & 1u ? i : kPanels - 1 - i) * Out<TYPE>::kPanel;
                const bool there = n0 + c < p.N && rows > 0;
                uint32_t w[32];
                if (there) panel_half<TYPE>(tmem + ((uint32_t)(q * 32) << 16) + (it & 1u) * kPairShift + c, half, w);
                if (i == 0) taken(&t_early[it & 1u]);
                if (i == kPanels - 1) taken(&t_empty[it & 1u]);
                if (there) put_out<TYPE>(w, panel, p, row0, rows, n0 + c, q, half, lane, ok, wide);
            }
        }
    }
    if (!ok && lane == 0) {
        pair_gave_up(end);
        if (p.ran_out) {
            *reinterpret_cast<volatile int*>(p.ran_out) = 1;
            __threadfence_system();
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    pair_end(end, rank, full, kPairStages, kPairStage);       // neither CTA's memory goes while the other still reads it or arrives there
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Few rows (decoding): the weights are the 128-row operand and stream once, the rows are the columns.  A cluster of S CTAs owns 128 weight rows, each
// CTA a range of stages.
//   warp 0    requests the CTA's weight codes and scales ahead of the rows, but not before the kernel's predecessor has ended, which may have written them (that takes
//             0.2 us of 32768 x 2048 with one row, 0.7 of 4096 x 4096 read from memory by one product after the other, nothing where another kernel lies between)
//   all warps round the CTA's share of the rows to MXFP4, straight into the layout of the MMA
//   warp 1    per stage the scales into tensor memory and its MMAs (M = 128, N = NB)
//   warps 2-5 take the accumulator out (weight row = lane); with S > 1 the shares meet in shared memory, in the order of the ranges
// Bound: the weights' bytes where there are many, latency else.  Every CTA rounds the rows by itself, which takes
// longer than a kernel in front that rounds them once and 128 x 128 tiles from some rows times stages of a CTA on (us, here / there, weights in L2: 2048 x 2048 1 row 4.8 / 8.6,
// 16 rows 5.8 / 9.0; 32768 x 2048 8.5 / 14.7, 8 rows 11.4 / 14.6, 16 rows - 128 stages rounded - 14.1 / 14.7; weights in memory: 32768 x 2048 8 rows 18 / 22, 16 rows
// 23 / 22; 32768 x 4096 1 row 31 / 30, 8 rows 37 / 30, 16 rows 46 / 34).  Tensor memory is taken behind the wait for the predecessor and in front of the signal to the successor:
// a CTA that waits for another kernel holds none of it, so neither can wait for the other.  Shared memory is asked for such that an SM holds three CTAs at most, whose
// tensor memory fits at the same time: CTAs of a cluster wait for one another.
constexpr int kFewMost = 16, kFewRounded = 100, NB = 16, kFewCols = 128, kFewSmemMost = 226 * 1024, kFewSmemLeast = 58 * 1024, kFewSlotsMost = 12;
static_assert(4 * kFewSmemLeast > 228 * 1024 && 4 * kFewCols <= 512, "CTAs on an SM");

struct FewProduct {
    const void* a; long long lda; int a_type, wide;
    const uint8_t* w_scales;
    void* y; int y_type;
    int M, N, K, per, slots;                                  // stages of a CTA, of the ring
    int* ran_out;
    unsigned polls;
};

__device__ __forceinline__ void put1(void* y, int type, size_t at, float v) {
    if (type == kTypeF32) reinterpret_cast<float*>(y)[at] = v;
    else if (type == kTypeBf16) reinterpret_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(y)[at] = __float2half_rn(v);
}

__global__ void __launch_bounds__(kFewThreads, 2) mxfp4_few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ FewProduct p) {
    constexpr int kSlot = kCodeTile + 1024, kRows = NB * 128 + 1024;       // a stage of weights, of rows
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[kFewSlotsMost], empty[kFewSlotsMost], t_full, done;
    __shared__ uint32_t tmem_slot;
    unsigned char* const ring = smem;
    unsigned char* const rows = ring + p.slots * kSlot;                     // [per][NB x 128 bytes | 2 x 512 bytes of scales]
    float* const part = reinterpret_cast<float*>(rows + p.per * kRows);     // [NB][128]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, S = gridDim.y, rank = blockIdx.y, n0 = blockIdx.x * 128, M = p.M;
    const int pieces = (p.K + 127) / 128, n_stage = (pieces + 1) / 2, s0 = rank * p.per, stages = max(0, min(p.per, n_stage - s0));
    const auto request = [&](int s, int slot) {
        unsigned char* const dst = ring + slot * kSlot;
        const uint32_t sc = kMxScaleBytes * min(2, pieces - 2 * (s0 + s));
        mbar_arrive_expect_tx(&full[slot], kCodeTile + sc);
        tma_load_2d(smem_u32(dst), &map_w, smem_u32(&full[slot]), (s0 + s) * (kStageK / 2), n0);
        bulk_g2s(dst + kCodeTile, p.w_scales + ((size_t)blockIdx.x * pieces + 2 * (s0 + s)) * kMxScaleBytes, sc, &full[slot]);
    };
    if (tid == 0) {
        for (int i = 0; i < p.slots; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        mbar_init(&t_full, 1);
        mbar_init(&done, 1);
        fence_mbar_init();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (tid == 0)
        for (int s = 0; s < min(stages, p.slots); ++s) request(s, s);
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kFewCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    // ---- the rows: eight channels an item, four neighbours a block; kBatch loads in flight (one after the other, 8 rows x 2048 took 11 of 18 us) ----
    const int per_row = stages * 32, items = M * per_row;
    const auto place = [&](int m, int c) { return rows + (c >> 5) * kRows + (m >> 3) * 1024 + (m & 7) * 128 + ((((c & 31) >> 2) ^ (m & 7)) << 4) + (c & 3) * 4; };
    const auto take = [&](auto type, auto wide) {
        constexpr int TYPE = decltype(type)::value, kBatch = TYPE == kTypeF32 ? 6 : 8;
        constexpr bool WIDE = decltype(wide)::value;
        for (int i0 = tid; i0 < items; i0 += kFewThreads * kBatch) {           // (a warp is in or out as a whole)
            Eight<TYPE, WIDE, false> x8[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int i = i0 + b * kFewThreads, m = i / per_row, k = s0 * kStageK + 8 * (i - m * per_row);
                x8[b].fetch(reinterpret_cast<const char*>(p.a) + (long long)m * p.lda * (TYPE == kTypeF32 ? 4 : 2), k, i < items ? p.K - k : 0);
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int i = i0 + b * kFewThreads, m = i / per_row, c = i - m * per_row;
                if (i >= items) break;
                float v[8];
                x8[b].widen(v);
                uint32_t scale;
                *reinterpret_cast<uint32_t*>(place(m, c)) = round_block(v, scale);
                if ((c & 3) == 0) rows[(c >> 5) * kRows + NB * 128 + ((c & 31) >> 4) * kMxScaleBytes + (m & 31) * 16 + (m >> 5) * 4 + ((c >> 2) & 3)] = (uint8_t)scale;
            }
        }
    };
    const auto take_type = [&](auto type) {
        if (p.wide) take(type, std::true_type());
        else take(type, std::false_type());
    };
    if (p.a_type == kTypeF32) take_type(std::integral_constant<int, kTypeF32>());
    else if (p.a_type == kTypeBf16) take_type(std::integral_constant<int, kTypeBf16>());
    else take_type(std::integral_constant<int, kTypeF16>());
    // (columns beyond M multiply whatever is there and go nowhere: numbers of 4 bits are all finite, a scale that is not stays in its column)
    fence_proxy_async();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            int s = min(stages, p.slots);
            for (; s < stages; ++s) {
                const int slot = s % p.slots;
                if (!lane_wait(&empty[slot], ((s / p.slots) & 1u) ^ 1u, p.polls)) { ok = false; break; }
                request(s, slot);
            }
            copies_landed(full, p.slots, s);
        }
    } else if (warp == 1) {
        const uint32_t idesc[2] = {mx_idesc(NB, 0), mx_idesc(NB, 1)};
        for (int s = 0; s < stages && ok; ++s) {
            const int slot = s % p.slots;
            if (!pair_wait(&full[slot], (s / p.slots) & 1u, p.polls)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t wa = smem_u32(ring + slot * kSlot), ra = smem_u32(rows + s * kRows);
            const uint64_t adesc = umma_desc(wa), bdesc = umma_desc(ra);
            const uint32_t sa = tmem + 64 + (s & 3) * 16, sb = sa + 8;
            const int here = min(2, pieces - 2 * (s0 + s));
            if (elect_one_sync()) {
                for (int c = 0; c < here; ++c) {
                    scales_to_tmem(sa + 4 * c, scale_desc(wa + kCodeTile + c * kMxScaleBytes));
                    scales_to_tmem(sb + 4 * c, scale_desc(ra + NB * 128 + c * kMxScaleBytes));
                }
                for (int c = 0; c < here; ++c)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        umma_mxfp4(tmem, adesc + 4 * c + 2 * j, bdesc + 4 * c + 2 * j, idesc[j], sa + 4 * c, sb + 4 * c, (s | c | j) != 0 ? 1u : 0u);
                umma_commit(&empty[slot]);
                if (s == stages - 1) umma_commit(&t_full);
            }
            __syncwarp();
        }
        mmas_ended<false>(&done);
    } else if (warp < 6) {
        ok = stages == 0 || pair_wait(&t_full, 0, p.polls);   // (the last CTAs of a cluster may have none: zeros)
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const int c = (warp & 3) * 32 + lane;
        const int n = n0 + c;
        uint32_t v[NB];
        tmem_columns16(tmem + ((uint32_t)((warp & 3) * 32) << 16), v);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int m = 0; m < NB; ++m) {
            const float f = !ok ? CUDART_NAN_F : stages ? __uint_as_float(v[m]) : 0.f;              // (NaN: no result)
            if (S > 1) part[m * 128 + c] = f;
            else if (m < M && n < p.N) put1(p.y, p.y_type, (size_t)m * p.N + n, f);
        }
    }
    if (!ok && lane == 0 && p.ran_out) {
        *reinterpret_cast<volatile int*>(p.ran_out) = 1;
        __threadfence_system();
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kFewCols));
    }
    if (S > 1) {
        cluster_sync_all();
        // the outputs of the tile, dealt to the cluster's CTAs
        for (int i = rank * kFewThreads + tid; i < M * 128; i += S * kFewThreads) {
            const int m = i >> 7, n = n0 + (i & 127);
            if (n >= p.N) continue;
            float u[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) u[r] = r < S ? load_remote(part + i, r) : 0.f;
            float v = u[0];
#pragma unroll
            for (int r = 1; r < 8; ++r)
                if (r < S) v += u[r];
            put1(p.y, p.y_type, (size_t)m * p.N + n, v);
        }
        cluster_sync_all();                                   // (the shares stay until every CTA has read them)
    }
}

// codes [rows][stride / 2] in boxes of box_rows x 128 bytes
bool codes_map(CUtensorMap* map, const void* codes, int rows, int K, int box_rows) {
    const EncodeTiledFn enc = encode_tiled();
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)(mx_stride(K) / 2), (cuuint64_t)rows};
    const cuuint64_t strides[1] = {dims[0]};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// scales, a row of all pieces per block of 128 rows, two pieces of `blocks` of them at a time
bool scales_map(CUtensorMap* map, const void* scales, int rows, int K, int blocks) {
    const EncodeTiledFn enc = encode_tiled();
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)(mx_stride(K) / kMxStride * (kMxScaleBytes / 4)), (cuuint64_t)((rows + 127) / 128)}, strides[1] = {dims[0] * 4};
    const cuuint32_t box[2] = {2 * kMxScaleBytes / 4, (cuuint32_t)blocks}, estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(scales), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether pairs of SMs are the shorter way: rounds of tiles times what a tile takes, in us.  Measured, a stage of 256 channels of a 128 x 128 tile 0.40, of a 256 x 256 tile of a
// pair 0.45, taking a tile out 1.0 and 2.4 (4096 x 16384, with the rounding of the rows, tiles of one SM / of pairs: 4096 channels 189 / 115, 1024 57 / 46, 256 35 / 40;
// 1000 x 8192 x 2048 20 / 17, 200 x 32768 x 256 11.3 / 11.8).
bool on_pairs(int M, int N, int K, int sms) {
    const long long single = ((M + 127LL) / 128 * ((N + 127LL) / 128) + sms - 1) / sms, pairs = ((M + 255LL) / 256 * ((N + kPairN - 1LL) / kPairN) + sms / 2 - 1) / (sms / 2);
    const double stages = (K + kStageK - 1) / kStageK;
    return M > 128 && pairs * std::max(0.45 * stages, 2.4) + 1.0 < single * std::max(0.4 * stages, 1.0);
}

// clusters of two CTAs of the pair kernel that run at the same time
template <int TYPE>
cudaError_t pairs_of(int dev, int* out) {
    static std::atomic<int> known[64];
    if (dev >= 0 && dev < 64 && (*out = known[dev].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = kPairSmem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaFuncSetAttribute(mxfp4_pair_kernel<TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(out, mxfp4_pair_kernel<TYPE>, &cfg);
    if (e != cudaSuccess) return e;
    if (*out < 1) return cudaErrorNotSupported;
    if (dev >= 0 && dev < 64) known[dev].store(*out, std::memory_order_relaxed);
    return cudaSuccess;
}

template <int TYPE>
cudaError_t run_tiled(const Mxfp4Product& p, const uint8_t* a_codes, const uint8_t* a_scales, int dev, int sms, cudaStream_t st) {
    const cudaError_t e = ask_smem<mxfp4_product_kernel<TYPE>>(dev, kSmem4);
    if (e != cudaSuccess) return e;
    const TiledProduct q{a_scales, reinterpret_cast<const uint8_t*>(p.w_scales), p.y, p.M, p.N, p.K, p.ran_out, p.polls};
    cudaLaunchConfig_t cfg = {};
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    CUtensorMap ma, mw;
    const bool pair = on_pairs(p.M, p.N, p.K, sms);
    if (!codes_map(&ma, a_codes, p.M, p.K, kBM) || !codes_map(&mw, p.w_codes, p.N, p.K, pair ? kPairN / 2 : kBN)) return cudaErrorNotSupported;
    if (pair) {
        int pairs = 0;
        CUtensorMap mas, mws;
        const cudaError_t known = pairs_of<TYPE>(dev, &pairs);
        if (known != cudaSuccess) return known;
        if (!scales_map(&mas, a_scales, p.M, p.K, 1) || !scales_map(&mws, p.w_scales, p.N, p.K, 2)) return cudaErrorNotSupported;
        const long long n_tiles = (long long)((p.M + 255) / 256) * ((p.N + kPairN - 1) / kPairN);
        cfg.gridDim = dim3(2 * (unsigned)std::min<long long>(n_tiles, pairs));
        cfg.blockDim = dim3(kPairThreads);
        cfg.dynamicSmemBytes = kPairSmem;
        return cudaLaunchKernelEx(&cfg, mxfp4_pair_kernel<TYPE>, ma, mw, mas, mws, q);
    }
    const long long n_tiles = (long long)((p.M + kBM - 1) / kBM) * ((p.N + kBN - 1) / kBN);
    cfg.gridDim = dim3((unsigned)std::min<long long>(n_tiles, sms));
    cfg.blockDim = dim3(kThreads4);
    cfg.dynamicSmemBytes = kSmem4;
    return cudaLaunchKernelEx(&cfg, mxfp4_product_kernel<TYPE>, ma, mw, q);
}

// CTAs of a cluster, and what they hold: as many CTAs as the chip has SMs, two stages each while there are that many (one beyond that would cost more in joining
// shares than it saves)
bool few_plan(int M, int N, int K, int& S, int& per, int& slots, size_t& smem) {
    if (M > kFewMost) return false;
    const long long tiles = (N + 127) / 128, n_stage = (mx_stride(K) / 128 + 1) / 2;
    const size_t slot = kCodeTile + 1024, row = NB * 128 + 1024;
    for (S = 1; S < 8 && n_stage >= 2 * S && tiles * S < 120; S *= 2) {}
    for (;; S *= 2) {
        if (S > 8) return false;
        const long long each = (n_stage + S - 1) / S;
        const size_t fixed = 1024 + each * row + (S > 1 ? NB * 512 : 0);
        if (fixed + std::min<long long>(each, 2) * slot > (size_t)kFewSmemMost) continue;
        per = (int)each;
        if (M * each > kFewRounded) return false;
        slots = (int)std::min<long long>(each, kFewSlotsMost);
        // two CTAs on an SM where four stages fit: more of them load at a time, and the next launch's come while this one runs (32768 x 2048, 1 row: 8.5 us, else 14.6)
        while (slots > 4 && fixed + slots * slot > (size_t)kFewSmemMost / 2) --slots;
        while (fixed + slots * slot > (size_t)kFewSmemMost) --slots;
        smem = std::max<size_t>(fixed + slots * slot, kFewSmemLeast);
        return tiles <= 0x7fffffffLL;
    }
}

cudaError_t run_few(const Mxfp4Product& p, int S, int per, int slots, size_t smem, int dev, cudaStream_t st) {
    const cudaError_t e = ask_smem<mxfp4_few_rows_kernel>(dev, kFewSmemMost);
    if (e != cudaSuccess) return e;
    CUtensorMap mw;
    if (!codes_map(&mw, p.w_codes, p.N, p.K, 128)) return cudaErrorNotSupported;
    const int wide = wide_rows(p.a, p.a_type, p.lda, p.K);
    const FewProduct q{p.a, p.lda, p.a_type, wide, reinterpret_cast<const uint8_t*>(p.w_scales), p.y, p.y_type, p.M, p.N, p.K, per, slots, p.ran_out, p.polls};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((p.N + 127) / 128, S);
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = S;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = S > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, mxfp4_few_rows_kernel, mw, q);
}

// more rows than a grid has room for: 65535 x 128 at a time
template <typename F>
cudaError_t launch_in_parts(int rows, const F& launch) {
    constexpr long long most = 65535LL * 128;
    for (long long r0 = 0; r0 < rows; r0 += most) {
        const cudaError_t e = launch(r0, (int)std::min(most, rows - r0));
        if (e != cudaSuccess) return e;
        if (r0) ++extra_launches();
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_mxfp4_quantize(const void* x, int type, long long ld, int rows, int K, void* codes, void* scales, cudaStream_t st, bool early) {
    const dim3 grid((K + 255) / 256, (rows + 127) / 128);
    if (grid.y > 65535u) return launch_in_parts(rows, [&](long long r0, int n) {
        return launch_mxfp4_quantize(reinterpret_cast<const char*>(x) + r0 * ld * type_bytes(type), type, ld, n, K, reinterpret_cast<uint8_t*>(codes) + mx_code_bytes(r0, K),
                                     reinterpret_cast<uint8_t*>(scales) + mx_scale_bytes(r0, K), st);
    });
    const auto run = [&](auto kernel) { kernel<<<grid, kQuantThreads, 0, st>>>(x, ld, rows, K, reinterpret_cast<uint32_t*>(codes), reinterpret_cast<uint8_t*>(scales), early); };
    const bool wide = wide_rows(x, type, ld, K);
    if (type == kTypeF32) wide ? run(mxfp4_quantize_kernel<kTypeF32, true>) : run(mxfp4_quantize_kernel<kTypeF32, false>);
    else if (type == kTypeBf16) wide ? run(mxfp4_quantize_kernel<kTypeBf16, true>) : run(mxfp4_quantize_kernel<kTypeBf16, false>);
    else wide ? run(mxfp4_quantize_kernel<kTypeF16, true>) : run(mxfp4_quantize_kernel<kTypeF16, false>);
    return cudaGetLastError();
}

cudaError_t launch_mxfp4_dequantize(const void* codes, const void* scales, int rows, int K, void* out, int type, cudaStream_t st) {
    const dim3 grid((K + 255) / 256, (rows + 127) / 128);
    if (grid.y > 65535u) return launch_in_parts(rows, [&](long long r0, int n) {
        return launch_mxfp4_dequantize(reinterpret_cast<const uint8_t*>(codes) + mx_code_bytes(r0, K), reinterpret_cast<const uint8_t*>(scales) + mx_scale_bytes(r0, K), n, K,
                                       reinterpret_cast<char*>(out) + (size_t)r0 * K * type_bytes(type), type, st);
    });
    const int wide = K % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const auto kernel = type == kTypeF32 ? mxfp4_dequantize_kernel<kTypeF32> : type == kTypeBf16 ? mxfp4_dequantize_kernel<kTypeBf16> : mxfp4_dequantize_kernel<kTypeF16>;
    kernel<<<grid, kQuantThreads, 0, st>>>(reinterpret_cast<const uint8_t*>(codes), reinterpret_cast<const uint8_t*>(scales), rows, K, out, wide);
    return cudaGetLastError();
}

size_t mxfp4_linear_work_bytes(int M, int N, int K) {
    int S, per, slots;
    size_t smem;
    if (few_plan(M, N, K, S, per, slots, smem)) return 0;
    return (mx_code_bytes(M, K) + 127) / 128 * 128 + mx_scale_bytes(M, K);
}

cudaError_t launch_mxfp4_linear(Mxfp4Product p, void* work, cudaStream_t st) {
    int dev = 0, sms = 0;
    cudaError_t e = current_sms(&dev, &sms);
    if (e != cudaSuccess) return e;
    p.ran_out = split_attention_ran_out(dev, st);
    p.polls = gemm_pair_polls();
    if (take_ran_out(dev, st)) return cudaErrorLaunchTimeout;
    int S, per, slots;
    size_t smem;
    if (few_plan(p.M, p.N, p.K, S, per, slots, smem)) return run_few(p, S, per, slots, smem, dev, st);
    uint8_t* const codes = reinterpret_cast<uint8_t*>(work);
    uint8_t* const scales = codes + (mx_code_bytes(p.M, p.K) + 127) / 128 * 128;
    e = launch_mxfp4_quantize(p.a, p.a_type, p.lda, p.M, p.K, codes, scales, st, true);
    if (e != cudaSuccess) return e;
    ++extra_launches();
    return p.y_type == kTypeF32    ? run_tiled<kTypeF32>(p, codes, scales, dev, sms, st)
           : p.y_type == kTypeBf16 ? run_tiled<kTypeBf16>(p, codes, scales, dev, sms, st)
                                   : run_tiled<kTypeF16>(p, codes, scales, dev, sms, st);
}

}  // namespace lm
