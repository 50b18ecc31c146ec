// lm_mxfp4.cu - microscaled 4-bit numbers: rounding rows to them, their values, and products on the tensor cores' own 4-bit path.
//
// Rounding (OCP Microscaling Formats, version 1.0): a block of 32 channels has the scale 2^e, e = floor(log2(largest magnitude)) - 2 (2 is the exponent of the largest
// E2M1 number, 6), at least 2^-127; its elements are x 2^-e to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (half way: to the even code), 6 beyond.  Both steps are exact
// but for that last one, so every implementation of the rule has the same bits.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_split.h"
#include "engine_internal.h"
#include "gemm_tcgen05.h"
#include "lm_mxfp4.h"
#include "tensor_cores.cuh"

namespace lm {
namespace {

using namespace dia;

// ---- rounding and values -------------------------------------------------------------------------------------------------------------------

// eight neighbouring channels of a row; those at or beyond `n` are zero.  wide: 16-byte loads
template <int TYPE>
__device__ __forceinline__ void load8(const void* row, int k, int n, bool wide, float (&v)[8]) {
    if (wide && n >= 8) {
        if (TYPE == kTypeF32) {
            const float4 a = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + k)[0];
            const float4 b = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(row) + k)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(row) + k);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (TYPE == kTypeBf16) {
                    v[2 * e] = __uint_as_float(w[e] << 16);
                    v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
                } else {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                    v[2 * e] = f.x;
                    v[2 * e + 1] = f.y;
                }
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = 0.f;
        if (e < n)
            v[e] = TYPE == kTypeF32    ? reinterpret_cast<const float*>(row)[k + e]
                   : TYPE == kTypeBf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[k + e])
                                       : __half2float(reinterpret_cast<const __half*>(row)[k + e]);
    }
}

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

// place of a scale in the pieces of 128 rows x 128 channels (block: 32 channels)
__device__ __forceinline__ size_t scale_at(long long row, int block, int pieces) {
    return ((size_t)(row >> 7) * pieces + (block >> 2)) * kMxScaleBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// A thread takes eight channels, four neighbours a block.  Rows behind the last one of a piece get scales of zero.
constexpr int kQuantThreads = 256, kQuantItems = 4;
template <int TYPE>
__global__ void __launch_bounds__(kQuantThreads) mxfp4_quantize_kernel(const void* __restrict__ x, long long ld, int rows, int K, int wide, uint32_t* __restrict__ codes,
                                                                       uint8_t* __restrict__ scales) {
    const int per_row = (int)((K + 127) / 128 * 16), pieces = per_row / 16;
    const long long n = (long long)((rows + 127) / 128 * 128) * per_row;
    const long long i0 = (long long)blockIdx.x * (kQuantThreads * kQuantItems) + threadIdx.x;
    float v[kQuantItems][8];
#pragma unroll
    for (int j = 0; j < kQuantItems; ++j) {
        const long long i = i0 + j * kQuantThreads, r = i / per_row;
        const int k = (int)(i - r * per_row) * 8;
        load8<TYPE>(reinterpret_cast<const char*>(x) + r * ld * (TYPE == kTypeF32 ? 4 : 2), k, r < rows ? K - k : 0, wide, v[j]);
    }
#pragma unroll
    for (int j = 0; j < kQuantItems; ++j) {
        const long long i = i0 + j * kQuantThreads, r = i / per_row;
        const int c = (int)(i - r * per_row);
        uint32_t scale;
        const uint32_t code = round_block(v[j], scale);       // (n is a multiple of 32: a warp is in or out as a whole)
        if (i >= n) continue;
        if (r < rows) codes[i] = code;
        if ((c & 3) == 0) scales[scale_at(r, c >> 2, pieces)] = (uint8_t)scale;
    }
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

template <int TYPE>
__global__ void __launch_bounds__(256) mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int K, void* __restrict__ out,
                                                               int wide) {
    const int per_row = (K + 7) / 8, stride = (int)((K + 127) / 128 * 16);
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, r = i / per_row;
    if (r >= rows) return;
    const int c = (int)(i - r * per_row), k = 8 * c;
    const uint32_t code = codes[r * stride + c];
    const float f = scale_value(scales[scale_at(r, c >> 2, stride / 16)]);
    float v[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 t = two_values((code >> (8 * e)) & 255u);
        v[2 * e] = t.x * f;
        v[2 * e + 1] = t.y * f;
    }
    const size_t at = (size_t)r * K + k;
    put4<TYPE>(out, at, make_float4(v[0], v[1], v[2], v[3]), K - k, wide);
    put4<TYPE>(out, at + 4, make_float4(v[4], v[5], v[6], v[7]), K - k - 4, wide);
}

// ---- the product -----------------------------------------------------------------------------------------------------------------------------

constexpr int kBM = 128, kBN = 128, kStageK = 256;            // rows of A and of W in a tile, channels of a stage
constexpr int kCodeTile = 128 * 128;                          // 128 rows x 256 channels, 16 KB
constexpr int kStageBytes = 2 * kCodeTile + 2 * 1024;         // A, W, their scales
constexpr int kStages = 5;
constexpr int kThreads4 = 192;
constexpr int kTurnBytes = 4 * 4096;
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

// One CTA per SM walks 128 x 128 tiles.
//   warp 0    one lane: a stage's codes (TMA, 128-byte swizzle) and scales (plain bulk copies)
//   warp 1    one elected lane: the stage's scales into tensor memory, then its MMAs of 64 channels
//   warps 2-5 take a finished accumulator out through shared memory while the next tile fills the other
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
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(t_empty + 2);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pieces = (p.K + 127) / 128, n_stage = (pieces + 1) / 2;
    const int tiles_m = (p.M + kBM - 1) / kBM, n_tiles = tiles_m * ((p.N + kBN - 1) / kBN);

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&t_full[i], 1); mbar_init(&t_empty[i], 4); }
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
            unsigned i = 0;
            for (int t = blockIdx.x; t < n_tiles && ok; t += gridDim.x) {
                const int tn = t / tiles_m, tm = t % tiles_m;
                for (int s = 0; s < n_stage; ++s, ++i) {
                    const unsigned at = i % kStages;
                    if (!lane_wait(&empty[at], ((i / kStages) & 1u) ^ 1u, p.polls)) { ok = false; break; }
                    unsigned char* const dst = smem + at * kStageBytes;
                    const uint32_t sc = kMxScaleBytes * min(2, pieces - 2 * s);
                    mbar_arrive_expect_tx(&full[at], 2 * kCodeTile + 2 * sc);
                    tma_load_2d(smem_u32(dst), &map_a, smem_u32(&full[at]), s * (kStageK / 2), tm * kBM);
                    tma_load_2d(smem_u32(dst + kCodeTile), &map_w, smem_u32(&full[at]), s * (kStageK / 2), tn * kBN);
                    bulk_g2s(dst + 2 * kCodeTile, p.a_scales + ((size_t)tm * pieces + 2 * s) * kMxScaleBytes, sc, &full[at]);
                    bulk_g2s(dst + 2 * kCodeTile + 1024, p.w_scales + ((size_t)tn * pieces + 2 * s) * kMxScaleBytes, sc, &full[at]);
                }
            }
            // (copies in flight arrive before the CTA goes)
            for (unsigned j = i > (unsigned)kStages ? i - kStages : 0; j < i && !ok; ++j) (void)lane_wait(&full[j % kStages], (j / kStages) & 1u, p.polls);
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
    } else {
        const int q = warp & 3, rr = lane >> 3, ch = lane & 7;
        float* const blk = reinterpret_cast<float*>(turn + (warp - 2) * 4096);
        const bool wide = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
        unsigned it = 0;
        for (int t = blockIdx.x; t < n_tiles; t += gridDim.x, ++it) {
            const int n0 = t / tiles_m * kBN, row0 = t % tiles_m * kBM + q * 32, rows = min(32, p.M - row0);
            ok = ok && pair_wait(&t_full[it & 1u], (it >> 1) & 1u, p.polls);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int cb = 0; cb < kBN / 32; ++cb) {
                const int n = n0 + cb * 32 + 4 * ch;
                if (n0 + cb * 32 >= p.N || rows <= 0) break;
                uint32_t v[32];
                tmem_columns32(tmem + ((uint32_t)(q * 32) << 16) + (it & 1u) * kBN + cb * 32, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                // lane = row: its 16-byte piece c goes to place c ^ (row % 8) of its 128 bytes, and is read a row per eight lanes
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    *reinterpret_cast<uint4*>(blk + lane * 32 + ((c ^ (lane & 7)) << 2)) = make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
                __syncwarp();
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const int r = 4 * g + rr;
                    if (r >= rows || n >= p.N) break;
                    float4 f = *reinterpret_cast<const float4*>(blk + r * 32 + ((ch ^ (r & 7)) << 2));
                    if (!ok) f = make_float4(CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F);      // (no result)
                    put4<TYPE>(p.y, (size_t)(row0 + r) * p.N + n, f, p.N - n, wide);
                }
                __syncwarp();
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

template <int TYPE>
cudaError_t run_tiled(const Mxfp4Product& p, const uint8_t* a_codes, const uint8_t* a_scales, int dev, int sms, cudaStream_t st) {
    const cudaError_t e = ask_smem<mxfp4_product_kernel<TYPE>>(dev, kSmem4);
    if (e != cudaSuccess) return e;
    CUtensorMap ma, mw;
    if (!codes_map(&ma, a_codes, p.M, p.K, kBM) || !codes_map(&mw, p.w_codes, p.N, p.K, kBN)) return cudaErrorNotSupported;
    const TiledProduct q{a_scales, reinterpret_cast<const uint8_t*>(p.w_scales), p.y, p.M, p.N, p.K, p.ran_out, p.polls};
    const long long n_tiles = (long long)((p.M + kBM - 1) / kBM) * ((p.N + kBN - 1) / kBN);
    mxfp4_product_kernel<TYPE><<<(int)std::min<long long>(n_tiles, sms), kThreads4, kSmem4, st>>>(ma, mw, q);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mxfp4_quantize(const void* x, int type, long long ld, int rows, int K, void* codes, void* scales, cudaStream_t st) {
    const long long n = (long long)((rows + 127) / 128 * 128) * (mx_stride(K) / 8), per = kQuantThreads * kQuantItems, blocks = (n + per - 1) / per;
    if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
    const int wide = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && ld * type_bytes(type) % 16 == 0;
    const auto kernel = type == kTypeF32 ? mxfp4_quantize_kernel<kTypeF32> : type == kTypeBf16 ? mxfp4_quantize_kernel<kTypeBf16> : mxfp4_quantize_kernel<kTypeF16>;
    kernel<<<(unsigned)blocks, kQuantThreads, 0, st>>>(x, ld, rows, K, wide, reinterpret_cast<uint32_t*>(codes), reinterpret_cast<uint8_t*>(scales));
    return cudaGetLastError();
}

cudaError_t launch_mxfp4_dequantize(const void* codes, const void* scales, int rows, int K, void* out, int type, cudaStream_t st) {
    const long long blocks = ((long long)rows * ((K + 7) / 8) + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
    const int wide = K % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const auto kernel = type == kTypeF32 ? mxfp4_dequantize_kernel<kTypeF32> : type == kTypeBf16 ? mxfp4_dequantize_kernel<kTypeBf16> : mxfp4_dequantize_kernel<kTypeF16>;
    kernel<<<(unsigned)blocks, 256, 0, st>>>(reinterpret_cast<const uint32_t*>(codes), reinterpret_cast<const uint8_t*>(scales), rows, K, out, wide);
    return cudaGetLastError();
}

size_t mxfp4_linear_work_bytes(int M, int K) { return (mx_code_bytes(M, K) + 127) / 128 * 128 + mx_scale_bytes(M, K); }

cudaError_t launch_mxfp4_linear(Mxfp4Product p, void* work, cudaStream_t st) {
    int dev = 0, sms = 0;
    cudaError_t e = current_sms(&dev, &sms);
    if (e != cudaSuccess) return e;
    p.ran_out = split_attention_ran_out(dev, st);
    p.polls = gemm_pair_polls();
    if (take_ran_out(dev, st)) return cudaErrorLaunchTimeout;
    uint8_t* const codes = reinterpret_cast<uint8_t*>(work);
    uint8_t* const scales = codes + (mx_code_bytes(p.M, p.K) + 127) / 128 * 128;
    e = launch_mxfp4_quantize(p.a, p.a_type, p.lda, p.M, p.K, codes, scales, st);
    if (e != cudaSuccess) return e;
    ++extra_launches();
    return p.y_type == kTypeF32    ? run_tiled<kTypeF32>(p, codes, scales, dev, sms, st)
           : p.y_type == kTypeBf16 ? run_tiled<kTypeBf16>(p, codes, scales, dev, sms, st)
                                   : run_tiled<kTypeF16>(p, codes, scales, dev, sms, st);
}

}  // namespace lm
