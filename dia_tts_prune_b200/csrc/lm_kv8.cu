// lm_kv8.cu - a cache of keys and values in 8 bits: rows written into it, numbers read back, and the attention of few rows.
//
// The tokens of a page and head share 2^e.  e is the smallest exponent, at least -100, for which the largest magnitude is at most 448 2^e (E4M3) or 127 2^e (two's
// complement): nothing saturates.  A page fills token by token, so e may have to grow; then the codes that are there are rounded again, to the new step.  A power of two
// is what makes that cheap in accuracy: E4M3 codes stay what they are until they fall below its smallest exponent, and no code is ever rounded twice to the same step.
// A number that is not finite makes the page's scale NaN: all of the page's head then stands for NaNs, until its first token is written again.  Codes themselves are
// always finite, so that a weight of zero times a code of a token that nobody sees is zero.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gemm_tcgen05.h"
#include "lm_device.cuh"
#include "lm_kv8.cuh"
#include "lm_kv8.h"

namespace lm {
namespace {

constexpr int kLowestExp = -100;

// 2^e, e from -126 to 127; smaller ones are 0 (a code times that rounds to zero)
__device__ __forceinline__ float power(int e) { return e < -126 ? 0.f : __uint_as_float((unsigned)(e + 127) << 23); }

// The exponent that the largest magnitude (as bits) needs: magnitudes up to 1.75 2^(x + 8) = 448 2^x, or 1.984375 2^(x + 6) = 127 2^x.
template <int FORMAT>
__device__ __forceinline__ int needed(uint32_t most) {
    constexpr int kShift = FORMAT == kKvE4m3 ? 8 : 6;
    constexpr uint32_t kPart = FORMAT == kKvE4m3 ? 0x600000u : 0x7e0000u;
    return max((int)(most >> 23) - 127 - kShift + ((most & 0x7fffffu) > kPart), kLowestExp);
}

template <int FORMAT>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {        // |each| at most 448 or 127
    uint32_t r;
    if constexpr (FORMAT == kKvE4m3) {
        asm("{\n\t.reg .b16 lo, hi;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
            "mov.b32 %0, {lo, hi};\n\t}"
            : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
    } else {
        r = (__float2int_rn(a) & 255) | (__float2int_rn(b) & 255) << 8 | (__float2int_rn(c) & 255) << 16 | (uint32_t)__float2int_rn(d) << 24;
    }
    return r;
}
// Eight channels of a row from channel k on, those at or beyond n are zero.  WIDE: rows of whole 16 bytes, n is a multiple of 8.
template <int TYPE, bool WIDE>
struct Eight {
    uint4 w[TYPE == kTypeF32 ? 2 : 1];
    __device__ __forceinline__ void fetch(const Element<TYPE>* p, int n) {
        constexpr int kWords = TYPE == kTypeF32 ? 2 : 1;
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = n > 0 ? reinterpret_cast<const uint4*>(p)[i] : make_uint4(0u, 0u, 0u, 0u);
        } else {
            Element<TYPE> v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : narrow<Element<TYPE>>(0.f);
            memcpy(w, v, sizeof(v));
        }
    }
    __device__ __forceinline__ void numbers(float (&f)[8]) const {
        Element<TYPE> v[8];
        memcpy(v, w, sizeof(v));
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = widen(v[e]);
    }
};

// ---- rows into pages -----------------------------------------------------------------------------------------------------------------------
// A warp takes what comes into one page of one head, keys or values: it reads the rows for their largest magnitude, makes the page's step as large as it has to be, rounds the
// codes that are there if it grew, and writes the new ones.  Eight groups of eight channels a lane stay in registers in between (16 tokens of 128 channels); what is beyond is
// read again, from L2.  `chunk` rows in turn belong to a warp: a page border or a sequence's first row among them starts a page.
constexpr int kAppendThreads = 128, kKept = 8;
template <int FORMAT, int TYPE, bool WIDE>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(Kv8Cache c, Kv8Step s, Kv8Rows k, Kv8Rows v, int chunk) {
    const int lane = threadIdx.x & 31;
    const long long task = ((long long)blockIdx.x * kAppendThreads + threadIdx.x) >> 5;
    const int sides = 2 * c.kv_heads, side = (int)(task % sides), head = side >> 1;
    const long long row0 = task / sides * chunk;
    if (row0 >= s.rows) return;
    const Kv8Rows in = side & 1 ? v : k;
    uint8_t* const codes = side & 1 ? c.values : c.keys;
    float* const scales = side & 1 ? c.value_scales : c.key_scales;
    const Element<TYPE>* const x = reinterpret_cast<const Element<TYPE>*>(in.x) + head * in.head;
    const int groups = (c.dim + 7) >> 3, page_size = 1 << c.page_shift, last = (int)min(row0 + chunk, (long long)s.rows);
    int row = (int)row0, seq = s.sequence_of(row);
    while (row < last) {
        if (seq < 0) {                                        // no row of a sequence: on to the next one that is
            if (++row < last) seq = s.sequence_of(row);
            continue;
        }
        const int begin = s.begin(seq), end = s.end(seq), past = s.past[seq];
        const long long pos = (long long)past + (row - begin);
        const int place = (int)(pos & (page_size - 1));
        const int ends = min(end, row + page_size - place);    // of the rows that go into this page
        if (past >= 0 && (row == begin || place == 0)) {
            const int page = s.page(seq, pos >> c.page_shift, c.pages), n = (ends - row) * groups;
            if (page >= 0) {
                Eight<TYPE, WIDE> kept[kKept];
                uint32_t most = 0;
                const auto fetch = [&](Eight<TYPE, WIDE>& e, int i) {
                    const int r = i / groups, g = i - r * groups;
                    if (i < n) e.fetch(x + (row + r) * in.row + 8 * g, c.dim - 8 * g);
                    else e = {};
                };
                const auto look = [&](const Eight<TYPE, WIDE>& e) {
                    float f[8];
                    e.numbers(f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(f[j]) & 0x7fffffffu);
                };
#pragma unroll
                for (int j = 0; j < kKept; ++j) fetch(kept[j], lane + 32 * j);
#pragma unroll
                for (int j = 0; j < kKept; ++j) look(kept[j]);
                for (int i = lane + 32 * kKept; i < n; i += 32) {
                    Eight<TYPE, WIDE> e;
                    fetch(e, i);
                    look(e);
                }
                most = __reduce_max_sync(0xffffffffu, most);
                float* const scale = scales + (size_t)page * c.kv_heads + head;
                uint8_t* const at = codes + (((size_t)page * c.kv_heads + head) << c.page_shift) * c.stride;
                const uint32_t old = place ? __float_as_uint(*scale) & 0x7fffffffu : 0u;
                const bool bad = most >= 0x7f800000u || old >= 0x7f800000u;
                int e = needed<FORMAT>(most);
                if (place && !bad) {
                    const int before = (int)(old >> 23) - 127;
                    if (before >= e) {
                        e = before;
                    } else {
                        const float f = power(before - e);
                        for (int i = lane; i < place * (c.stride >> 4); i += 32) {
                            uint4* const p = reinterpret_cast<uint4*>(at) + i;
                            uint4 w = *p;
                            uint32_t* const u = &w.x;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float4 t = values4<FORMAT>(u[j], f);
                                u[j] = encode4<FORMAT>(t.x, t.y, t.z, t.w);
                            }
                            *p = w;
                        }
                    }
                }
                __syncwarp();                                  // (every lane has read the old scale)
                if (lane == 0) *scale = bad ? __uint_as_float(0x7fc00000u) : power(e);
                const float f = power(-e);
                const auto write = [&](const Eight<TYPE, WIDE>& g8, int i) {
                    if (i >= n) return;
                    const int r = i / groups, g = i - r * groups;
                    float t[8];
                    g8.numbers(t);
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[j] = bad ? 0.f : t[j] * f;
                    const uint2 w = make_uint2(encode4<FORMAT>(t[0], t[1], t[2], t[3]), encode4<FORMAT>(t[4], t[5], t[6], t[7]));
                    uint2* const p = reinterpret_cast<uint2*>(at + (size_t)(place + r) * c.stride) + g;
                    p[0] = w;
                    if (g == groups - 1 && (groups & 1)) p[1] = make_uint2(0u, 0u);        // (up to the row's 16 bytes)
                };
#pragma unroll
                for (int j = 0; j < kKept; ++j) write(kept[j], lane + 32 * j);
                for (int i = lane + 32 * kKept; i < n; i += 32) {
                    Eight<TYPE, WIDE> g8;
                    fetch(g8, i);
                    write(g8, i);
                }
            }
        }
        row = ends;
        if (row == end && row < last) seq = s.sequence_of(row);
    }
}

// ---- numbers out of pages ------------------------------------------------------------------------------------------------------------------
// A CTA takes kReadRows rows (fewer where there are few): where each of them lies is looked up once, then a thread takes 16 bytes of what goes out.
constexpr int kReadThreads = 256, kReadMostRows = 32;
template <int FORMAT, int TYPE, bool WIDE>
__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(Kv8Cache c, Kv8Step s, Element<TYPE>* k, Element<TYPE>* v, int rows_each) {
    __shared__ long long where[kReadMostRows];                // the row's page and place in it, in rows of a head; -1: not there
    const int row0 = blockIdx.x * rows_each, n = min(rows_each, s.rows - row0);
    if (threadIdx.x < n) {
        const int row = row0 + threadIdx.x, seq = s.sequence_of(row);
        long long at = -1;
        if (seq >= 0) {
            const int past = s.past[seq];
            const long long pos = (long long)past + (row - s.begin(seq));
            const int page = past >= 0 ? s.page(seq, pos >> c.page_shift, c.pages) : -1;
            if (page >= 0) at = (long long)page << 32 | (pos & ((1 << c.page_shift) - 1));
        }
        where[threadIdx.x] = at;
    }
    __syncthreads();
    constexpr int kEach = 16 / sizeof(Element<TYPE>);
    const int parts = (c.dim + kEach - 1) / kEach, per_row = 2 * c.kv_heads * parts;
    for (int i = threadIdx.x; i < n * per_row; i += kReadThreads) {
        const int r = i / per_row, j = i - r * per_row, side = j / (c.kv_heads * parts), hp = j - side * c.kv_heads * parts, head = hp / parts, part = hp - head * parts;
        const long long at = where[r];
        Element<TYPE> out[kEach];
        if (at >= 0) {
            const size_t page_head = (size_t)(at >> 32) * c.kv_heads + head;
            const uint8_t* const p = (side ? c.values : c.keys) + ((page_head << c.page_shift) + (uint32_t)at) * c.stride + part * kEach;
            const float scale = (side ? c.value_scales : c.key_scales)[page_head];
#pragma unroll
            for (int e = 0; e < kEach; e += 4) {
                const float4 t = values4<FORMAT>(*reinterpret_cast<const uint32_t*>(p + e), scale);
                out[e] = narrow<Element<TYPE>>(t.x);
                out[e + 1] = narrow<Element<TYPE>>(t.y);
                out[e + 2] = narrow<Element<TYPE>>(t.z);
                out[e + 3] = narrow<Element<TYPE>>(t.w);
            }
        } else {
#pragma unroll
            for (int e = 0; e < kEach; ++e) out[e] = narrow<Element<TYPE>>(0.f);
        }
        Element<TYPE>* const to = (side ? v : k) + ((size_t)(row0 + r) * c.kv_heads + head) * c.dim + part * kEach;
        if constexpr (WIDE) {
            uint4 w;
            memcpy(&w, out, 16);
            *reinterpret_cast<uint4*>(to) = w;
        } else {
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (part * kEach + e < c.dim) to[e] = out[e];
        }
    }
}

// ---- attention of few rows -----------------------------------------------------------------------------------------------------------------
// x = scale log2(e) q . key in powers of two, p = 2^(x - max x), o = sum p value / (sum p + 2^(sink log2(e) - max x)).
//
// What bounds it is the cache's bytes.  The 16 rows of a tile are (token, query head) pairs that share a key head, so a token's codes are read once for the group; tiles of a
// sequence lie next to one another in the order of the work.  Work is counted in blocks of 16 tokens over all sequences, heads and tiles and dealt to the CTAs in equal runs, so that
// one long sequence fills the GPU and lengths need not be alike; runs that share a tile leave (max, sum, output) and a second kernel joins them, always in the same order.
//
// A warp keeps its own ring of blocks in shared memory, filled by asynchronous copies that swizzle 16-byte pieces (rows lie 128 bytes apart, which would be the same banks), and
// multiplies on the tensor cores (mma.sync, 16 x 8 x 16: eight columns are what a token group has, and nothing is waited for across warps; the tensor pipe is far from what
// bounds it).  A thread's four codes of a 32-bit word are four channels of a key, whichever: queries are laid out to match; a thread's word of a value is transposed against
// those of three other tokens by byte permutations.
//
// Codes are exact in fp16.  A row of queries is scaled by a power of two to below 2^14 and taken as one fp16 term (bf16 and fp16 rows: exact but for channels 2^-27 below the
// row's largest), or two (fp32: 22 bits).  Weights: the page's value scale is part of the exponent, 2^(x + e - max (x + e)) 2^14, so that the largest contribution, not the largest
// weight, is what fp16's 11 bits count from (fp32 rows: two terms, 22 bits); sums, maxima and outputs are fp32, and the denominator is summed from fp32 weights without the scale.
constexpr int kRowTile = 16, kFewWarps = 4, kFewThreads = 32 * kFewWarps, kMetaBlocks = 256;
constexpr int kMinBlocks = 8;                                  // of a CTA's run

template <int DP, int TERMS>
struct Few {
    static constexpr int kSide = kKvBlock * DP;               // bytes of a block's keys, or values
    static constexpr int kStages = DP == 64 ? 8 : DP == 128 ? 4 : 3;
    static constexpr int kRing = kFewWarps * kStages * 2 * kSide;
    static constexpr int kQ = TERMS * (DP / 16) * 32 * 16;    // fragments of the queries
    static constexpr int kSmem = kRing + kQ + kMetaBlocks * 12 + 16 * 4 + kFewWarps * 16 * 12 + 256;
    static constexpr int kCtas = DP == 256 ? 1 : DP * TERMS > 128 ? 2 : 3;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// where 16-byte piece `c` of row `r` of a block lies
template <int DP>
__device__ __forceinline__ int piece_at(int r, int c) {
    if constexpr (DP == 64) return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) << 4);
    else return r * DP + ((c ^ ((r & 2) | (((r << 2) ^ r) & 4))) << 4);
}

// Blocks of 16 tokens that a sequence's rows look at, and its share of the work
struct Span {
    int begin, n, past, low, blocks, tiles;                   // low: the first block
    __device__ __forceinline__ long long units(int kv_heads) const { return (long long)kv_heads * tiles * blocks; }
};
__device__ __forceinline__ Span span_of(const Kv8Step& s, const Kv8Attention& a, int i, int group, int page_shift) {
    const int window = a.window;
    Span p;
    p.begin = s.begin(i);
    p.n = max(s.end(i) - p.begin, 0);
    p.past = s.past[i];
    p.low = window > 0 ? (int)(max(0ll, (long long)p.past + 1 - window) / kKvBlock) : 0;
    const long long end = min((long long)max(p.past, 0) + p.n, (long long)s.max_pages << page_shift);
    p.blocks = max(1, (int)((end + kKvBlock - 1) / kKvBlock) - p.low);
    p.tiles = (long long)p.n * group > a.few_most ? 0 : (p.n * group + kRowTile - 1) / kRowTile;
    return p;
}

// The sequence that holds the unit `per * nth` of all, where per = what a CTA takes (all threads; seq < 0: there is none)
struct Place {
    int seq;
    long long base, per, total;
};
__device__ __forceinline__ Place find_place(const Kv8Step& s, const Kv8Attention& a, int kv_heads, int group, int page_shift, int ctas, int nth) {
    __shared__ long long sums[kFewWarps];
    __shared__ Place found;
    const int each = (s.sequences + kFewThreads - 1) / kFewThreads, i0 = threadIdx.x * each, i1 = min(i0 + each, s.sequences);
    long long mine = 0;
    for (int i = i0; i < i1; ++i) mine += span_of(s, a, i, group, page_shift).units(kv_heads);
    long long upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, upto, d);
        if ((threadIdx.x & 31) >= d) upto += o;
    }
    if ((threadIdx.x & 31) == 31) sums[threadIdx.x >> 5] = upto;
    if (threadIdx.x == 0) found.seq = -1;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
        if (w < (threadIdx.x >> 5)) upto += sums[w];
        total += sums[w];
    }
    const long long per = max((total + ctas - 1) / ctas, (long long)kMinBlocks), unit = per * nth;
    if (unit >= upto - mine && unit < upto) {
        long long base = upto - mine;
        int i = i0;
        for (;; ++i) {
            const long long u = span_of(s, a, i, group, page_shift).units(kv_heads);
            if (unit < base + u) break;
            base += u;
        }
        found = {i, base, per, total};
    }
    __syncthreads();
    return found;
}

template <int DP, int FORMAT, int TERMS>
__global__ void __launch_bounds__(kFewThreads, Few<DP, TERMS>::kCtas) kv8_attention_few_kernel(Kv8Cache c, Kv8Step s, Kv8Attention a, float* part, RowStats* part_stats) {
    using F = Few<DP, TERMS>;
    constexpr int kSteps = DP / 16, kHalves = DP == 256 ? 2 : 1, kWords = DP == 64 ? 2 : 4, kCols = kHalves * kWords * 4;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const ring = smem + (threadIdx.x >> 5) * (F::kStages * 2 * F::kSide);
    uint4* const q_frags = reinterpret_cast<uint4*>(smem + F::kRing);
    int* const meta_page = reinterpret_cast<int*>(smem + F::kRing + F::kQ);
    float* const meta_ks = reinterpret_cast<float*>(meta_page + kMetaBlocks);
    float* const meta_ev = meta_ks + kMetaBlocks;
    float* const row_scale = meta_ev + kMetaBlocks;                                // [16] of the queries, with the scores' scale
    RowStats* const stats = reinterpret_cast<RowStats*>(row_scale + 16);           // [warps][16]
    float* const sums = reinterpret_cast<float*>(smem);                            // [warps][16][DP], when the ring is empty
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, group = a.heads / c.kv_heads;
    zero_rows_of_none(s, a, c.dim, (long long)blockIdx.x * kFewThreads + threadIdx.x, (long long)gridDim.x * kFewThreads);
    Place at = find_place(s, a, c.kv_heads, group, c.page_shift, gridDim.x, blockIdx.x);
    if (at.seq < 0) return;
    long long unit = at.per * blockIdx.x;
    const long long unit_end = min(unit + at.per, at.total);
    Span sp = span_of(s, a, at.seq, group, c.page_shift);

    while (unit < unit_end) {
        while (unit >= at.base + sp.units(c.kv_heads)) {                             // (sequences without rows have no units)
            at.base += sp.units(c.kv_heads);
            sp = span_of(s, a, ++at.seq, group, c.page_shift);
        }
        const long long item = (unit - at.base) / sp.blocks;
        const int b0 = (int)(unit - at.base - item * sp.blocks), count = (int)min((long long)sp.blocks - b0, unit_end - unit);
        const int head = (int)(item / sp.tiles), tile = (int)(item - (long long)head * sp.tiles);
        const int rows = min(kRowTile, sp.n * group - tile * kRowTile), p0 = tile * kRowTile;
        unit += count;

        // queries: a warp scales four rows and leaves them as the products' fragments
        for (int r = warp; r < kRowTile; r += kFewWarps) {
            const int p = p0 + r, row = sp.begin + p / group;
            const long long q_at = row * a.q.row + (head * group + p % group) * a.q.head;
            float v[DP / 32];
            uint32_t most = 0;
#pragma unroll
            for (int j = 0; j < DP / 32; ++j) {
                const int d = lane + 32 * j;
                v[j] = r < rows && d < c.dim ? load_q(a, q_at + d) : 0.f;
                most = max(most, __float_as_uint(v[j]) & 0x7fffffffu);
            }
            most = __reduce_max_sync(0xffffffffu, most);
            const uint32_t e = most == 0 ? 127u : max(most >> 23, 14u);
            const float f = __uint_as_float((267u - e) << 23), back = __uint_as_float((e - 13u) << 23);      // 2^(140 - e): to below 2^14, and the way back
            if (lane == 0) row_scale[r] = e == 255u ? __uint_as_float(0x7fc00000u) : back * (a.scale * kLog2e);
#pragma unroll
            for (int j = 0; j < DP / 32; ++j) {
                const int d = lane + 32 * j, chunk = d >> 4, step = (chunk >> 2) * 4 + ((d & 15) >> 2), x = d & 3, reg = (x >> 1) * 2 + (r >> 3);
                __half* const to = reinterpret_cast<__half*>(q_frags) + ((step * 32 + (r & 7) * 4 + (chunk & 3)) * 4 + reg) * 2 + (x & 1);
                const float y = e == 255u ? 0.f : v[j] * f;
                const __half hi = __float2half_rn(y);
                to[0] = hi;
                if constexpr (TERMS == 2) to[kSteps * 32 * 8] = __float2half_rn(y - __half2float(hi));
            }
        }
        __syncthreads();
        constexpr bool kInRegs = DP * TERMS <= 128;
        uint4 qf[kInRegs ? TERMS * kSteps : 1];
        if constexpr (kInRegs) {
#pragma unroll
            for (int j = 0; j < TERMS * kSteps; ++j) qf[j] = q_frags[j * 32 + lane];
        }
        const float f0 = row_scale[g], f1 = row_scale[g + 8];
        // positions of the tile's rows, first and last, and of this thread's two
        const long long pos_a = (long long)sp.past + p0 / group, pos_b = (long long)sp.past + (p0 + rows - 1) / group;
        const long long pos0 = (long long)sp.past + min(p0 + g, p0 + rows - 1) / group, pos1 = (long long)sp.past + min(p0 + g + 8, p0 + rows - 1) / group;
        const long long back = a.window > 0 ? a.window - 1 : (1ll << 40);
        const long long seen_from = max(0ll, pos_a - back), clear_from = max(0ll, pos_b - back);

        float o[kCols][4], m0 = -INFINITY, m1 = -INFINITY, w0 = -INFINITY, w1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int j = 0; j < kCols; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.f;

        for (int m_at = 0; m_at < count; m_at += kMetaBlocks) {
            const int m_n = min(kMetaBlocks, count - m_at);
            if (m_at) __syncthreads();                                               // (the last ones have been read)
            for (int i = threadIdx.x; i < m_n; i += kFewThreads) {
                const long long tok = (long long)(sp.low + b0 + m_at + i) * kKvBlock;
                int page = -1;
                if (sp.past >= 0 && tok <= pos_b && tok + kKvBlock > seen_from) page = s.page(at.seq, tok >> c.page_shift, c.pages);
                meta_page[i] = page;
                if (page >= 0) {
                    const size_t ph = (size_t)page * c.kv_heads + head;
                    const uint32_t vs = __float_as_uint(c.value_scales[ph]);
                    meta_ks[i] = c.key_scales[ph];
                    meta_ev[i] = vs >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : (float)((int)(vs >> 23) - 127);
                }
            }
            __syncthreads();
            const auto issue = [&](int i, int stage) {                               // block i of the list into a slot of the ring
                if (i < m_n && meta_page[i] >= 0) {
                    const long long tok = (long long)(sp.low + b0 + m_at + i) * kKvBlock;
                    const size_t from = ((((size_t)meta_page[i] * c.kv_heads + head) << c.page_shift) + (size_t)(tok & ((1 << c.page_shift) - 1))) * c.stride;
                    const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring + stage * 2 * F::kSide);
#pragma unroll
                    for (int j = 0; j < DP / 32; ++j) {
                        const int x = lane + 32 * j, r = x / (DP / 16), p = x % (DP / 16), n = p * 16 < c.stride ? 16 : 0;
                        const size_t off = from + (size_t)r * c.stride + (n ? p * 16 : 0);
                        const uint32_t d = to + piece_at<DP>(r, p);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(c.keys + off), "r"(n) : "memory");
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + F::kSide), "l"(c.values + off), "r"(n) : "memory");
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
#pragma unroll
            for (int j = 0; j < F::kStages - 1; ++j) issue(warp + kFewWarps * j, j);
            int stage = 0;
            for (int i = warp; i < m_n; i += kFewWarps) {
                asm volatile("cp.async.wait_group %0;" ::"n"(F::kStages - 2) : "memory");
                __syncwarp();                                                        // the block is there for every lane, and the slot in front has been read by all
                issue(i + kFewWarps * (F::kStages - 1), stage == 0 ? F::kStages - 1 : stage - 1);
                const uint8_t* const keys = ring + stage * 2 * F::kSide;
                const uint8_t* const values = keys + F::kSide;
                stage = stage + 1 == F::kStages ? 0 : stage + 1;
                if (meta_page[i] < 0) continue;

                float x[2][4] = {};
#pragma unroll
                for (int h = 0; h < DP / 64; ++h) {
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint4 w4 = *reinterpret_cast<const uint4*>(keys + piece_at<DP>(8 * b + g, t + 4 * h));
                        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t lo, hi;
                            decode4<FORMAT>(w[j], lo, hi);
#pragma unroll
                            for (int e = 0; e < TERMS; ++e) {
                                const int f = e * kSteps + 4 * h + j;
                                mma16816(x[b], kInRegs ? qf[kInRegs ? f : 0] : q_frags[f * 32 + lane], lo, hi);
                            }
                        }
                    }
                }
                const float ks = meta_ks[i], ev = meta_ev[i], k0 = f0 * ks, k1 = f1 * ks;
#pragma unroll
                for (int b = 0; b < 2; ++b) { x[b][0] *= k0; x[b][1] *= k0; x[b][2] *= k1; x[b][3] *= k1; }
                const long long tok = (long long)(sp.low + b0 + m_at + i) * kKvBlock;
                const bool clear = tok + kKvBlock - 1 <= pos_a && tok >= clear_from;   // every row sees all of the block
                uint32_t hidden = 0;
                if (!clear) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const long long key = tok + 8 * b + 2 * t + (e & 1), pos = e < 2 ? pos0 : pos1;
                            if (key > pos || key < pos - back) {
                                x[b][e] = -INFINITY;
                                hidden |= 1u << (4 * b + e);
                            }
                        }
                }
                float t0 = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1])), t1 = fmaxf(fmaxf(x[0][2], x[0][3]), fmaxf(x[1][2], x[1][3]));
                t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
                t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
                t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
                t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
                const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1), u0 = fmaxf(w0, t0 + ev), u1 = fmaxf(w1, t1 + ev);
                if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1 || u0 > w0 || u1 > w1)) {
                    const float a0 = lower_to(m0, n0), a1 = lower_to(m1, n1), c0 = lower_to(w0, u0), c1 = lower_to(w1, u1);
                    l0 *= a0;
                    l1 *= a1;
#pragma unroll
                    for (int j = 0; j < kCols; ++j) { o[j][0] *= c0; o[j][1] *= c0; o[j][2] *= c1; o[j][3] *= c1; }
                    m0 = n0; m1 = n1; w0 = u0; w1 = u1;
                }
                // (rows that have seen nothing yet: any reference will do)
                const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
                const float s0 = (w0 == -INFINITY ? 0.f : w0) - ev - kWeightBits, s1 = (w1 == -INFINITY ? 0.f : w1) - ev - kWeightBits;
                float p[2][4];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    l0 += exp2_fast(x[b][0] - r0) + exp2_fast(x[b][1] - r0);
                    l1 += exp2_fast(x[b][2] - r1) + exp2_fast(x[b][3] - r1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[b][e] = exp2_fast(x[b][e] - (e < 2 ? s0 : s1));
                        if (!clear && (hidden >> (4 * b + e) & 1)) p[b][e] = 0.f;     // (whatever the page's scales are)
                    }
                }
                const uint4 hi = make_uint4(pack_half(p[0][0], p[0][1]), pack_half(p[0][2], p[0][3]), pack_half(p[1][0], p[1][1]), pack_half(p[1][2], p[1][3]));
                uint4 lo = hi;
                if constexpr (TERMS == 2) {
                    const auto rest = [](float x, float y, uint32_t h) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
                        return pack_half(x - f.x, y - f.y);
                    };
                    lo = make_uint4(rest(p[0][0], p[0][1], hi.x), rest(p[0][2], p[0][3], hi.y), rest(p[1][0], p[1][1], hi.z), rest(p[1][2], p[1][3], hi.w));
                }
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    uint32_t w[4][4];                                                // [token 2 t, 2 t + 1, 2 t + 8, 2 t + 9][word]
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 2 * t + (e & 1) + 8 * (e >> 1);
                        if constexpr (DP == 64) {
                            const uint2 v2 = *reinterpret_cast<const uint2*>(values + piece_at<DP>(r, g >> 1) + 8 * (g & 1));
                            w[e][0] = v2.x; w[e][1] = v2.y;
                        } else {
                            const uint4 v4 = *reinterpret_cast<const uint4*>(values + piece_at<DP>(r, 8 * h + g));
                            w[e][0] = v4.x; w[e][1] = v4.y; w[e][2] = v4.z; w[e][3] = v4.w;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < kWords; ++j) {
                        uint32_t b0[4], b1[4];                                       // of four channels: the pairs of tokens
                        decode4<FORMAT>(__byte_perm(w[0][j], w[1][j], 0x5140), b0[0], b0[1]);
                        decode4<FORMAT>(__byte_perm(w[0][j], w[1][j], 0x7362), b0[2], b0[3]);
                        decode4<FORMAT>(__byte_perm(w[2][j], w[3][j], 0x5140), b1[0], b1[1]);
                        decode4<FORMAT>(__byte_perm(w[2][j], w[3][j], 0x7362), b1[2], b1[3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            mma16816(o[(h * kWords + j) * 4 + e], hi, b0[e], b1[e]);
                            if constexpr (TERMS == 2) mma16816(o[(h * kWords + j) * 4 + e], lo, b0[e], b1[e]);
                        }
                    }
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }

        // the warps' sums meet in shared memory
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        __syncthreads();                                                             // every warp is done with its ring
        if (t == 0) {
            stats[warp * 16 + g] = {m0, w0, l0};
            stats[warp * 16 + g + 8] = {m1, w1, l1};
        }
        // column 2 t (or 2 t + 1) of product (h, j) is channel 128 h + 16 (2 t) + j, eight products of 64 channels 8 (2 t) + j
        constexpr int kRun = DP == 64 ? 8 : 16;
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float* const to = sums + (size_t)(warp * 16 + g + 8 * (e >> 1)) * DP + 128 * h + kRun * (2 * t + (e & 1));
#pragma unroll
                for (int j = 0; j < kRun; j += 4)
                    *reinterpret_cast<float4*>(to + j) = make_float4(o[h * 16 + j][e], o[h * 16 + j + 1][e], o[h * 16 + j + 2][e], o[h * 16 + j + 3][e]);
            }
        __syncthreads();
        const bool whole = b0 == 0 && count == sp.blocks;
        const size_t slot = 2 * (size_t)blockIdx.x + (b0 == 0);
        for (int i = threadIdx.x; i < rows * (DP / 4); i += kFewThreads) {
            const int r = i / (DP / 4), d = i % (DP / 4) * 4;
            float m = -INFINITY, w = -INFINITY, l = 0.f;
#pragma unroll
            for (int v = 0; v < kFewWarps; ++v) {
                m = fmaxf(m, stats[v * 16 + r].m);
                w = fmaxf(w, stats[v * 16 + r].w);
            }
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int v = 0; v < kFewWarps; ++v) {
                const RowStats y = stats[v * 16 + r];
                const float f = lower_to(y.w, w);
                const float4 z = *reinterpret_cast<const float4*>(sums + (size_t)(v * 16 + r) * DP + d);
                l += y.l * lower_to(y.m, m);
                sum.x += f * z.x; sum.y += f * z.y; sum.z += f * z.z; sum.w += f * z.w;
            }
            if (whole) {
                const int p = p0 + r, h = head * group + p % group;
                const float f = row_factor(a, h, m, w, l);
                const size_t to = ((size_t)(sp.begin + p / group) * a.heads + h) * c.dim + d;
                const float y[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < c.dim) store_out(a, to + e, f * y[e]);
            } else {
                *reinterpret_cast<float4*>(part + (slot * 16 + r) * DP + d) = sum;
                if (d == 0) part_stats[slot * 16 + r] = {m, w, l};
            }
        }
        __syncthreads();                                                             // (the ring and the queries' room are taken again)
    }
}

// A tile that several runs share: a CTA per border between runs, and per row.  The first border inside the tile joins it.
template <int DP>
__global__ void __launch_bounds__(kFewThreads) kv8_attention_join_kernel(Kv8Cache c, Kv8Step s, Kv8Attention a, int ctas, const float* part, const RowStats* part_stats) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float tops[kFewWarps][2];
    __shared__ __align__(16) float sums[kFewWarps][DP];
    __shared__ float totals[kFewWarps];
    const int nth = blockIdx.x + 1, r = blockIdx.y, group = a.heads / c.kv_heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Place at = find_place(s, a, c.kv_heads, group, c.page_shift, ctas, nth);
    if (at.seq < 0) return;
    const Span sp = span_of(s, a, at.seq, group, c.page_shift);
    const long long item = (at.per * nth - at.base) / sp.blocks, start = at.base + item * sp.blocks;
    const int c0 = (int)(start / at.per), c1 = (int)((start + sp.blocks - 1) / at.per);
    const int head = (int)(item / sp.tiles), tile = (int)(item - (long long)head * sp.tiles), p = tile * kRowTile + r;
    if (start == at.per * nth || nth != c0 + 1 || p >= sp.n * group) return;
    const auto slot = [&](int i) { return ((size_t)2 * i + (i == c0)) * 16 + r; };
    float m = -INFINITY, w = -INFINITY;
    for (int i = c0 + threadIdx.x; i <= c1; i += kFewThreads) {
        const RowStats y = part_stats[slot(i)];
        m = fmaxf(m, y.m);
        w = fmaxf(w, y.w);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, d));
    }
    if (lane == 0) { tops[warp][0] = m; tops[warp][1] = w; }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kFewWarps; ++v) { m = fmaxf(m, tops[v][0]); w = fmaxf(w, tops[v][1]); }
    constexpr int kEach = DP / 32;
    float sum[kEach] = {}, l = 0.f;
#pragma unroll 4
    for (int i = c0 + warp; i <= c1; i += kFewWarps) {
        const RowStats y = part_stats[slot(i)];
        const float f = lower_to(y.w, w);
        l += y.l * lower_to(y.m, m);
#pragma unroll
        for (int j = 0; j < kEach; ++j) sum[j] += f * part[slot(i) * DP + lane + 32 * j];
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) sums[warp][lane + 32 * j] = sum[j];
    if (lane == 0) totals[warp] = l;
    __syncthreads();
    const int h = head * group + p % group;
    l = 0.f;
#pragma unroll
    for (int v = 0; v < kFewWarps; ++v) l += totals[v];
    const float f = row_factor(a, h, m, w, l);
    for (int d = threadIdx.x; d < c.dim; d += kFewThreads) {
        float y = 0.f;
#pragma unroll
        for (int v = 0; v < kFewWarps; ++v) y += sums[v][d];
        store_out(a, ((size_t)(sp.begin + p / group) * a.heads + h) * c.dim + d, f * y);
    }
}

inline bool wide(const Kv8Rows& x, int type, int dim) {
    const long long b = type_bytes(type);
    return (reinterpret_cast<uintptr_t>(x.x) & 15) == 0 && x.row * b % 16 == 0 && x.head * b % 16 == 0 && dim % 8 == 0;
}
inline int padded_dim(const Kv8Cache& c) { return c.dim <= 64 ? 64 : c.dim <= 128 ? 128 : 256; }
inline int terms_of(int type) { return type == kTypeF32 ? 2 : 1; }
constexpr int kFewSms = 148;
template <int DP, int TERMS> constexpr int few_ctas() { return kFewSms * Few<DP, TERMS>::kCtas; }
inline int few_ctas(int dp, int terms) {
    return dp == 64 ? (terms == 2 ? few_ctas<64, 2>() : few_ctas<64, 1>()) : dp == 128 ? (terms == 2 ? few_ctas<128, 2>() : few_ctas<128, 1>()) : (terms == 2 ? few_ctas<256, 2>() : few_ctas<256, 1>());
}

template <int DP, int FORMAT, int TERMS>
cudaError_t run_few(const Kv8Cache& c, const Kv8Step& s, const Kv8Attention& a, void* work, cudaStream_t st) {
    using F = Few<DP, TERMS>;
    constexpr int kCtas = few_ctas<DP, TERMS>();
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    e = dia::ask_smem<kv8_attention_few_kernel<DP, FORMAT, TERMS>>(dev, F::kSmem);
    if (e != cudaSuccess) return e;
    float* const part = reinterpret_cast<float*>(work);
    RowStats* const stats = reinterpret_cast<RowStats*>(part + (size_t)2 * kCtas * 16 * DP);
    kv8_attention_few_kernel<DP, FORMAT, TERMS><<<kCtas, kFewThreads, F::kSmem, st>>>(c, s, a, part, stats);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    ++dia::extra_launches();
    const int most = (int)std::min<long long>(kRowTile, (long long)s.rows * (a.heads / c.kv_heads));
    return launch_pdl(kv8_attention_join_kernel<DP>, dim3(kCtas - 1, most), dim3(kFewThreads), 0, st, c, s, a, kCtas, part, stats);
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8Cache& c, const Kv8Step& s, Kv8Rows k, Kv8Rows v, int type, cudaStream_t st) {
    // a warp per row where sequences have few of them (a decoding step's pages side by side), per page's worth where they have many
    const int chunk = s.rows > 4ll * s.sequences ? 1 << c.page_shift : 1;
    const long long tasks = ((long long)s.rows + chunk - 1) / chunk * 2 * c.kv_heads, blocks = (tasks * 32 + kAppendThreads - 1) / kAppendThreads;
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    const bool w = wide(k, type, c.dim) && wide(v, type, c.dim);
    const auto run = [&](auto kernel) { kernel<<<(unsigned)blocks, kAppendThreads, 0, st>>>(c, s, k, v, chunk); };
#define KV8_APPEND(FORMAT, TYPE) (w ? run(kv8_append_kernel<FORMAT, TYPE, true>) : run(kv8_append_kernel<FORMAT, TYPE, false>))
    if (c.format == kKvE4m3) type == kTypeF32 ? KV8_APPEND(kKvE4m3, kTypeF32) : type == kTypeBf16 ? KV8_APPEND(kKvE4m3, kTypeBf16) : KV8_APPEND(kKvE4m3, kTypeF16);
    else type == kTypeF32 ? KV8_APPEND(kKvInt8, kTypeF32) : type == kTypeBf16 ? KV8_APPEND(kKvInt8, kTypeBf16) : KV8_APPEND(kKvInt8, kTypeF16);
#undef KV8_APPEND
    return cudaGetLastError();
}

cudaError_t launch_kv8_read(const Kv8Cache& c, const Kv8Step& s, void* k, void* v, int type, cudaStream_t st) {
    const int each = s.rows >= 148 * 4 * kReadMostRows ? kReadMostRows : 8;
    const unsigned blocks = (unsigned)(((long long)s.rows + each - 1) / each);
    const bool w = c.dim % (16 / type_bytes(type)) == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
    const auto run = [&](auto kernel, auto* to) { kernel<<<blocks, kReadThreads, 0, st>>>(c, s, to, reinterpret_cast<decltype(to)>(v), each); };
#define KV8_READ(FORMAT, TYPE) (w ? run(kv8_read_kernel<FORMAT, TYPE, true>, reinterpret_cast<Element<TYPE>*>(k)) : run(kv8_read_kernel<FORMAT, TYPE, false>, reinterpret_cast<Element<TYPE>*>(k)))
    if (c.format == kKvE4m3) type == kTypeF32 ? KV8_READ(kKvE4m3, kTypeF32) : type == kTypeBf16 ? KV8_READ(kKvE4m3, kTypeBf16) : KV8_READ(kKvE4m3, kTypeF16);
    else type == kTypeF32 ? KV8_READ(kKvInt8, kTypeF32) : type == kTypeBf16 ? KV8_READ(kKvInt8, kTypeBf16) : KV8_READ(kKvInt8, kTypeF16);
#undef KV8_READ
    return cudaGetLastError();
}

namespace {
// Pairs of a sequence from which on tiles of 256 rows are the shorter way
constexpr int kFewMost = 64;
inline bool some_in_tiles(const Kv8Cache& c, const Kv8Step& s, int heads, int type) { return kv8_tiles_ok(c, type) && (long long)s.rows * (heads / c.kv_heads) > kFewMost; }
}  // namespace

size_t kv8_attention_work_bytes(const Kv8Cache& c, const Kv8Step& s, int heads, int type) {
    const int dp = padded_dim(c);
    const size_t few = (size_t)2 * few_ctas(dp, terms_of(type)) * 16 * (dp * sizeof(float) + sizeof(RowStats));
    return some_in_tiles(c, s, heads, type) ? std::max(few, kv8_tiles_work_bytes(c)) : few;
}

cudaError_t launch_kv8_attention(const Kv8Cache& c, const Kv8Step& s, Kv8Attention a, void* work, cudaStream_t st) {
    const int dp = padded_dim(c);
    const bool two = terms_of(a.type) == 2;
    a.few_most = 0x7fffffff;
    if (some_in_tiles(c, s, a.heads, a.type)) {
        const bool alone = s.sequences == 1;                  // (then whatever its rows are)
        a.few_most = alone ? 0 : kFewMost;
        const cudaError_t e = launch_kv8_tiles(c, s, a, alone, work, st);
        if (e != cudaSuccess || alone) return e;
        ++dia::extra_launches();
    }
#define KV8_FEW(DP, FORMAT) (two ? run_few<DP, FORMAT, 2>(c, s, a, work, st) : run_few<DP, FORMAT, 1>(c, s, a, work, st))
    if (c.format == kKvE4m3) return dp == 64 ? KV8_FEW(64, kKvE4m3) : dp == 128 ? KV8_FEW(128, kKvE4m3) : KV8_FEW(256, kKvE4m3);
    return dp == 64 ? KV8_FEW(64, kKvInt8) : dp == 128 ? KV8_FEW(128, kKvInt8) : KV8_FEW(256, kKvInt8);
#undef KV8_FEW
}

}  // namespace lm
