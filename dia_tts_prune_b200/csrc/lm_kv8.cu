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
    // the largest magnitude so far, as bits (two of the 16-bit types side by side), and as those of an fp32 number
    __device__ __forceinline__ void look(uint32_t& most) const {
        const uint32_t* const u = &w[0].x;
#pragma unroll
        for (int i = 0; i < (TYPE == kTypeF32 ? 8 : 4); ++i) most = TYPE == kTypeF32 ? max(most, u[i] & 0x7fffffffu) : __vmaxu2(most, u[i] & 0x7fff7fffu);
    }
    static __device__ __forceinline__ uint32_t looked(uint32_t most) {
        const uint32_t half = max(most & 0xffffu, most >> 16);
        return TYPE == kTypeF32 ? most : TYPE == kTypeBf16 ? half << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)half)));
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
// Bound: a chain of loads (the row's sequence, its rows and the page's number, the page's scale) for every warp; rows are asked for before the page is known.
constexpr int kAppendThreads = 128, kKept = 8, kSearchMost = 1024;

// The sequence of a row, by a warp: how many begin at or before it (one look for 32 sequences; where there are very many, by halves)
__device__ __forceinline__ int sequence_by_warp(const Kv8Step& s, int row) {
    if (!s.first || s.sequences > kSearchMost) return s.sequence_of(row);
    int n = 0;
    for (int i = 0; i <= s.sequences; i += 32) {
        const int at = i + (threadIdx.x & 31);
        n += __popc(__ballot_sync(0xffffffffu, at <= s.sequences && s.first[at] <= row));
    }
    return n > 0 && n <= s.sequences ? n - 1 : -1;
}

template <int FORMAT, int TYPE, bool WIDE>
__global__ void __launch_bounds__(kAppendThreads, 4) kv8_append_kernel(Kv8Cache c, Kv8Step s, Kv8Rows k, Kv8Rows v, int chunk) {
    const int lane = threadIdx.x & 31;
    const long long task = ((long long)blockIdx.x * kAppendThreads + threadIdx.x) >> 5;
    const int sides = 2 * c.kv_heads, side = (int)(task % sides) & 1, head = (int)(task % sides) >> 1;
    const long long row0 = task / sides * chunk;
    if (row0 >= s.rows) return;
    const Kv8Rows in = side ? v : k;
    uint8_t* const codes = side ? c.values : c.keys;
    float* const scales = side ? c.value_scales : c.key_scales;
    const Element<TYPE>* const x = reinterpret_cast<const Element<TYPE>*>(in.x) + head * in.head;
    const int groups = (c.dim + 7) >> 3, page_size = 1 << c.page_shift, last = (int)min(row0 + chunk, (long long)s.rows);
    // a lane's groups: group lane of the rows in turn, the next one 32 further on
    struct At {
        int r, g;
    };
    const int step_r = 32 / groups, step_g = 32 - step_r * groups;
    const At first{lane / groups, lane - lane / groups * groups};
    const auto next = [&](At& at) {
        at.r += step_r;
        at.g += step_g;
        if (at.g >= groups) {
            at.g -= groups;
            ++at.r;
        }
    };
    int row = (int)row0, seq = sequence_by_warp(s, row);
    while (row < last) {
        const int begin = s.begin(max(seq, 0)), end = s.end(max(seq, 0));
        // no row of a sequence: on to the next one that is.  (Where `first` decreases, the look-up may name a sequence that does not have the row.  Past this a turn goes at least one row on.)
        if (seq < 0 || row < begin || row >= end) {
            if (++row < last) seq = sequence_by_warp(s, row);
            continue;
        }
        const int past = s.past[seq];
        const long long pos = (long long)past + (row - begin);
        const int place = (int)(pos & (page_size - 1));
        const int ends = min(end, row + page_size - place);    // of the rows that go into this page
        if (past >= 0 && (row == begin || place == 0)) {
            const int n = ends - row;
            Eight<TYPE, WIDE> kept[kKept];
            const auto fetch = [&](Eight<TYPE, WIDE>& e, const At& at) {
                if (at.r < n) e.fetch(x + (row + at.r) * in.row + 8 * at.g, c.dim - 8 * at.g);
                else e = {};
            };
            At beyond = first;
#pragma unroll
            for (int j = 0; j < kKept; ++j) {
                fetch(kept[j], beyond);
                next(beyond);
            }
            const int page = s.page(seq, pos >> c.page_shift, c.pages);
            if (page >= 0) {
                const size_t page_head = (size_t)page * c.kv_heads + head;
                float* const scale = scales + page_head;
                uint8_t* const to = codes + (page_head << c.page_shift) * c.stride;
                const uint32_t old = place ? __float_as_uint(*scale) & 0x7fffffffu : 0u;
                uint32_t most = 0;
#pragma unroll
                for (int j = 0; j < kKept; ++j) kept[j].look(most);
#pragma unroll 1
                for (At i = beyond; i.r < n; next(i)) {
                    Eight<TYPE, WIDE> e;
                    fetch(e, i);
                    e.look(most);
                }
                most = __reduce_max_sync(0xffffffffu, Eight<TYPE, WIDE>::looked(most));
                const bool bad = most >= 0x7f800000u || old >= 0x7f800000u;
                int e = needed<FORMAT>(most);
                if (place && !bad) {
                    const int before = (int)(old >> 23) - 127;
                    if (before >= e) {
                        e = before;
                    } else {
                        const float f = power(before - e);
#pragma unroll 1
                        for (int i = lane; i < place * (c.stride >> 4); i += 32) {
                            uint4* const p = reinterpret_cast<uint4*>(to) + i;
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
                const auto write = [&](const Eight<TYPE, WIDE>& g8, const At& at) {
                    if (at.r >= n) return;
                    float t[8];
                    g8.numbers(t);
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[j] = bad ? 0.f : t[j] * f;
                    const uint2 w = make_uint2(encode4<FORMAT>(t[0], t[1], t[2], t[3]), encode4<FORMAT>(t[4], t[5], t[6], t[7]));
                    uint2* const p = reinterpret_cast<uint2*>(to + (size_t)(place + at.r) * c.stride) + at.g;
                    p[0] = w;
                    if (at.g == groups - 1 && (groups & 1)) p[1] = make_uint2(0u, 0u);     // (up to the row's 16 bytes)
                };
                At at = first;
#pragma unroll
                for (int j = 0; j < kKept; ++j) {
                    write(kept[j], at);
                    next(at);
                }
#pragma unroll 1
                for (At i = beyond; i.r < n; next(i)) {
                    Eight<TYPE, WIDE> g8;
                    fetch(g8, i);
                    write(g8, i);
                }
            }
        }
        row = ends;
        if (row == end && row < last) seq = sequence_by_warp(s, row);
    }
}

// ---- numbers out of pages ------------------------------------------------------------------------------------------------------------------
// A CTA takes kReadMostRows rows (8 where there are few): where each of them lies is looked up once.  A thread has 16 bytes of what goes out, the same head and channels of row
// after row, four rows on their way at a time.
constexpr int kReadThreads = 256, kReadMostRows = 32, kReadAhead = 4;
template <int FORMAT, int TYPE, bool WIDE>
__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(Kv8Cache c, Kv8Step s, Element<TYPE>* k, Element<TYPE>* v, int rows_each) {
    __shared__ int firsts[kSearchMost + 1];
    __shared__ long long where[kReadMostRows];                // the row's page (from the 32nd bit on) and place in it; -1: not there
    const int row0 = blockIdx.x * rows_each, n = min(rows_each, s.rows - row0);
    const bool near = s.first && s.sequences <= kSearchMost;
    if (near) {
        for (int i = threadIdx.x; i <= s.sequences; i += kReadThreads) firsts[i] = s.first[i];
        __syncthreads();
    }
    if (threadIdx.x < n) {
        Kv8Step of = s;
        if (near) of.first = firsts;
        const int row = row0 + threadIdx.x, seq = of.sequence_of(row);
        long long at = -1;
        if (seq >= 0) {
            const int past = s.past[seq];
            const long long pos = (long long)past + (row - of.begin(seq));
            const int page = past >= 0 ? s.page(seq, pos >> c.page_shift, c.pages) : -1;
            if (page >= 0) at = (long long)page << 32 | (pos & ((1 << c.page_shift) - 1));
        }
        where[threadIdx.x] = at;
    }
    __syncthreads();
    constexpr int kEach = 16 / sizeof(Element<TYPE>), kCodeWords = kEach / 4;
    const int parts = (c.dim + kEach - 1) / kEach, per_row = 2 * c.kv_heads * parts, beside = max(1, kReadThreads / per_row);
    for (int j = per_row <= kReadThreads ? threadIdx.x % per_row : threadIdx.x; j < per_row; j += per_row <= kReadThreads ? per_row : kReadThreads) {
        const int side = j / (c.kv_heads * parts), hp = j - side * c.kv_heads * parts, head = hp / parts, part = hp - head * parts, r0 = per_row <= kReadThreads ? threadIdx.x / per_row : 0;
        if (r0 >= beside) break;
        const uint8_t* const codes = (side ? c.values : c.keys) + part * kEach;
        const float* const scales = side ? c.value_scales : c.key_scales;
        Element<TYPE>* const to = (side ? v : k) + ((size_t)row0 * c.kv_heads + head) * c.dim + part * kEach;
        for (int r = r0; r < n; r += beside * kReadAhead) {
            uint32_t w[kReadAhead][kCodeWords];
            float scale[kReadAhead];
#pragma unroll
            for (int i = 0; i < kReadAhead; ++i) {
                const long long at = r + i * beside < n ? where[r + i * beside] : -1;
                scale[i] = 0.f;
#pragma unroll
                for (int e = 0; e < kCodeWords; ++e) w[i][e] = 0;
                if (at < 0) continue;
                const size_t page_head = (size_t)(at >> 32) * c.kv_heads + head;
                const uint8_t* const p = codes + ((page_head << c.page_shift) + (uint32_t)at) * c.stride;
                if constexpr (kCodeWords == 2) {
                    const uint2 u = *reinterpret_cast<const uint2*>(p);
                    w[i][0] = u.x;
                    w[i][kCodeWords - 1] = u.y;
                } else {
                    w[i][0] = *reinterpret_cast<const uint32_t*>(p);
                }
                scale[i] = scales[page_head];
            }
#pragma unroll
            for (int i = 0; i < kReadAhead; ++i) {
                if (r + i * beside >= n) break;
                Element<TYPE> out[kEach];
#pragma unroll
                for (int e = 0; e < kEach; e += 4) {
                    const float4 t = values4<FORMAT>(w[i][e / 4], scale[i]);      // (of a row that is not there: zeros times zero)
                    out[e] = narrow<Element<TYPE>>(t.x);
                    out[e + 1] = narrow<Element<TYPE>>(t.y);
                    out[e + 2] = narrow<Element<TYPE>>(t.z);
                    out[e + 3] = narrow<Element<TYPE>>(t.w);
                }
                Element<TYPE>* const p = to + (size_t)(r + i * beside) * c.kv_heads * c.dim;
                if constexpr (WIDE) {
                    uint4 u;
                    memcpy(&u, out, 16);
                    *reinterpret_cast<uint4*>(p) = u;
                } else {
#pragma unroll
                    for (int e = 0; e < kEach; ++e)
                        if (part * kEach + e < c.dim) p[e] = out[e];
                }
            }
        }
    }
}

// ---- attention of few rows -----------------------------------------------------------------------------------------------------------------
// x = scale log2(e) q . key in powers of two, p = 2^(x - max x), o = sum p value / (sum p + 2^(sink log2(e) - max x)).
//
// What bounds it is the cache's bytes.  The rows of a tile (8, or 16) are (token, query head) pairs that share a key head, so a token's codes are read once for the group; tiles of
// a sequence lie next to one another in the order of the work.  Work is counted in blocks of 16 tokens over all sequences, heads and tiles and dealt to the CTAs in
// equal runs, so that one long sequence fills the GPU and lengths need not be alike; runs that share a tile leave (max, sum, output), and the last one to come joins them, always in
// the same order (a second kernel for that took 6 us after one request's 1024 tokens, 11 after 131072, 26 after 64 requests).  Few short tiles go to a cluster each.
// Measured: 64 requests of up to 24576 tokens 226 us (5.9 TB/s of the 6.5 that a copy reaches); one behind 131071 28 us, of which the cache's bytes are 10, the first loads 4 and the two
// joins 9; one of 1025 9.8 us: a launch and a chain of looks at the sequence, its page, its scale, its codes.
//
// A warp keeps its own ring of blocks in shared memory, filled by asynchronous copies that swizzle 16-byte pieces (rows lie 128 bytes apart, which would be the same banks), and
// multiplies on the tensor cores (mma.sync, 16 x 8 x 16: a block's 16 tokens, or 16 channels of their values, by eight rows: what a group has, and nothing is waited for across warps).
// A thread's four codes of a 32-bit word are four channels of a key, whichever: queries are laid out to match; a thread's word of a value is transposed against those of three other
// tokens by byte permutations, and the weights by movmatrix.
//
// Codes are exact in fp16.  A row of queries is scaled by a power of two to below 2^14 and taken as one fp16 term (bf16 and fp16 rows: exact but for channels 2^-27 below the
// row's largest), or two (fp32: 22 bits).  Weights: the page's value scale is part of the exponent, 2^(x + e - W) 2^14, W = max (x + e), so that the largest contribution, not the largest
// weight, is what fp16's 11 bits count from (11 are what results in fp16 have themselves, and three more than bf16's; the largest weight is a power of two and loses nothing, which is what rows
// with one large weight live by: with W a whole number results in fp16 were off by 2.6e-4, not 2.1e-4).  fp32 rows have two terms, 22 bits, and whole references, max (floor(x) + e): what lies
// between two of them, or between them and a page's exponent, is then exact (with fractions of scores in them outputs were off by up to 8e-7 of the sum of weighted magnitudes, 3e-6 where values
// are 2^100; so they are by 3e-7; a prompt of 4096 takes 1 % more, single tokens no more).  Sums, maxima and outputs are fp32, and the denominator is summed from fp32 weights without the scale.
// A tensor-core sum is cut off at every step: fp32 rows add the second terms' sums and every block's outputs to theirs by fp32 additions.
constexpr int kMetaBlocks = 256, kMostPeers = 8;               // CTAs of a cluster

template <int DP, int TERMS, int NT>
struct Few {
    // Two CTAs on an SM where registers allow: one computes while the other is between two tiles
    static constexpr int kPerSm = TERMS == 2 || DP == 256 ? 1 : 2, kCtas = 148 * kPerSm;
    static constexpr int kWarps = kPerSm == 1 ? 8 : NT == 1 ? 8 : 6, kThreads = 32 * kWarps, kRows = 8 * NT;
    static constexpr int kSide = kKvBlock * DP;               // bytes of a block's keys, or values
    static constexpr int kStages = 192 * 1024 / kPerSm / (kWarps * 2 * kSide) > 8 ? 8 : 192 * 1024 / kPerSm / (kWarps * 2 * kSide);
    static constexpr int kRing = kWarps * kStages * 2 * kSide;
    static constexpr int kQ = TERMS * NT * (DP / 16) * 32 * 8;                    // fragments of the queries
    static constexpr int kSums = kWarps * kRows * DP * 4 + kCtas * kRows * 4;     // and the weights of runs that share a tile (where the ring lies)
    static constexpr int kSmem = (kRing > kSums ? kRing : kSums) + kQ + kMetaBlocks * 16 + kRows * 4 + kWarps * kRows * 12 + 128;
};
constexpr int kMostCtas = 2 * 148, kJoin = 12;                // (runs that are joined in one go: about the root of how many there may be)

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {          // of 8 x 8 fp16, a row in four lanes
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// x, y as fp16, and what that leaves
__device__ __forceinline__ uint32_t rest_of(float x, float y, uint32_t h) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return pack_half(x - f.x, y - f.y);
}

// where 16-byte piece `c` of row `r` of a block lies
template <int DP>
__device__ __forceinline__ int piece_at(int r, int c) {
    if constexpr (DP == 64) return (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) << 4);
    else return r * DP + ((c ^ ((r & 2) | (((r << 2) ^ r) & 4))) << 4);
}

// Blocks of 16 tokens that a sequence's rows look at, and its share of the work.  run: blocks that a CTA takes of one tile, which then goes in equal parts of at most so many, a unit
// each; 0: units are blocks, which CTAs take in a row across tiles, and a tile costs kTileCost more: its rows are laid out and its warps' sums met, which takes 3 us (64 requests of up to 24576
// tokens: 252 us without, 242 with 16, 228 with 32, 226 with 48, 231 with 96; 256 requests of up to 1000: 178, 115, 101, 100, 113)
constexpr int kWholeRun = 0x7fffffff, kTileCost = 48;
struct Span {
    int begin, n, past, low, blocks, tiles, share;            // low: the first block; share: units of work in a tile
    __device__ __forceinline__ long long units(int kv_heads) const { return (long long)kv_heads * tiles * share; }
};
template <int ROWS>
__device__ __forceinline__ Span span_of(const Kv8Step& s, const Kv8Attention& a, int i, int group, int page_shift, int run) {
    Span p;
    p.begin = s.begin(i);
    p.n = max(s.end(i) - p.begin, 0);
    p.past = s.past[i];
    p.low = a.window > 0 ? (int)(max(0ll, (long long)p.past + 1 - a.window) / kKvBlock) : 0;
    const long long end = min((long long)max(p.past, 0) + p.n, (long long)s.max_pages << page_shift);
    p.blocks = max(1, (int)((end + kKvBlock - 1) / kKvBlock) - p.low);
    p.tiles = (long long)p.n * group > a.few_most ? 0 : (p.n * group + ROWS - 1) / ROWS;
    p.share = run == 0 ? p.blocks + kTileCost : (int)(((long long)p.blocks + run - 1) / run);
    return p;
}

// The sequence that holds the unit `per * nth` of all, where per = what a CTA takes (one warp; seq < 0: there is none).  Where there are two CTAs for a tile, no CTA has parts of two:
// parts of `run` blocks are as many as the CTAs, and two blocks for every warp at least (eight requests of 4096 tokens: 23 us as units in a row, 21 so; five of at most 1024: 31 and 17,
// beside prompt portions 52 with one block for a warp and 42 with two).
struct Place {
    int seq, run;
    long long base, per, total;
};
template <int ROWS>
__device__ __forceinline__ Place find_place(const Kv8Step& s, const Kv8Attention& a, int kv_heads, int group, int page_shift, int ctas, int warps, int nth) {
    const int lane = threadIdx.x & 31, each = (s.sequences + 31) / 32, i0 = lane * each, i1 = min(i0 + each, s.sequences);
    const Span first = span_of<ROWS>(s, a, min(i0, s.sequences - 1), group, page_shift, kWholeRun);       // (a lane's only one, mostly)
    const auto at = [&](int i, int run) {
        if (i != i0) return span_of<ROWS>(s, a, i, group, page_shift, run);
        Span p = first;
        p.share = run == 0 ? p.blocks + kTileCost : (int)(((long long)p.blocks + run - 1) / run);
        return p;
    };
    Place place{-1, kWholeRun, 0, 1, 0};
    if (!a.whole) {
        long long blocks = 0, tiles = 0;
        for (int i = i0; i < i1; ++i) {
            const Span p = at(i, kWholeRun);
            tiles += p.units(kv_heads);
            blocks += p.units(kv_heads) * p.blocks;
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            tiles += __shfl_xor_sync(0xffffffffu, tiles, d);
            blocks += __shfl_xor_sync(0xffffffffu, blocks, d);
        }
        place.run = 2 * tiles <= ctas ? max((int)((blocks + ctas - tiles - 1) / (ctas - tiles)), 2 * warps) : 0;
    }
    long long mine = 0;
    for (int i = i0; i < i1; ++i) mine += at(i, place.run).units(kv_heads);
    long long upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
    }
    place.total = __shfl_sync(0xffffffffu, upto, 31);
    place.per = max((place.total + ctas - 1) / ctas, place.run ? 1ll : (long long)warps);
    place.base = upto - mine;
    const long long unit = place.per * nth;
    const bool here = unit >= place.base && unit < upto;
    if (here) {
        for (place.seq = i0;; ++place.seq) {
            const long long u = at(place.seq, place.run).units(kv_heads);
            if (unit < place.base + u) break;
            place.base += u;
        }
    }
    const unsigned who = __ballot_sync(0xffffffffu, here);
    const int from = who ? __ffs(who) - 1 : 0;
    place.seq = __shfl_sync(0xffffffffu, place.seq, from);
    place.base = __shfl_sync(0xffffffffu, place.base, from);
    return place;
}

// Clusters of CTAs (of one, where a launch has none)
__device__ __forceinline__ unsigned cluster_size() { unsigned v; asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(v)); return v; }
__device__ __forceinline__ unsigned cluster_rank() { unsigned v; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(v)); return v; }
__device__ __forceinline__ unsigned cluster_index() { unsigned v; asm("mov.u32 %0, %%clusterid.x;" : "=r"(v)); return v; }
__device__ __forceinline__ void cluster_met() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t shared_of(const void* p, unsigned rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float load_of(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float4 load4_of(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

template <int DP, int FORMAT, int TERMS, int NT>
__global__ void __launch_bounds__(Few<DP, TERMS, NT>::kThreads, Few<DP, TERMS, NT>::kPerSm) kv8_attention_few_kernel(Kv8Cache c, Kv8Step s, Kv8Attention a, int beside, float* part, RowStats* part_stats, unsigned* arrived) {
    using F = Few<DP, TERMS, NT>;
    constexpr int kSteps = DP / 16, kHalves = DP == 256 ? 2 : 1, kWords = DP == 64 ? 2 : 4, kCols = kHalves * kWords * 2, kWarps = F::kWarps, kRows = F::kRows;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const ring = smem + (threadIdx.x >> 5) * (F::kStages * 2 * F::kSide);
    float* const sums = reinterpret_cast<float*>(smem);                            // [warps][rows][DP], when the ring is empty
    uint2* const q_frags = reinterpret_cast<uint2*>(smem + (F::kRing > F::kSums ? F::kRing : F::kSums));
    long long* const meta_at = reinterpret_cast<long long*>(q_frags + F::kQ / 8);  // where a block's codes lie; -1: it is not there
    float2* const meta = reinterpret_cast<float2*>(meta_at + kMetaBlocks);         // (key scale, exponent of the values)
    float* const row_scale = reinterpret_cast<float*>(meta + kMetaBlocks);         // [rows] of the queries, with the scores' scale
    RowStats* const stats = reinterpret_cast<RowStats*>(row_scale + kRows);        // [warps][rows]
    __shared__ Place place;
    __shared__ int last;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, group = a.heads / c.kv_heads;
    const int peers = (int)cluster_size(), rank = (int)cluster_rank();               // CTAs that have a part each of the same tiles
    // a lane's pieces of 16 bytes: row lane / (DP / 16) and so on, where they go, and whether rows have them (zeros come in their place)
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring), swizzled = piece_at<DP>(lane / (DP / 16), lane % (DP / 16));
    const int lane_bytes = lane % (DP / 16) * 16 < c.stride ? 16 : 0, lane_off = lane / (DP / 16) * c.stride + (lane_bytes ? lane % (DP / 16) * 16 : 0);
    if (warp == 0) {
        const Place found = find_place<kRows>(s, a, c.kv_heads, group, c.page_shift, (int)gridDim.x / peers, kWarps, (int)cluster_index());
        if (lane == 0) place = found;
    }
    zero_rows_of_none(s, a, c.dim, (long long)blockIdx.x * F::kThreads + threadIdx.x, (long long)gridDim.x * F::kThreads);
    __syncthreads();
    Place at = place;
    long long unit = at.seq < 0 ? at.total : at.per * cluster_index();
    const long long unit_end = min(unit + at.per, at.total);
    Span sp = span_of<kRows>(s, a, max(at.seq, 0), group, c.page_shift, at.run);

    while (unit < unit_end) {
        while (unit >= at.base + sp.units(c.kv_heads)) {                             // (sequences without rows have no units)
            at.base += sp.units(c.kv_heads);
            sp = span_of<kRows>(s, a, ++at.seq, group, c.page_shift, at.run);
        }
        const long long item = (unit - at.base) / sp.share;
        const int u0 = (int)(unit - at.base - item * sp.share), taken = at.run ? 1 : (int)min((long long)sp.share - u0, unit_end - unit);
        // (a cluster's CTAs take a tile that nobody shares together)
        const long long parts = (long long)sp.share * peers, nth = (long long)u0 * peers + rank;
        const int b0 = at.run ? (int)(nth * sp.blocks / parts) : u0, b1 = at.run ? (int)((nth + 1) * sp.blocks / parts) : min(u0 + taken, sp.blocks), count = b1 - b0;
        const int head = (int)(item / sp.tiles), tile = (int)(item - (long long)head * sp.tiles);
        const int p0 = tile * kRows, rows = min(kRows, sp.n * group - p0);
        unit += taken;
        if (count <= 0 && !at.run) continue;                                                    // (what a tile costs besides)
        // positions of the tile's rows, first and last
        const auto position = [&](int r) { return (long long)sp.past + (p0 + min(r, rows - 1)) / group; };
        const long long back = a.window > 0 ? a.window - 1 : (1ll << 40);
        const long long pos_a = position(0), pos_b = position(kRows), seen_from = max(0ll, pos_a - back), clear_from = max(0ll, pos_b - back);
        const auto token = [&](int i) { return (long long)(sp.low + b0 + i) * kKvBlock; };      // of block i of the run
        const auto look_up = [&](int m_at, int m_n) {                                // pages and scales of the run's blocks from m_at on
            for (int i = threadIdx.x; i < m_n; i += F::kThreads) {
                const long long tok = token(m_at + i);
                int page = -1;
                if (sp.past >= 0 && tok <= pos_b && tok + kKvBlock > seen_from) page = s.page(at.seq, tok >> c.page_shift, c.pages);
                if (page >= 0) {
                    const size_t ph = (size_t)page * c.kv_heads + head;
                    const uint32_t vs = __float_as_uint(c.value_scales[ph]);
                    meta_at[i] = (long long)(((ph << c.page_shift) + (size_t)(tok & ((1 << c.page_shift) - 1))) * c.stride);
                    meta[i] = make_float2(c.key_scales[ph], vs >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : (float)((int)(vs >> 23) - 127));
                } else {
                    meta_at[i] = -1;
                }
            }
        };
        const auto issue = [&](int m_n, int i, int stage) {                          // block i of the list into a slot of the ring
            const long long from = i < m_n ? meta_at[i] : -1;
            if (from >= 0) {
                const uint32_t to = ring_at + stage * 2 * F::kSide;
#pragma unroll
                for (int j = 0; j < DP / 32; ++j) {
                    // (a lane's pieces lie 32 on from one to the next: the swizzle differs by what it does to those bits of the row)
                    const uint32_t d = to + 512 * j + (DP == 64 ? swizzled : DP == 128 ? swizzled ^ ((j & 1) << 6) : swizzled ^ ((j & 1) << 5) ^ ((j & 2) << 5));
                    const size_t off = (size_t)from + (uint32_t)(lane_off + j * (512 / DP) * c.stride);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(c.keys + off), "r"(lane_bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + F::kSide), "l"(c.values + off), "r"(lane_bytes) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        look_up(0, min(kMetaBlocks, count));
        // queries: a warp scales some rows and leaves them as the products' fragments
        for (int r = warp; r < kRows; r += kWarps) {
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
            const float f = __uint_as_float((267u - e) << 23), way_back = __uint_as_float((e - 13u) << 23);      // 2^(140 - e): to below 2^14, and the way back
            if (lane == 0) row_scale[r] = e == 255u ? __uint_as_float(0x7fc00000u) : way_back * (a.scale * kLog2e);
#pragma unroll
            for (int j = 0; j < DP / 32; ++j) {
                const int d = lane + 32 * j, chunk = d >> 4, step = (chunk >> 2) * 4 + ((d & 15) >> 2), x = d & 3;
                __half* const to = reinterpret_cast<__half*>(q_frags) + ((((r >> 3) * kSteps + step) * 32 + (r & 7) * 4 + (chunk & 3)) * 2 + (x >> 1)) * 2 + (x & 1);
                const float y = e == 255u ? 0.f : v[j] * f;
                const __half hi = __float2half_rn(y);
                to[0] = hi;
                if constexpr (TERMS == 2) to[NT * kSteps * 32 * 4] = __float2half_rn(y - __half2float(hi));
            }
        }
        __syncthreads();
        // the thread's rows of each tile of eight: 2 t and 2 t + 1
        float scale_of[NT][2], m[NT][2], w[NT][2], l[NT][2], o[NT][kCols][4];
        constexpr bool kInRegs = DP * TERMS * NT <= 256;
        uint2 qf[kInRegs ? TERMS * NT * kSteps : 1];
        if constexpr (kInRegs) {
#pragma unroll
            for (int j = 0; j < TERMS * NT * kSteps; ++j) qf[j] = q_frags[j * 32 + lane];
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                scale_of[n][e] = row_scale[8 * n + 2 * t + e];
                m[n][e] = w[n][e] = -INFINITY;
                l[n][e] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < kCols; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][j][e] = 0.f;
        }

        for (int m_at = 0; m_at < count; m_at += kMetaBlocks) {
            const int m_n = min(kMetaBlocks, count - m_at);
            if (m_at) {
                __syncthreads();                                                     // (the last ones have been read)
                look_up(m_at, m_n);
                __syncthreads();
            }
#pragma unroll 1
            for (int j = 0; j < F::kStages - 1; ++j) issue(m_n, warp + kWarps * j, j);
            int stage = 0;
#pragma unroll 1
            for (int i = warp; i < m_n; i += kWarps) {
                asm volatile("cp.async.wait_group %0;" ::"n"(F::kStages - 2) : "memory");
                __syncwarp();                                                        // the block is there for every lane, and the slot in front has been read by all
                issue(m_n, i + kWarps * (F::kStages - 1), stage == 0 ? F::kStages - 1 : stage - 1);
                const uint8_t* const keys = ring + stage * 2 * F::kSide;
                const uint8_t* const values = keys + F::kSide;
                stage = stage + 1 == F::kStages ? 0 : stage + 1;
                if (meta_at[i] < 0) continue;

                // scores: token g of row 2 t and of row 2 t + 1, token g + 8 of either
                float x[NT][4], rest[TERMS == 2 ? NT : 1][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[n][e] = rest[TERMS == 2 ? n : 0][e] = 0.f;
#pragma unroll
                for (int h = 0; h < DP / 64; ++h) {
                    const uint4 u4 = *reinterpret_cast<const uint4*>(keys + piece_at<DP>(g, t + 4 * h)), v4 = *reinterpret_cast<const uint4*>(keys + piece_at<DP>(8 + g, t + 4 * h));
                    const uint32_t u[4] = {u4.x, u4.y, u4.z, u4.w}, v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t a0, a1, a2, a3;
                        decode4<FORMAT>(u[j], a0, a2);
                        decode4<FORMAT>(v[j], a1, a3);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const int f = n * kSteps + 4 * h + j;
                            mma16816(x[n], a0, a1, a2, a3, kInRegs ? qf[kInRegs ? f : 0] : q_frags[f * 32 + lane]);
                            if constexpr (TERMS == 2) mma16816(rest[n], a0, a1, a2, a3, kInRegs ? qf[kInRegs ? NT * kSteps + f : 0] : q_frags[(NT * kSteps + f) * 32 + lane]);
                        }
                    }
                }
                const float ks = meta[i].x, ev = meta[i].y;
                const long long tok = token(m_at + i);
                const bool clear = tok + kKvBlock - 1 <= pos_a && tok >= clear_from;   // every row sees all of the block
                uint2 hi[NT], lo[TERMS == 2 ? NT : 1];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint32_t hidden = 0;
                    float top[2];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (TERMS == 2) x[n][e] += rest[n][e];
                        x[n][e] *= scale_of[n][e & 1] * ks;
                    }
                    if (!clear) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const long long key = tok + g + 8 * (e >> 1), pos = position(8 * n + 2 * t + (e & 1));
                            if (key > pos || key < pos - back) {
                                x[n][e] = -INFINITY;
                                hidden |= 1u << e;
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        top[e] = fmaxf(x[n][e], x[n][e + 2]);
                        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 4));
                        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 8));
                        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 16));
                    }
                    // (of two terms: whole references, so that what they differ by is exact, whatever the pages' exponents are.  Of one: the largest weight itself is 2^14, which fp16 has as it is)
                    if constexpr (TERMS == 2) {
                        top[0] = floorf(top[0]);
                        top[1] = floorf(top[1]);
                    }
                    const float m0 = fmaxf(m[n][0], top[0]), m1 = fmaxf(m[n][1], top[1]), w0 = fmaxf(w[n][0], top[0] + ev), w1 = fmaxf(w[n][1], top[1] + ev);
                    if (__any_sync(0xffffffffu, m0 > m[n][0] || m1 > m[n][1] || w0 > w[n][0] || w1 > w[n][1])) {
                        const float c0 = lower_to(w[n][0], w0), c1 = lower_to(w[n][1], w1);
                        l[n][0] *= lower_to(m[n][0], m0);
                        l[n][1] *= lower_to(m[n][1], m1);
#pragma unroll
                        for (int j = 0; j < kCols; ++j) { o[n][j][0] *= c0; o[n][j][1] *= c1; o[n][j][2] *= c0; o[n][j][3] *= c1; }
                        m[n][0] = m0; m[n][1] = m1; w[n][0] = w0; w[n][1] = w1;
                    }
                    float p[4];
                    if constexpr (TERMS == 2) {
                        // counted from the block's own largest, which the sum and the products take to their references
                        float to_l[2], to_w[2], from[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const bool none = top[e] == -INFINITY;                   // (nothing of the block is seen)
                            from[e] = none ? 0.f : top[e];
                            to_l[e] = none ? 0.f : exp2_fast(top[e] - m[n][e]);
                            to_w[e] = none ? 0.f : exp2_fast(top[e] + ev - w[n][e] + kWeightBits);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float y = exp2_fast(x[n][e] - from[e & 1]);
                            l[n][e & 1] = fmaf(y, to_l[e & 1], l[n][e & 1]);
                            p[e] = y * to_w[e & 1];
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            // (rows that have seen nothing yet: any reference will do)
                            const float r = m[n][e & 1] == -INFINITY ? 0.f : m[n][e & 1], q = (w[n][e & 1] == -INFINITY ? 0.f : w[n][e & 1]) - ev - kWeightBits;
                            l[n][e & 1] += exp2_fast(x[n][e] - r);
                            p[e] = exp2_fast(x[n][e] - q);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!clear && (hidden >> e & 1)) p[e] = 0.f;                  // (whatever the page's scales are)
                    const uint32_t h0 = pack_half(p[0], p[1]), h1 = pack_half(p[2], p[3]);
                    hi[n] = make_uint2(transposed(h0), transposed(h1));
                    if constexpr (TERMS == 2) lo[n] = make_uint2(transposed(rest_of(p[0], p[1], h0)), transposed(rest_of(p[2], p[3], h1)));
                }
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    uint32_t v[4][4];                                                // [token 2 t, 2 t + 1, 2 t + 8, 2 t + 9][word]
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 2 * t + (e & 1) + 8 * (e >> 1);
                        if constexpr (DP == 64) {
                            const uint2 v2 = *reinterpret_cast<const uint2*>(values + piece_at<DP>(r, g >> 1) + 8 * (g & 1));
                            v[e][0] = v2.x; v[e][1] = v2.y;
                        } else {
                            const uint4 v4 = *reinterpret_cast<const uint4*>(values + piece_at<DP>(r, 8 * h + g));
                            v[e][0] = v4.x; v[e][1] = v4.y; v[e][2] = v4.z; v[e][3] = v4.w;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < kWords; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {                                // channels 2 e and 2 e + 1 of the word
                            uint32_t a0, a1, a2, a3;
                            decode4<FORMAT>(__byte_perm(v[0][j], v[1][j], e ? 0x7362 : 0x5140), a0, a1);
                            decode4<FORMAT>(__byte_perm(v[2][j], v[3][j], e ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float (&to)[4] = o[n][(h * kWords + j) * 2 + e];
                                if constexpr (TERMS == 2) {
                                    float y[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma16816(y, a0, a1, a2, a3, lo[n]);
                                    mma16816(y, a0, a1, a2, a3, hi[n]);
#pragma unroll
                                    for (int z = 0; z < 4; ++z) to[z] += y[z];
                                } else {
                                    mma16816(to, a0, a1, a2, a3, hi[n]);
                                }
                            }
                        }
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }

        // the warps' sums meet in shared memory
        __syncthreads();                                                             // every warp is done with its ring
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * n + 2 * t + e;
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
                if (g == 0) stats[warp * kRows + r] = {m[n][e], w[n][e], l[n][e]};
                if (r >= rows) continue;
                // products (h, j) of this thread are channels 128 h + 16 g + 2 j and the next one (of 64 channels: 8 g + 2 j)
                constexpr int kRun = DP == 64 ? 8 : 16;
#pragma unroll
                for (int h = 0; h < kHalves; ++h)
#pragma unroll
                    for (int j = 0; j < kRun; j += 4)
                        *reinterpret_cast<float4*>(sums + (size_t)(warp * kRows + r) * DP + 128 * h + kRun * g + j) =
                            make_float4(o[n][h * 8 + j / 2][e], o[n][h * 8 + j / 2][e + 2], o[n][h * 8 + j / 2 + 1][e], o[n][h * 8 + j / 2 + 1][e + 2]);
            }
        __syncthreads();
        const bool whole = peers == 1 && count == sp.blocks;
        const auto write = [&](int r, int d, float f, const float4& sum) {
            const int p = p0 + r, h = head * group + p % group;
            const size_t to = ((size_t)(sp.begin + p / group) * a.heads + h) * c.dim + d;
            const float y[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < c.dim) store_out(a, to + e, f * y[e]);
        };
        // sums of `n` parts of row r below their common maxima, channels d to d + 3
        const auto meet = [&](int n, const RowStats* of, const float* from, int stride, int r, int d, RowStats& top) {
            top = {-INFINITY, -INFINITY, 0.f};
            for (int v = 0; v < n; ++v) {
                top.m = fmaxf(top.m, of[v * stride + r].m);
                top.w = fmaxf(top.w, of[v * stride + r].w);
            }
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int v = 0; v < n; ++v) {
                const RowStats y = of[v * stride + r];
                const float f = lower_to(y.w, top.w);
                const float4 z = *reinterpret_cast<const float4*>(from + (size_t)(v * stride + r) * DP + d);
                top.l += y.l * lower_to(y.m, top.m);
                sum.x += f * z.x; sum.y += f * z.y; sum.z += f * z.z; sum.w += f * z.w;
            }
            return sum;
        };
        const int tasks = rows * (DP / 4);
        RowStats* const met = reinterpret_cast<RowStats*>(sums + kWarps * kRows * DP);
        const size_t slot = 2 * (size_t)blockIdx.x + (b0 == 0);
        for (int i = threadIdx.x; i < tasks; i += F::kThreads) {
            const int r = i / (DP / 4), d = i % (DP / 4) * 4;
            RowStats top;
            const float4 sum = meet(kWarps, stats, sums, kRows, r, d, top);
            if (whole) {
                write(r, d, row_factor(a, head * group + (p0 + r) % group, top.m, top.w, top.l), sum);
            } else if (peers > 1) {
                *reinterpret_cast<float4*>(sums + r * DP + d) = sum;                 // (where this thread has read)
                if (d == 0) met[r] = top;
            } else {
                *reinterpret_cast<float4*>(part + (slot * kRows + r) * DP + d) = sum;
                if (d == 0) part_stats[slot * kRows + r] = top;
            }
        }
        if (peers > 1) {
            // every CTA joins some channels of all
            cluster_met();
            for (int i = threadIdx.x * peers + rank; i < tasks; i += F::kThreads * peers) {
                const int r = i / (DP / 4), d = i % (DP / 4) * 4;
                RowStats y[kMostPeers], top{-INFINITY, -INFINITY, 0.f};
                float4 z[kMostPeers], sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int v = 0; v < kMostPeers; ++v) {
                    y[v] = {-INFINITY, -INFINITY, 0.f};
                    z[v] = sum;
                    if (v >= peers) continue;
                    const uint32_t of = shared_of(met + r, v);
                    y[v] = {load_of(of), load_of(of + 4), load_of(of + 8)};
                    z[v] = load4_of(shared_of(sums + r * DP + d, v));
                    top.m = fmaxf(top.m, y[v].m);
                    top.w = fmaxf(top.w, y[v].w);
                }
#pragma unroll
                for (int v = 0; v < kMostPeers; ++v) {
                    const float f = lower_to(y[v].w, top.w);
                    top.l += y[v].l * lower_to(y[v].m, top.m);
                    sum = make_float4(sum.x + f * z[v].x, sum.y + f * z[v].y, sum.z + f * z[v].z, sum.w + f * z[v].w);
                }
                write(r, d, row_factor(a, head * group + (p0 + r) % group, top.m, top.w, top.l), sum);
            }
            cluster_met();                                                           // (nobody reads here any more)
        } else if (!whole) {
            // Runs c0 to c1 share the tile; the last of them to come joins all, in their order.  (A run is the first one of at most one shared tile, whose counter it lends.)
            // Where they are many, the last of every kJoin in turn joins those, in the first one's place, and the last of these their sums.  (Their counter is lent by the last run
            // of the kJoin, which is no other tile's but as its first.)
            const long long start = at.base + item * sp.share;
            const int c0 = (int)(start / at.per), all = (int)((start + (at.run ? sp.share : sp.blocks) - 1) / at.per) - c0 + 1;
            const bool twice = all > 2 * kJoin;
            const int run0 = (int)blockIdx.x - c0;
            int from = twice ? run0 / kJoin * kJoin : 0, n = twice ? min(kJoin, all - from) : all, apart = 1;
#pragma unroll 1
            for (bool ends = !twice;; ends = true) {
                __threadfence();
                __syncthreads();
                if (threadIdx.x == 0) {
                    if (!beside) asm volatile("griddepcontrol.wait;" ::: "memory");  // (the counters are zeros)
                    last = atomicAdd(arrived + c0 + (ends ? 0 : kMostCtas + from + n - 1), 1u) == (unsigned)(n - 1);
                }
                __syncthreads();
                if (!last) break;
                __threadfence();
                // rows' weights of the runs first, where the rings lay, then their channels; threads that these leave over take runs of their own
                float* const weights = sums + kWarps * kRows * DP;                   // [run][row]
                const int groups = max(1, min(F::kThreads / tasks, kWarps)), mine = threadIdx.x / tasks;
                const auto at_run = [&](int v, int r) { const int run = from + v * apart; return ((size_t)2 * (c0 + run) + (run == 0)) * kRows + r; };
                // (Loads go out many at a time: one after the other, those of 148 runs took 12 us.)
                for (int r = warp; r < rows; r += kWarps) {
                    constexpr int kMine = (F::kCtas + 31) / 32;
                    RowStats y[kMine], top{-INFINITY, -INFINITY, 0.f};
#pragma unroll
                    for (int j = 0; j < kMine; ++j) {
                        const int v = lane + 32 * j;
                        y[j] = {-INFINITY, -INFINITY, 0.f};
                        if (v < n) y[j] = {__ldcg(&part_stats[at_run(v, r)].m), __ldcg(&part_stats[at_run(v, r)].w), __ldcg(&part_stats[at_run(v, r)].l)};
                    }
#pragma unroll
                    for (int j = 0; j < kMine; ++j) top = {fmaxf(top.m, y[j].m), fmaxf(top.w, y[j].w), 0.f};
#pragma unroll
                    for (int d = 16; d; d >>= 1) {
                        top.m = fmaxf(top.m, __shfl_xor_sync(0xffffffffu, top.m, d));
                        top.w = fmaxf(top.w, __shfl_xor_sync(0xffffffffu, top.w, d));
                    }
#pragma unroll
                    for (int j = 0; j < kMine; ++j) {
                        top.l += y[j].l * lower_to(y[j].m, top.m);
                        if (lane + 32 * j < n) weights[(lane + 32 * j) * kRows + r] = lower_to(y[j].w, top.w);
                    }
#pragma unroll
                    for (int d = 16; d; d >>= 1) top.l += __shfl_xor_sync(0xffffffffu, top.l, d);
                    if (lane == 0) {
                        row_scale[r] = row_factor(a, head * group + (p0 + r) % group, top.m, top.w, top.l);
                        if (!ends) part_stats[at_run(0, r)] = top;
                    }
                }
                __syncthreads();
                const auto out = [&](int r, int d, const float4& sum) {
                    if (ends) write(r, d, row_scale[r], sum);
                    else *reinterpret_cast<float4*>(part + at_run(0, r) * DP + d) = sum;
                };
                for (int i = groups == 1 ? threadIdx.x : threadIdx.x % tasks; i < tasks && mine < groups; i += groups == 1 ? F::kThreads : tasks) {
                    const int r = i / (DP / 4), d = i % (DP / 4) * 4;
                    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                    constexpr int kAtOnce = 16;
#pragma unroll 1
                    for (int v0 = groups == 1 ? 0 : mine; v0 < n; v0 += kAtOnce * groups) {
                        float4 z[kAtOnce];
#pragma unroll
                        for (int j = 0; j < kAtOnce; ++j) {
                            const int v = v0 + j * groups;
                            z[j] = v < n ? __ldcg(reinterpret_cast<const float4*>(part + at_run(v, r) * DP + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        }
#pragma unroll
                        for (int j = 0; j < kAtOnce; ++j) {
                            const float f = v0 + j * groups < n ? weights[(v0 + j * groups) * kRows + r] : 0.f;
                            sum = make_float4(sum.x + f * z[j].x, sum.y + f * z[j].y, sum.z + f * z[j].z, sum.w + f * z[j].w);
                        }
                    }
                    if (groups == 1) out(r, d, sum);
                    else *reinterpret_cast<float4*>(sums + (size_t)(mine * kRows + r) * DP + d) = sum;
                }
                if (groups > 1) {
                    __syncthreads();
                    if (threadIdx.x < tasks) {
                        const int r = threadIdx.x / (DP / 4), d = threadIdx.x % (DP / 4) * 4;
                        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (int v = 0; v < groups; ++v) {
                            const float4 z = *reinterpret_cast<const float4*>(sums + (size_t)(v * kRows + r) * DP + d);
                            sum = make_float4(sum.x + z.x, sum.y + z.y, sum.z + z.z, sum.w + z.w);
                        }
                        out(r, d, sum);
                    }
                }
                if (ends) break;
                from = 0;
                n = (all + kJoin - 1) / kJoin;
                apart = kJoin;
            }
        }
        __syncthreads();                                                             // (the ring and the queries' room are taken again)
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");        // (the sequences of many rows, which may still be on their way beside this)
}

// Zeros for the counters of both kernels, which start meanwhile (a memset in front of them takes 3 us)
constexpr int kCounterThreads = 512;
__global__ void kv8_counters_kernel(unsigned* counters, int n) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int i = threadIdx.x; i < n; i += kCounterThreads) counters[i] = 0u;
}

inline bool wide(const Kv8Rows& x, int type, int dim) {
    const long long b = type_bytes(type);
    return (reinterpret_cast<uintptr_t>(x.x) & 15) == 0 && x.row * b % 16 == 0 && x.head * b % 16 == 0 && dim % 8 == 0;
}
// Room of the runs' parts, and how many of a shared tile's have come
struct FewWork {
    float* part;
    RowStats* stats;
    unsigned* arrived;
};
inline int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
inline int terms_of(int type) { return type == kTypeF32 ? 2 : 1; }
// tiles of eight rows where sequences have no more of them on average (the products of 16 rows take twice the registers and the tensor cores' time: 64 requests 226 and 305 us, eight of
// fp32 19 and 24; two tiles of eight would read the cache twice).  The average is over all of a step's rows: beside prompts single tokens get tiles of 16, as
// which sequence has how many rows is known on the device alone.
inline bool eight_rows(int kv_heads, int rows, int heads, int sequences) { return (long long)rows * (heads / kv_heads) <= 8ll * sequences; }

template <int DP, int FORMAT, int TERMS, int NT>
cudaError_t run_few(const Kv8Cache& c, const Kv8Step& s, const Kv8Attention& a, bool early, bool beside, const FewWork& work, cudaStream_t st) {
    using F = Few<DP, TERMS, NT>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = dia::ask_smem<kv8_attention_few_kernel<DP, FORMAT, TERMS, NT>>(dev, F::kSmem);
    if (e != cudaSuccess) return e;
    const auto kernel = kv8_attention_few_kernel<DP, FORMAT, TERMS, NT>;
    if (a.whole > 1) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(F::kCtas / a.whole * a.whole));
        cfg.blockDim = dim3(F::kThreads);
        cfg.dynamicSmemBytes = F::kSmem;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)a.whole;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kernel, c, s, a, (int)beside, work.part, work.stats, work.arrived);
    }
    return launch_pdl_if(early, kernel, dim3(F::kCtas), dim3(F::kThreads), F::kSmem, st, c, s, a, beside, work.part, work.stats, work.arrived);
}
template <int DP, int FORMAT>
cudaError_t run_few(const Kv8Cache& c, const Kv8Step& s, const Kv8Attention& a, bool beside, const FewWork& work, cudaStream_t st) {
    const bool early = !a.whole;                              // (behind the counters' kernel, or the tiles')
    const bool eight = eight_rows(c.kv_heads, s.rows, a.heads, s.sequences);
    if (terms_of(a.type) == 2) return eight ? run_few<DP, FORMAT, 2, 1>(c, s, a, early, beside, work, st) : run_few<DP, FORMAT, 2, 2>(c, s, a, early, beside, work, st);
    return eight ? run_few<DP, FORMAT, 1, 1>(c, s, a, early, beside, work, st) : run_few<DP, FORMAT, 1, 2>(c, s, a, early, beside, work, st);
}

}  // namespace

cudaError_t launch_kv8_append(const Kv8Cache& c, const Kv8Step& s, Kv8Rows k, Kv8Rows v, int type, cudaStream_t st) {
    // a warp per row where sequences have few of them (a decoding step's pages side by side: 4 us, by the page 12), per page's worth where they have many (8192 rows of prompts: 15 us, row
    // by row 74)
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
    // (98304 tokens: 56 us with 32 rows a CTA, 69 with 8; 992 tokens: 7.5 with 32, 4.4 with 8)
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
// Pairs of a sequence up to which tiles of 16 of them are the shorter way (four heads a key head; these and those of 256 rows: 36 pairs behind 1000 tokens 14 and 22 us, behind 16000
// 36 and 31; 68 pairs 17 and 25, 40 and 37, of eight sequences behind 8000 tokens 97 and 53).  How long pasts are moves the border and is known on the device alone, as is which sequence has how many
// rows: a step of more pairs in all gets both kernels.  So do single tokens, without `first` too, where the host could know that none of them needs the tiles': 17 of four heads a key head
// behind 1000 tokens take 18.3 us, 16 of them 12.0.
constexpr int kFewMost = 64;
// Tables of up to so many tokens for each of a cluster's CTAs: no tile is shared by others, which would need counters (a launch more) and sums by way of memory.  One request of 1025
// tokens: 14.3 us by one CTA a tile, 13.2 shared, 9.7 by eight; of 4000: 11.7 and 14.0 shared; of 16000: 21.6 and 20.0; nine of 8000: 29.2 by four and 24.0.  (Lengths are on the device, so that a
// table with room for more goes the shared way however short its sequences are.)
constexpr int kWholeTokens = 1024;
// and at least so many (of 128 tokens: 8.1 us alone, 9.0 by eight)
constexpr int kPeerTokens = 128;
inline bool some_in_tiles(int kv_heads, int dim, int rows, int heads, int type) { return kv8_tiles_ok(dim, type) && (long long)rows * (heads / kv_heads) > kFewMost; }
// CTAs of a cluster that takes tiles by itself: as many as there are for each tile; 0: tables are too long for that
inline int whole_tiles(int kv_heads, int dim, int rows, int heads, int type, int sequences, long long tokens) {
    if (some_in_tiles(kv_heads, dim, rows, heads, type)) return 0;
    const int each = eight_rows(kv_heads, rows, heads, sequences) ? 8 : 16, ctas = terms_of(type) == 2 || dim > 128 ? 148 : 296;      // (as Few has them)
    const long long tiles = kv_heads * (((long long)rows * (heads / kv_heads) + (long long)std::min(sequences, rows) * (each - 1)) / each);
    int peers = kMostPeers;
    while (peers > 1 && (tiles * peers > ctas || tokens <= peers / 2 * kPeerTokens)) peers /= 2;
    return tokens <= (long long)peers * kWholeTokens ? peers : 0;
}
}  // namespace

// Counters first: those of both kernels are set to zero in one go.
namespace {
constexpr size_t kCounters = (2 * kMostCtas + kKvTileCounters) * sizeof(unsigned);
inline size_t few_bytes(int dp) { return (size_t)2 * kMostCtas * 16 * (dp * sizeof(float) + sizeof(RowStats)); }
inline size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }
}  // namespace

size_t kv8_attention_work_bytes(int kv_heads, int dim, int rows, int heads, int type, int sequences, long long tokens) {
    if (whole_tiles(kv_heads, dim, rows, heads, type, sequences, tokens)) return 0;
    return rounded(kCounters) + rounded(few_bytes(padded_dim(dim))) + (some_in_tiles(kv_heads, dim, rows, heads, type) ? kv8_tiles_work_bytes(dim) : 0);
}

cudaError_t launch_kv8_attention(const Kv8Cache& c, const Kv8Step& s, Kv8Attention a, void* work, cudaStream_t st) {
    const int dp = padded_dim(c.dim);
    const bool tiles = some_in_tiles(c.kv_heads, c.dim, s.rows, a.heads, a.type), alone = tiles && s.sequences == 1;        // (alone: in tiles whatever its rows are)
    unsigned* const counters = reinterpret_cast<unsigned*>(work);
    float* const part = reinterpret_cast<float*>(reinterpret_cast<char*>(work) + rounded(kCounters));
    a.whole = whole_tiles(c.kv_heads, c.dim, s.rows, a.heads, a.type, s.sequences, (long long)s.max_pages << c.page_shift);
    cudaError_t e = cudaSuccess;
    if (!a.whole) {
        kv8_counters_kernel<<<1, kCounterThreads, 0, st>>>(counters, (int)(kCounters / sizeof(unsigned)));
        e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        ++dia::extra_launches();
    }
    a.few_most = !tiles ? 0x7fffffff : alone ? 0 : kFewMost;
    if (tiles) {
        e = launch_kv8_tiles(c, s, a, alone, reinterpret_cast<char*>(part) + rounded(few_bytes(dp)), counters + 2 * kMostCtas, st);
        if (e != cudaSuccess || alone) return e;
        ++dia::extra_launches();
    }
    const FewWork few{part, reinterpret_cast<RowStats*>(part + (size_t)2 * kMostCtas * 16 * dp), counters};
    if (c.format == kKvE4m3) return dp == 64 ? run_few<64, kKvE4m3>(c, s, a, tiles, few, st) : dp == 128 ? run_few<128, kKvE4m3>(c, s, a, tiles, few, st) : run_few<256, kKvE4m3>(c, s, a, tiles, few, st);
    return dp == 64 ? run_few<64, kKvInt8>(c, s, a, tiles, few, st) : dp == 128 ? run_few<128, kKvInt8>(c, s, a, tiles, few, st) : run_few<256, kKvInt8>(c, s, a, tiles, few, st);
}

}  // namespace lm
