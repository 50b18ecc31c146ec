// lm_kv8_tiles.cu - attention of many rows over the cache in 8 bits, on the 5th-generation tensor cores.
//
// A CTA takes 256 (token, query head) rows that share a key head and walks their keys 128 at a time:
//   warps 0-3, 4-7   one thread per row, 128 rows each: 64 scores at a time from tensor memory, softmax weights back to where they lay.  A half has two places for scores, so
//                    that the next ones are there when it has weighed these
//   warps 8-15       four warps the keys, four the values, 16 tokens of a step each: codes into shared memory by bulk copies, four steps ahead, and from there to fp16 operands
//   warps 16, 17     one elected lane each issues tcgen05.mma for a half: S = Q K^T (M = 128, N = 64), and O += P V with P as the operand in tensor memory
//   warp 18          looks up pages and scales, some tiles ahead
//
// Numbers.  t = scale log2(e) q . key + e - E in powers of two, e the exponent of the page's values and E the largest of the CTA's pages; P = 2^(t - R + 7) in fp16, with R the
// row's reference: about its largest t so far, raised (and O and the sum with it) only when one of 64 scores lies more than 8 above it, so P is at most 2^15.  That the page's value
// scale is inside
// the weight lets codes be multiplied as they are, and the 11 bits of P (a result in fp16 has no more, one in bf16 eight) count from the largest contribution.  The denominator takes
// 2^(E - e) out again, per 16 tokens.  Pages are those that the rows see; whose values are 2^80 below the largest page's are taken as zeros.  Queries are scaled by a power of two per row
// (exact but for channels 2^-27 below the row's largest).  Sums are fp32; O's live in tensor memory for the whole run of keys, and lose up to one unit in the last place per 16 keys (2^-24 on
// average: 2^-11 of the sum after 131072 keys, an eighth of what the result's rounding to bf16 may be off by, and as much as that to fp16).
//
// Bound: per 256 x 128 tile and dim 128 the tensor pipe takes 2048 cycles, the exponentials (16 a cycle) 2048, and shared memory 2048 (the scores' operands 1024, the values 512,
// the codes turned into operands 512).
#include <algorithm>
#include <type_traits>

#include "attention_split.h"
#include "engine_internal.h"
#include "gemm_tcgen05.h"
#include "lm_device.cuh"
#include "lm_kv8.cuh"
#include "lm_kv8.h"
#include "tensor_cores.cuh"

namespace lm {
namespace {

using namespace dia;

constexpr int kKeys = 128, kStepKeys = 64, kHalfRows = 128, kTileRows = 2 * kHalfRows, kThreads = 640, kSms = 148;
constexpr int kBlocks = kKeys / kKvBlock;                      // blocks of 16 tokens in a tile of keys
constexpr int kMinChunk = 4;                                   // tiles of keys that are worth a CTA of their own
constexpr float kSlack = 8.f, kBits = 7.f;                     // see above
constexpr int kSpread = 80;
constexpr int kLaunchRegs = 96, kSoftmaxRegs = 144, kFetchRegs = 48, kIssueRegs = 88;
static_assert(128 * (2 * kSoftmaxRegs + 2 * kFetchRegs + kIssueRegs) <= kThreads * kLaunchRegs, "the split is within the launch's registers");
static_assert(kSoftmaxRegs >= kLaunchRegs && kFetchRegs <= kLaunchRegs && kIssueRegs <= kLaunchRegs, "who gives registers and who takes them");
constexpr int kJoinOnce = 8;                                     // chunks that are joined in one go
constexpr int kAhead = 4;                                      // tiles whose pages and scales are known

template <int DP>
struct Tiles {
    static constexpr int kStages = DP == 64 ? 6 : 3, kSide = kStepKeys * DP * 2;      // operands of a step, keys or values
    static constexpr int kDepth = 4, kCodes = kStepKeys * DP; // and its codes
    static constexpr int kQ = kTileRows * DP * 2, kSmem = kQ + 2 * kStages * kSide + 2 * kDepth * kCodes;
};

// ---- who takes what ------------------------------------------------------------------------------------------------------------------------
// Items are (sequence, key head, 256 rows).  Where there are fewer than SMs, the keys of an item go in chunks, as many as all of them fill the GPU once with; the last
// chunk to come joins them.  Items of a sequence go last rows first: those see the most keys.
struct Sequence {
    int begin, n, past, tiles, low, high;                     // low, high: tiles of keys that its rows look at
};
__device__ __forceinline__ Sequence sequence_at(const Kv8Step& s, const Kv8Attention& a, int i, int group, int page_shift) {
    Sequence q;
    q.begin = s.begin(i);
    q.n = max(s.end(i) - q.begin, 0);
    q.past = s.past[i];
    const long long rows = (long long)q.n * group;
    q.tiles = rows > a.few_most ? (int)((rows + kTileRows - 1) / kTileRows) : 0;
    q.low = a.window > 0 ? (int)(max(0ll, (long long)q.past + 1 - a.window) / kKeys) : 0;
    const long long end = min((long long)max(q.past, 0) + q.n, (long long)s.max_pages << page_shift);
    q.high = q.past < 0 ? q.low : max((int)((end + kKeys - 1) / kKeys), q.low);
    return q;
}
struct Work {
    int seq, head, tile, chunk, chunks, first_cta, length;    // seq -1: nothing; length: of a chunk in tiles of keys
};
constexpr int kWhole = 0x7fffffff;
constexpr int kMostItems = 0x3000000;                          // above what a launch has (2^31 pairs / 256, and / 65 for the sequences' last ones), and 32 lanes' sums are below 2^31
// One warp: what the CTA of this index takes
__device__ __forceinline__ Work find_work(const Kv8Cache& c, const Kv8Step& s, const Kv8Attention& a, int group, int index) {
    const int lane = threadIdx.x & 31, each = (s.sequences + 31) / 32, i0 = lane * each, i1 = min(i0 + each, s.sequences);
    const auto before = [&](int v) {                          // sums of the lanes before this one, and of all
        int upto = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        return make_int2(upto - v, __shfl_sync(0xffffffffu, upto, 31));
    };
    const Sequence mine = sequence_at(s, a, min(i0, s.sequences - 1), group, c.page_shift);       // (a lane's only one, mostly)
    const auto at = [&](int i) { return i == i0 ? mine : sequence_at(s, a, i, group, c.page_shift); };
    int items = 0, most = 0, ctas = 0;
    for (int i = i0; i < i1; ++i) {
        const Sequence q = at(i);
        items = min(items + q.tiles * c.kv_heads, kMostItems);    // (offsets that decrease may count rows many times)
        if (q.tiles) most = max(most, q.high - q.low);
    }
    const int2 of_items = before(items);
    const int longest = (int)__reduce_max_sync(0xffffffffu, (unsigned)most);
    Work work{-1, 0, 0, 0, 1, 0, kWhole};
    if (of_items.y == 0) return work;
    const int share = of_items.y >= kSms ? 0 : kSms / of_items.y;
    const int length = share == 0 ? kWhole : max(kMinChunk, (longest + share - 1) / share);
    const auto chunks_of = [&](const Sequence& q) { return length == kWhole ? 1 : max(1, (q.high - q.low + length - 1) / length); };
    for (int i = i0; i < i1; ++i) {
        const Sequence q = at(i);
        ctas = min(ctas + q.tiles * c.kv_heads * chunks_of(q), kMostItems);
    }
    int base = before(ctas).x;
    const bool here = index >= base && index < base + ctas;
    if (here) {
        for (int i = i0;; ++i) {
            const Sequence q = at(i);
            const int chunks = chunks_of(q), units = q.tiles * c.kv_heads * chunks;
            if (index < base + units) {
                const unsigned local = index - base, item = local / (unsigned)chunks;
                work = {i, (int)(item % (unsigned)c.kv_heads), q.tiles - 1 - (int)(item / (unsigned)c.kv_heads), (int)(local - item * chunks), chunks, base + (int)item * chunks, length};
                break;
            }
            base += units;
        }
    }
    const unsigned who = __ballot_sync(0xffffffffu, here);
    const int from = who ? __ffs(who) - 1 : 0;
    const auto told = [&](int v) { return __shfl_sync(0xffffffffu, v, from); };
    return {told(work.seq), told(work.head), told(work.tile), told(work.chunk), told(work.chunks), told(work.first_cta), told(work.length)};
}

// A place in a ring of N, and which of a barrier's phases is its use's
template <int N>
struct Turn {
    int at = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++at == N) {
            at = 0;
            phase ^= 1u;
        }
    }
};

// ---- tensor memory and shared memory -------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_load32(uint32_t addr, float* v) {
    uint32_t u[32];
    tmem_columns32(addr, u);
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(u[e]);
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
        "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
        "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Operands lie in blocks of 8 rows x 16 bytes, [row / 8][channel / 8]: lead / stride are the bytes between blocks along the contraction / the rows (scores: the contraction runs
// over channels; values: over rows, and the channels are what is far apart)
__device__ __forceinline__ uint64_t block_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    const uint32_t lo = ((addr & 0x3FFFFu) >> 4) | ((lead >> 4) << 16), hi = (stride >> 4) | (1u << 14);
    return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ void mma_weights(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {      // A in tensor memory
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

struct Beside {                                               // rows between neighbouring chunks, known when it is compiled
    __device__ __forceinline__ operator int() const { return kTileRows; }
};

template <int DP, int FORMAT>
__global__ void __launch_bounds__(kThreads, 1) kv8_attention_tiles_kernel(Kv8Cache c, Kv8Step s, Kv8Attention a, int alone, float* part, RowStats* part_stats, unsigned* arrived, int* ran_out, unsigned polls) {
    using T = Tiles<DP>;
    constexpr int kStages = T::kStages, kDepth = T::kDepth, kSteps = DP / 16;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* const q_tile = smem;                             // [half]
    uint8_t* const k_ring = smem + T::kQ;
    uint8_t* const v_ring = k_ring + kStages * T::kSide;
    uint8_t* const codes = v_ring + kStages * T::kSide;       // [keys, values][kDepth]
    __shared__ uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], m_full[kAhead], m_empty[kAhead], c_full[8][kDepth], s_full[2][2], p_ready[2][2], pv_done[2][2], done[2];
    __shared__ float4 blocks[kAhead][kBlocks];                // (key scale, e - E, 2^(E - e), page) of 16 tokens
    __shared__ uint3 which[kAhead];                           // of a tile's blocks: those that are there, whose values are taken as zeros, that stand for numbers
    __shared__ uint32_t tmem_slot;
    __shared__ int largest;                                   // exponent of the values' pages
    __shared__ uint64_t q_ready;
    __shared__ Work found;
    __shared__ Sequence found_rows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.heads / c.kv_heads;
    if (warp == 0) {
        const Work work = find_work(c, s, a, group, blockIdx.x);
        if (lane == 0) {
            found = work;
            if (work.seq >= 0) found_rows = sequence_at(s, a, work.seq, group, c.page_shift);
        }
    } else if (threadIdx.x == 32) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&k_full[i], 4);
            mbar_init(&v_full[i], 4);
            mbar_init(&k_empty[i], 2);
            mbar_init(&v_empty[i], 2);
        }
        for (int i = 0; i < kAhead; ++i) {
            mbar_init(&m_full[i], 1);
            mbar_init(&m_empty[i], 16);
        }
        for (int w = 0; w < 8; ++w)
            for (int i = 0; i < kDepth; ++i) mbar_init(&c_full[w][i], 1);
        for (int g = 0; g < 2; ++g) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(&s_full[g][i], 1);
                mbar_init(&p_ready[g][i], 4);
                mbar_init(&pv_done[g][i], 1);
            }
            mbar_init(&done[g], 1);
        }
        mbar_init(&q_ready, 8);
        largest = -1000;
        fence_mbar_init();
    } else if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    } else if (warp == 19) {
        // The counters are zeros behind this; the kernel of the sequences of few rows, which wants them too, may start (its writes are its own)
        asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        if (alone) zero_rows_of_none(s, a, c.dim, (long long)blockIdx.x * 32 + lane, (long long)gridDim.x * 32);
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;                          // scores (and weights) of the halves 0, 128; outputs 256, 384
    const Work work = found;
    if (work.seq < 0) {
        if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
        return;
    }
    const Sequence q = found_rows;
    // tiles of keys: the first one, and how many of them the halves of the rows look at
    const int pairs = q.n * group, p0 = work.tile * kTileRows;
    const auto position = [&](int p) { return (long long)q.past + min(p, pairs - 1) / group; };
    const long long back = a.window > 0 ? a.window - 1 : (1ll << 40);
    const int from = max(max(q.low, (int)(max(0ll, position(p0) - back) / kKeys)), work.length == kWhole ? 0 : q.low + work.chunk * work.length);
    const int limit = work.length == kWhole ? q.high : (int)min((long long)q.high, (long long)q.low + (long long)(work.chunk + 1) * work.length);
    const auto steps_of = [&](int g) {
        if (p0 + g * kHalfRows >= pairs || q.past < 0) return 0;
        const long long end = min((long long)limit * kKeys, position(p0 + g * kHalfRows + kHalfRows - 1) + 1) - (long long)from * kKeys;
        return (int)max(0ll, (end + kStepKeys - 1) / kStepKeys);
    };
    const int n0 = steps_of(0), n1 = steps_of(1), steps = max(n0, n1), n = (steps + 1) / 2;      // of the halves, and tiles
    // the page of a block of 16 tokens.  Places of the table behind the sequence's last token, and in front of the first one that these rows see, may hold anything: no page there
    const long long seen_from = max(0ll, position(p0) - back), seen_to = (long long)q.past + q.n;
    const auto page_at = [&](long long token) { return token < seen_to && token + kKvBlock > seen_from ? s.page(work.seq, token >> c.page_shift, c.pages) : -1; };
    const auto find_largest = [&] {                           // the largest exponent of the values' pages (all warps but the rows')
        int most = -1000;
        for (int b = threadIdx.x - 256; b < n * kBlocks; b += kThreads - 256) {
            const int page = page_at((long long)from * kKeys + (long long)b * kKvBlock);
            if (page < 0) continue;
            const uint32_t v = __float_as_uint(c.value_scales[(size_t)page * c.kv_heads + work.head]);
            if (v < 0x7f800000u) most = max(most, (int)(v >> 23) - 127);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0 && most > -1000) atomicMax(&largest, most);
        asm volatile("bar.sync 1, %0;" ::"n"(kThreads - 256) : "memory");
    };
    bool ok = true;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        float row_scale = 0.f;
        {
            // queries: a warp takes its 32 rows, eight at a time, a lane DP / 4 channels of one in pieces of eight
            constexpr int kPieces = DP / 32;
            const int sub = lane & 7;
            const bool wide = c.dim % 8 == 0 && (reinterpret_cast<uintptr_t>(a.q.x) & 15) == 0 && a.q.row % 8 == 0 && a.q.head % 8 == 0;
            uint4 w[4][kPieces];
#pragma unroll
            for (int r8 = 0; r8 < 4; ++r8) {
                const int p = p0 + warp * 32 + r8 * 8 + sub, in = min(p, pairs - 1);
                const uint16_t* const row = reinterpret_cast<const uint16_t*>(a.q.x) + (q.begin + (long long)(in / group)) * a.q.row + (long long)(work.head * group + in % group) * a.q.head;
#pragma unroll
                for (int j = 0; j < kPieces; ++j) {
                    const int d = 8 * ((lane >> 3) + 4 * j);
                    w[r8][j] = make_uint4(0u, 0u, 0u, 0u);
                    if (p >= pairs || d >= c.dim) continue;
                    if (wide) {
                        w[r8][j] = *reinterpret_cast<const uint4*>(row + d);
                    } else {
                        uint16_t y[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = d + e < c.dim ? row[d + e] : 0;
                        memcpy(&w[r8][j], y, 16);
                    }
                }
            }
            const auto numbers = [&](uint32_t u) {
                if (a.type == kTypeBf16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
                return __half22float2(*reinterpret_cast<const __half2*>(&u));
            };
#pragma unroll
            for (int r8 = 0; r8 < 4; ++r8) {
                uint32_t most = 0;
#pragma unroll
                for (int j = 0; j < kPieces; ++j) {
                    const uint32_t u[4] = {w[r8][j].x, w[r8][j].y, w[r8][j].z, w[r8][j].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = numbers(u[e]);
                        most = max(most, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
                    }
                }
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 8));
                most = max(most, __shfl_xor_sync(0xffffffffu, most, 16));
                const uint32_t e = most == 0 ? 127u : max(most >> 23, 14u);
                const float f = __uint_as_float((267u - e) << 23), way_back = __uint_as_float((e - 13u) << 23);       // 2^(140 - e): to below 2^14, and the way back
                // (a thread's own row is 8 r8 + sub of its warp's.  Below zero: its query is not finite, and its operand is zeros, so that what it does not see stays hidden)
                if (r8 == lane >> 3) row_scale = e == 255u ? -1.f : way_back * (a.scale * kLog2e);
                uint8_t* const to = q_tile + (warp >> 2) * (kHalfRows * DP * 2) + ((warp & 3) * 4 + r8) * (DP * 16) + sub * 16;
#pragma unroll
                for (int j = 0; j < kPieces; ++j) {
                    uint32_t u[4] = {w[r8][j].x, w[r8][j].y, w[r8][j].z, w[r8][j].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 y = numbers(u[i]);
                        u[i] = e == 255u ? 0u : pack_half(y.x * f, y.y * f);
                    }
                    *reinterpret_cast<uint4*>(to + ((lane >> 3) + 4 * j) * 128) = make_uint4(u[0], u[1], u[2], u[3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_ready);
        }
        const int g = warp >> 2, count = g ? n1 : n0;
        const uint32_t lanes = (uint32_t)(warp & 3) * 32u << 16, t_scores = tmem + lanes + 128u * g, t_o = tmem + lanes + 256u + 128u * g;
        const int p = p0 + threadIdx.x;
        // the tokens that the row sees, and the ones that all 128 rows see, counted from the first tile on
        const long long tok0 = (long long)from * kKeys;
        const auto within = [&](long long v) { return (int)max(min(v - tok0, 0x7fffff00ll), -1ll); };
        const int hi = within(position(p)), lo = within(position(p) - back), all_hi = within(position(p0 + g * kHalfRows)), all_lo = within(position(p0 + g * kHalfRows + kHalfRows - 1) - back);
        // What a score is times.  Hidden ones are -infinity, so it must not be zero, which the product comes to where a page's step is 2^-100 (zeros) or none (never written) and the query or
        // the scale is small.  (Scores are below 2^30, so what is raised to 2^-126 moves by 2^-96 at most.)
        const auto factor = [&](float key_scale) { return fmaxf(key_scale * row_scale, 0x1p-126f); };
        float ref = -1e30f, l = 0.f;
        // (A step's scores come behind the value product of two steps before, not of the last one: what is told of every step has a barrier for the even ones and one for the odd.)
#pragma unroll 1
        for (int t = 0; t < count; ++t) {
            const int i = t >> 1, half = t & 1, slot = i % kAhead;
            if (half == 0 && !pair_wait(&m_full[slot], (uint32_t)(i / kAhead) & 1u, polls)) { ok = false; break; }
            const uint32_t numbers = which[slot].z >> (4 * half);
            const float4* const meta_of = &blocks[slot][4 * half];
            const int tok = t * kStepKeys;
            const uint32_t t_s = t_scores + kStepKeys * half;
            const bool clear = (numbers & 0xfu) == 0xfu && tok + kStepKeys - 1 <= all_hi && tok >= all_lo;
            if (!pair_wait(&s_full[g][half], i & 1, polls)) { ok = false; break; }
            fence_after();
            if (!clear) {
                // What a row does not see is -infinity, what it sees of a page that stands for NaNs is NaN: 16 scores a turn, in tensor memory, since this code should be short (it is
                // rarely needed, and what is in the loop at all costs all of it instruction fetches: 193 -> 191 us, 512 rows behind 16384, with 450 instructions less)
                const unsigned first = (unsigned)(lo - tok), many = (unsigned)(hi - lo);      // (what it sees in turn; nothing: hi is -1, or below lo)
                const bool none = hi < tok || hi < lo;
#pragma unroll 1
                for (int b = 0; b < 4; ++b) {
                    uint32_t v[16];
                    tmem_columns16(t_s + 16 * b, v);
                    tmem_loaded();
                    const bool nan = !(numbers >> b & 1u);
#pragma unroll
                    for (int e = 0; e < 16; ++e) v[e] = none || 16 * b + e - first > many ? 0xff800000u : nan ? 0x7fffffffu : v[e];
                    tmem_store16(t_s + 16 * b, v);
                }
                tmem_stored();
            }
            uint32_t x[2][32];
            tmem_columns32(t_s, x[0]);
            tmem_columns32(t_s + 32, x[1]);
            tmem_loaded();
            const auto score = [&](int b, int e) { return __uint_as_float(x[b / 2][16 * (b & 1) + e]); };
            float top = -INFINITY;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float2 meta = *reinterpret_cast<const float2*>(meta_of + b);
                float m = max3(score(b, 0), score(b, 1), score(b, 2));
#pragma unroll
                for (int e = 3; e < kKvBlock - 1; e += 2) m = max3(m, score(b, e), score(b, e + 1));
                top = fmaxf(top, fmaf(fmaxf(m, score(b, 15)), factor(meta.x), meta.y));
            }
            if (__any_sync(0xffffffffu, top > ref + kSlack)) {
                const float next = top > ref + kSlack ? top : ref, f = exp2_fast(ref - next);
                ref = next;
                l *= f;
                if (t > 0) {
                    if (!pair_wait(&pv_done[g][half ^ 1], (uint32_t)((t - 1) >> 1) & 1u, polls)) { ok = false; break; }
                    fence_after();
#pragma unroll 1
                    for (int j = 0; j < DP; j += 32) {
                        uint32_t o[32];
                        tmem_columns32(t_o + j, o);
                        tmem_loaded();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_store32(t_o + j, o);
                    }
                }
            }
            uint32_t w[32];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float4 meta = meta_of[b];
                const f2 k2 = twice(factor(meta.x)), c2 = twice(meta.y - ref + kBits);
                f2 sum[2] = {0, 0};
#pragma unroll
                for (int e = 0; e < kKvBlock; e += 2) {
                    float y0, y1;
                    unpack2(fma2(pack2(score(b, e), score(b, e + 1)), k2, c2), y0, y1);
                    y0 = exp2_fast(y0);
                    y1 = exp2_fast(y1);
                    sum[e / 2 & 1] = add2(sum[e / 2 & 1], pack2(y0, y1));
                    w[8 * b + e / 2] = pack_half(y0, y1);
                }
                float s0, s1;
                unpack2(add2(sum[0], sum[1]), s0, s1);
                l = fmaf(s0 + s1, meta.z, l);
            }
            tmem_store32(t_s, w);
            tmem_stored();
            fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&p_ready[g][half]);
                if (half == 1 || t + 1 == count) mbar_arrive(&m_empty[slot]);
            }
        }
        // (a half that looks at fewer tiles lets the others have the rest)
        for (int i = (count + 1) / 2; ok && i < n; ++i) {
            if (!pair_wait(&m_full[i % kAhead], (uint32_t)(i / kAhead) & 1u, polls)) ok = false;
            else if (lane == 0) mbar_arrive(&m_empty[i % kAhead]);
        }
        if (ok && count > 0 && !pair_wait(&pv_done[g][(count - 1) & 1], (uint32_t)((count - 1) >> 1) & 1u, polls)) ok = false;
        fence_after();
        if (row_scale < 0.f && l != 0.f) l = __uint_as_float(0x7fc00000u);               // (it saw something)
        // out
        const float spread = (float)(largest == -1000 ? 0 : largest);
        float m = ref - kBits, w = m + spread + kWeightBits;
        if (l == 0.f) m = w = -INFINITY;
        const bool in = p < pairs, whole = work.chunks == 1;
        const int h = work.head * group + min(p, pairs - 1) % group;
        const size_t to = ((size_t)(q.begin + min(p, pairs - 1) / group) * a.heads + h) * c.dim;
        float f = whole ? row_factor(a, h, m, w, l) : 1.f;
        if (!ok) f = __uint_as_float(0x7fc00000u);
        const size_t slot = ((size_t)work.first_cta + work.chunk) * kTileRows + threadIdx.x;
        if (!whole && in) part_stats[slot] = {m, w, l};
        const bool wide = c.dim % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
#pragma unroll 1
        for (int j = 0; j < DP; j += 32) {
            float o[32];
            if (count > 0) {
                tmem_load32(t_o + j, o);
                tmem_loaded();
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0.f;
            }
            if (!in) continue;
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(part + slot * DP + j + e) = make_float4(o[e] * f, o[e + 1] * f, o[e + 2] * f, o[e + 3] * f);
            } else if (wide) {
                uint16_t* const y = reinterpret_cast<uint16_t*>(a.out) + to + j;
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    if (j + e >= c.dim) break;
                    uint32_t u[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float y0 = o[e + 2 * k] * f, y1 = o[e + 2 * k + 1] * f;
                        if (a.type == kTypeBf16) {
                            const __nv_bfloat162 b = __floats2bfloat162_rn(y0, y1);
                            u[k] = *reinterpret_cast<const uint32_t*>(&b);
                        } else {
                            u[k] = pack_half(y0, y1);
                        }
                    }
                    *reinterpret_cast<uint4*>(y + e) = make_uint4(u[0], u[1], u[2], u[3]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (j + e < c.dim) store_out(a, to + j + e, o[e] * f);
            }
        }
    } else if (warp < 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFetchRegs));
        find_largest();
        // ---- codes to operands: four warps the keys, four the values, a block of every step each, eight rows of it a turn, a lane 16 channels of one.  Eight neighbouring lanes
        // take eight rows and as many different pieces, so that neither what they read nor what they write meets in a bank ----
        constexpr int kParts = DP / 64;                       // 16-byte pieces of a row that a lane takes
        const int side = (warp - 8) >> 2, block = warp & 3, sub = lane & 7;
        uint64_t* const full = side ? v_full : k_full;
        uint64_t* const empty = side ? v_empty : k_empty;
        uint8_t* const ring = side ? v_ring : k_ring;
        uint8_t* const mine = codes + (warp - 8) * kDepth * (T::kCodes / 4);      // this warp's codes of so many steps
        uint64_t* const arrived_codes = c_full[warp - 8];
        const auto lay = [&](const uint8_t* from, uint8_t* to, bool zeros) {
#pragma unroll
            for (int r8 = 0; r8 < 2; ++r8)
#pragma unroll
                for (int j = 0; j < kParts; ++j) {
                    const int piece = DP == 64 ? ((sub >> 1) + (lane >> 3)) & 3 : (sub + (lane >> 3) + 4 * j) & 7;
                    uint4 w = make_uint4(0u, 0u, 0u, 0u);
                    if (!zeros && piece * 16 < c.stride) w = *reinterpret_cast<const uint4*>(from + (8 * r8 + sub) * c.stride + piece * 16);
                    uint4 lo, hi;
                    decode4<FORMAT>(w.x, lo.x, lo.y);
                    decode4<FORMAT>(w.y, lo.z, lo.w);
                    decode4<FORMAT>(w.z, hi.x, hi.y);
                    decode4<FORMAT>(w.w, hi.z, hi.w);
                    uint8_t* const d = to + (2 * block + r8) * (DP * 16) + piece * 256 + sub * 16;
                    *reinterpret_cast<uint4*>(d) = lo;
                    *reinterpret_cast<uint4*>(d + 128) = hi;
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        };
        const uint8_t* const pages = side ? c.values : c.keys;
        const uint32_t bytes = (uint32_t)(kKvBlock * c.stride);
        unsigned issued = 0;
        const auto fetch = [&](int t, int slot) {             // step t's block, if it is there, by one bulk copy (a warp that issued them for all took 200 cycles each)
            const int i = t >> 1;
            if (!pair_wait(&m_full[i % kAhead], (uint32_t)(i / kAhead) & 1u, polls)) { ok = false; return; }
            if (lane == 0) {
                const int page = __float_as_int(blocks[i % kAhead][4 * (t & 1) + block].w);
                mbar_arrive_expect_tx(&arrived_codes[slot], page >= 0 ? bytes : 0u);
                if (page >= 0) {
                    const int in_page = (int)(((long long)from * kKeys + (long long)t * kStepKeys + block * kKvBlock) & ((1 << c.page_shift) - 1));
                    bulk_g2s(mine + slot * (T::kCodes / 4), pages + ((((size_t)page * c.kv_heads + work.head) << c.page_shift) + in_page) * c.stride, bytes, &arrived_codes[slot]);
                }
            }
            ++issued;
        };
        for (int t = 0; ok && t < min(kDepth, steps); ++t) fetch(t, t);
        Turn<kStages> out;
        Turn<kDepth> in;
#pragma unroll 1
        for (int t = 0; ok && t < steps; ++t, out.next(), in.next()) {
            if (!pair_wait(&arrived_codes[in.at], in.phase, polls) || (t >= kStages && !pair_wait(&empty[out.at], out.phase ^ 1u, polls))) { ok = false; break; }
            const int slot = (t >> 1) % kAhead, bit = 4 * (t & 1) + block;
            const uint3 of = which[slot];
            lay(mine + in.at * (T::kCodes / 4), ring + out.at * T::kSide, !(of.x >> bit & 1u) || (side && (of.y >> bit & 1u)));
            if (lane == 0) {
                mbar_arrive(&full[out.at]);
                if ((t & 1) || t + 1 == steps) mbar_arrive(&m_empty[slot]);
            }
            if (t + kDepth < steps) fetch(t + kDepth, in.at); // (all lanes have read what lay there: lay ends with a barrier of the warp)
        }
        if (!ok && lane == 0) copies_landed(arrived_codes, kDepth, issued);              // (nothing arrives behind the kernel)
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        find_largest();
        if (warp < 18) {
            const uint32_t idesc_s = (1u << 4) | ((uint32_t)(kStepKeys >> 3) << 17) | ((uint32_t)(kHalfRows >> 4) << 24);
            const uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(kHalfRows >> 4) << 24);
            // A warp for each half, so that one has its turn ready while the other's is in the tensor pipe.  What an instruction takes is broadcast from one lane, where it is
            // used, so that it is known to be the same in every lane.
            const auto same = [](uint32_t v) {
                asm volatile("" : "+r"(v));
                return __shfl_sync(0xffffffffu, v, 0);
            };
            const int g = warp - 16, mine = (int)same((uint32_t)(g ? n1 : n0)), un = (int)same((uint32_t)steps);
            const uint32_t q_at = smem_u32(q_tile) + g * (kHalfRows * DP * 2), t_g = tmem + 128u * g;
            Turn<kStages> keys, values;
            // The scores of step t, if it is this half's; the slot is free behind them
            const auto scores = [&](uint32_t ts, uint32_t qa, uint32_t ka, int t) {       // (one lane)
                if (t < mine) {
                    const uint64_t qd = block_desc(qa, 128u, DP * 16u), kd = block_desc(ka, 128u, DP * 16u);
#pragma unroll
                    for (uint32_t k = 0; k < kSteps; ++k) umma_bf16(ts, qd + 16u * k, kd + 16u * k, idesc_s, k != 0);
                    umma_commit(&s_full[g][t & 1]);
                }
                umma_commit(&k_empty[keys.at]);
            };
            if (un > 0 && !pair_wait(&q_ready, 0u, polls)) ok = false;
#pragma unroll 1
            for (int t = 0; ok && t < min(un, 2); ++t, keys.next()) {
                if (!pair_wait(&k_full[keys.at], keys.phase, polls)) { ok = false; break; }
                fence_after();
                const uint32_t ts = same(t_g + kStepKeys * t), qa = same(q_at), ka = same(smem_u32(k_ring + keys.at * T::kSide));
                if (elect_one_sync()) scores(ts, qa, ka, t);
                __syncwarp();
            }
            // A turn behind the weights of step t: their values, and the scores two steps on, whose place the weights had
#pragma unroll 1
            for (int t = 0; ok && t < un; ++t, values.next()) {
                const int h = t & 1;
                const bool more = t + 2 < un;
                if (!pair_wait(&v_full[values.at], values.phase, polls) || (more && !pair_wait(&k_full[keys.at], keys.phase, polls)) ||
                    (t < mine && !pair_wait(&p_ready[g][h], (uint32_t)(t >> 1) & 1u, polls))) {
                    ok = false;
                    break;
                }
                fence_after();
                const uint32_t ts = same(t_g + kStepKeys * h), to = same(t_g + 256u), va = same(smem_u32(v_ring + values.at * T::kSide)), qa = same(q_at),
                               ka = same(smem_u32(k_ring + keys.at * T::kSide)), later = t != 0;
                if (elect_one_sync()) {
                    if (t < mine) {
                        const uint64_t vd = block_desc(va, DP * 16u, 128u);
#pragma unroll
                        for (uint32_t k = 0; k < kStepKeys / 16; ++k) mma_weights(to, ts + 8u * k, vd + 2u * DP * k, idesc_o, k != 0 ? 1u : later);
                        umma_commit(&pv_done[g][h]);
                    }
                    umma_commit(&v_empty[values.at]);
                    if (more) scores(ts, qa, ka, t + 2);
                }
                __syncwarp();
                if (more) keys.next();
            }
            mmas_ended<false>(&done[warp - 16]);
        } else if (warp == 18) {
            // lanes 0 .. 7 look a block up each: its scales a tile ahead, its page two
            const auto page_of = [&](int i) { return lane < kBlocks && i < n ? page_at(((long long)from + i) * kKeys + lane * kKvBlock) : -1; };
            const auto scales_of = [&](int page) {
                const size_t at = (size_t)max(page, 0) * c.kv_heads + work.head;
                return page >= 0 ? make_float2(c.key_scales[at], c.value_scales[at]) : make_float2(0.f, 0.f);
            };
            int page = page_of(0), page_next = page_of(1);
            float2 scales = scales_of(page);
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const int slot = i % kAhead, page_now = page;
                const float2 now = scales;
                page = page_next;
                scales = scales_of(page);
                page_next = page_of(i + 2);
                // (a page that is not there: its scores are zeros, -infinity with the exponent.  One that stands for NaNs: the scores say so, and what is times them is finite.)
                const uint32_t k = __float_as_uint(now.x), v = __float_as_uint(now.y);
                const bool number = page_now >= 0 && k < 0x7f800000u && v < 0x7f800000u;
                const int e = (int)(v >> 23) - 127 - (largest == -1000 ? 0 : largest), kept = number ? max(e, -kSpread) : 0;
                if (i >= kAhead && !pair_wait(&m_empty[slot], (uint32_t)(i / kAhead + 1) & 1u, polls)) { ok = false; break; }
                const uint32_t there = __ballot_sync(0xffffffffu, page_now >= 0), zeros = __ballot_sync(0xffffffffu, number && e < -kSpread), numbers = __ballot_sync(0xffffffffu, number || page_now < 0);
                if (lane < kBlocks) blocks[slot][lane] = make_float4(number ? now.x : 1.f, page_now < 0 ? -INFINITY : (float)kept, __uint_as_float((uint32_t)(127 - kept) << 23), __int_as_float(page_now));
                if (lane == 0) which[slot] = make_uint3(there & 0xffu, zeros & 0xffu, numbers & 0xffu);
                __syncwarp();
                if (lane == 0) mbar_arrive(&m_full[slot]);
            }
        }
    }
    if (!ok && lane == 0 && ran_out) {
        *reinterpret_cast<volatile int*>(ran_out) = 1;
        __threadfence_system();
    }
    __syncwarp();
    if (work.chunks > 1) __threadfence();                     // (what this chunk leaves, for whoever joins)
    fence_before();
    __syncthreads();
    if (work.chunks > 1) {
        // The last chunk of an item to come joins all, in their order; where they are many, the last of every `each` in turn joins those, in the first one's place, and the last of
        // these their sums (one CTA reads 128 KB a chunk: 32 rows behind 16384 tokens, 37 chunks, 58 us in one go and 45 in two)
        const int rows = min(kTileRows, pairs - p0);
        float* const weights = reinterpret_cast<float*>(smem);                       // [chunk][row], and behind them what a row's sum is times: where the rings lay
        const auto arrive = [&](int at, int n) {              // true for the last of n
            if (threadIdx.x == 0) largest = atomicAdd(arrived + work.first_cta + at, 1u) == (unsigned)(n - 1);
            __syncthreads();
            if (largest) __threadfence();
            return largest != 0;
        };
        // rows' weights of n chunks that lie `next` rows apart
        const auto weigh = [&](const RowStats* stats, int n, auto next, auto&& told) {
            for (int r = threadIdx.x; r < rows; r += kThreads) {
                float m = -INFINITY, w = -INFINITY, l = 0.f;
                for (int i = 0; i < n; ++i) {
                    m = fmaxf(m, __ldcg(&stats[i * next + r].m));
                    w = fmaxf(w, __ldcg(&stats[i * next + r].w));
                }
                for (int i = 0; i < n; ++i) {
                    l += __ldcg(&stats[i * next + r].l) * lower_to(__ldcg(&stats[i * next + r].m), m);
                    weights[i * kTileRows + r] = lower_to(__ldcg(&stats[i * next + r].w), w);
                }
                told(r, RowStats{m, w, l});
            }
            __syncthreads();
        };
        const auto sum_of = [&](const float* from, int n, auto next, int r, int d) {
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = 0; k < n; ++k) {
                const float f = weights[k * kTileRows + r];
                const float4 z = __ldcg(reinterpret_cast<const float4*>(from + ((size_t)k * next + r) * DP + d));
                sum = make_float4(sum.x + f * z.x, sum.y + f * z.y, sum.z + f * z.z, sum.w + f * z.w);
            }
            return sum;
        };
        const Beside one;
        int each = 1;
        bool here = true;
        if (work.chunks > kJoinOnce) {
            while (each * each < work.chunks) ++each;
            const int from = work.chunk / each * each, n = min(each, work.chunks - from);
            here = arrive(kSms + from + n - 1, n);
            if (here) {
                RowStats* const stats = part_stats + (size_t)(work.first_cta + from) * kTileRows;
                float* const sums = part + (size_t)(work.first_cta + from) * kTileRows * DP;
                weigh(stats, n, one, [&](int r, const RowStats& top) { stats[r] = top; });
#pragma unroll 4
                for (int i = threadIdx.x; i < rows * (DP / 4); i += kThreads)        // (in the place that only this thread reads)
                    *reinterpret_cast<float4*>(sums + 4 * (size_t)i) = sum_of(sums, n, one, i / (DP / 4), i % (DP / 4) * 4);
                __threadfence();
                __syncthreads();
            }
        }
        const auto finish = [&](int n, auto next) {
            weigh(part_stats + (size_t)work.first_cta * kTileRows, n, next, [&](int r, const RowStats& top) {
                weights[n * kTileRows + r] = row_factor(a, work.head * group + (p0 + r) % group, top.m, top.w, top.l);
            });
#pragma unroll 4
            for (int i = threadIdx.x; i < rows * (DP / 4); i += kThreads) {
                const int r = i / (DP / 4), d = i % (DP / 4) * 4, p = p0 + r;
                const float4 sum = sum_of(part + (size_t)work.first_cta * kTileRows * DP, n, next, r, d);
                const float f = weights[n * kTileRows + r], y[4] = {sum.x, sum.y, sum.z, sum.w};
                const size_t to = ((size_t)(q.begin + p / group) * a.heads + work.head * group + p % group) * c.dim + d;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < c.dim) store_out(a, to + e, f * y[e]);
            }
        };
        const int left = (work.chunks + each - 1) / each;
        if (here && arrive(0, left)) {
            if (each == 1) finish(left, one);
            else finish(left, each * kTileRows);
        }
    }
    if (warp == 16) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

template <int DP, int FORMAT>
cudaError_t run_tiles(const Kv8Cache& c, const Kv8Step& s, const Kv8Attention& a, bool alone, void* work, unsigned* arrived, cudaStream_t st) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = ask_smem<kv8_attention_tiles_kernel<DP, FORMAT>>(dev, Tiles<DP>::kSmem);
    if (e != cudaSuccess) return e;
    int* const ran_out = split_attention_ran_out(dev, st);
    if (take_ran_out(dev, st)) return cudaErrorLaunchTimeout;
    float* const part = reinterpret_cast<float*>(work);
    RowStats* const stats = reinterpret_cast<RowStats*>(part + (size_t)kSms * kTileRows * DP);
    // items there may be: full ones, and one that is not for every sequence that has enough rows
    const long long pairs = (long long)s.rows * (a.heads / c.kv_heads), partly = std::min<long long>(s.sequences, pairs / (a.few_most + 1));
    const long long ctas = std::max<long long>(kSms, c.kv_heads * (pairs / kTileRows + partly));
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    return launch_pdl(kv8_attention_tiles_kernel<DP, FORMAT>, dim3((unsigned)ctas), dim3(kThreads), Tiles<DP>::kSmem, st, c, s, a, (int)alone, part, stats, arrived, ran_out, gemm_pair_polls());
}

}  // namespace

bool kv8_tiles_ok(int dim, int type) { return dim <= 128 && type != kTypeF32; }

size_t kv8_tiles_work_bytes(int dim) { return (size_t)kSms * kTileRows * ((dim <= 64 ? 64 : 128) * sizeof(float) + sizeof(RowStats)); }

cudaError_t launch_kv8_tiles(const Kv8Cache& c, const Kv8Step& s, const Kv8Attention& a, bool alone, void* work, unsigned* arrived, cudaStream_t st) {
    if (c.dim <= 64) return c.format == kKvE4m3 ? run_tiles<64, kKvE4m3>(c, s, a, alone, work, arrived, st) : run_tiles<64, kKvInt8>(c, s, a, alone, work, arrived, st);
    return c.format == kKvE4m3 ? run_tiles<128, kKvE4m3>(c, s, a, alone, work, arrived, st) : run_tiles<128, kKvInt8>(c, s, a, alone, work, arrived, st);
}

}  // namespace lm
